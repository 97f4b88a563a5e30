// Products of secret shares with cleartext weights in Z_{2^l}, grouped by expert:
//   out[r][o] = add[r][o] + sum_k (x[t][k] + x1[t][k]) * w[g][o][k]  mod 2^l,   t = rows[r], offsets[g] <= r < offsets[g+1]
//
// Mathematics.  Both operands are written in balanced base-256 digits, x = sum x_i 256^i and w = sum w_j 256^j with
// digits in [-128, 127]: with C = 0x80...80, the digits of v are the bytes of (v + C) ^ C (adding C makes every byte
// digit + 128, the exclusive or takes the 128 off again as a signed byte).  l bits need nx = ceil(l/8) digits of x (what
// lies above is a multiple of 2^l), the weights as many as the widest of all groups asks for, found when they are laid out (one
// 16-bit weight above 32639 makes them all three).  The product modulo 2^l is then sum over s < nx of 256^s * sum_{i+j=s} x_i w_j, every inner sum an exact i8 x i8 -> i32
// matrix product, nx accumulators per output.  |x_i w_j| <= 2^14 and at most nw products share an accumulator, so up to
// (2^17 - 1) / nw terms of k cannot overflow; longer k is added up in 64-bit pieces.  Everything is exact: the result does
// not depend on the order of the sums.
//
// Bounds.  nx nw - nw (nw - 1) / 2 byte products per multiplication (15 for 64 bits and two-byte weights), at the rate
// v_mfma_i32_32x32x32_i8 sustains on random digits from registers: 21 ns per instruction and SIMD, 3.2 P operations/s (4.2 P on
// constant ones: the chip lowers its clock; the 16x16x64 form reaches 0.6 of that).  Few rows: the bytes of the weights' digits.
#include <algorithm>
#include <new>

#include "common.hpp"

struct mmh_ring_weights {
  int device = 0;
  size_t groups = 0, rows = 0, cols = 0;
  int bw = 0, nx = 0, nw = 0;   // nw: digits stored per weight (a width the product kernels exist for)
  size_t k32 = 0, out32 = 0;    // fragments along the columns (an even number) and the outputs
  int8_t *d = nullptr;          // [group][out32][k32][digit][2][32 outputs][16 columns]: 1 KiB matrix-core fragments
};

namespace mmh {
constexpr size_t kRingGroups = 32767;   // row tiles, one more at most per group, are the second dimension of a grid (16 bits)
typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v16i __attribute__((ext_vector_type(16)));

struct RingArgs {
  const int8_t *w;
  const u64 *x, *x1, *add;
  const int64_t *rows, *offsets;
  u64 *out, *ws;               // ws: where the parts of k go that ring_join_kernel adds up (null: straight to out)
  size_t ldx, ldx1, ldadd, ldo, n_tokens, n_rows;
  int groups, cols, n_out, k32, out32, out_tiles, row_tiles;
  u64 mask;
  int zero_rest;
};

// Row tiles of BM rows; tiles do not cross groups.  A wave looks at 64 groups at a time, a group per lane, with a prefix sum of
// their tile counts.  Offsets are clamped to [0, n_rows], so nothing they hold leads out of bounds.
template <int BM>
struct RingGroups {
  long long s, e;   // rows of this lane's group
  u32 tiles, sum;   // its tiles, and those of all groups of the wave up to it
  __device__ __forceinline__ void load(const RingArgs &a, int g0) {
    const int lane = threadIdx.x & 63;
    s = e = 0;
    if (g0 + lane < a.groups) {
      const long long n = (long long)a.n_rows;
      s = a.offsets[g0 + lane], e = a.offsets[g0 + lane + 1];
      s = s < 0 ? 0 : s > n ? n : s;
      e = e < s ? s : e > n ? n : e;
    }
    tiles = (u32)((e - s + BM - 1) / BM);
    sum = tiles;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const u32 t = __shfl_up(sum, d);
      if (lane >= d) sum += t;
    }
  }
  __device__ __forceinline__ u32 total() const { return __builtin_amdgcn_readlane(sum, 63); }
};
struct RingTile {
  int g, ot;
  size_t lo, hi;
};
// row tile `tile`; `first` holds groups 0 .. 63
template <int BM>
__device__ __forceinline__ bool ring_find_tile(const RingArgs &a, const RingGroups<BM> &first, u32 tile, RingTile &t) {
  if (!a.offsets) {
    t.g = 0, t.lo = (size_t)tile * BM;
    t.hi = t.lo + BM < a.n_rows ? t.lo + BM : a.n_rows;
    return t.lo < a.n_rows;
  }
  RingGroups<BM> w = first;
  u32 before = 0;
  for (int g0 = 0;;) {
    const unsigned long long past = __ballot(before + w.sum > tile);
    if (past) {
      const int src = __ffsll(past) - 1;
      const u32 at = before + __builtin_amdgcn_readlane(w.sum - w.tiles, src);
      t.lo = make64(__builtin_amdgcn_readlane(lo32(w.s), src), __builtin_amdgcn_readlane(hi32(w.s), src)) + (u64)(tile - at) * BM;
      const size_t end = make64(__builtin_amdgcn_readlane(lo32(w.e), src), __builtin_amdgcn_readlane(hi32(w.e), src));
      t.hi = t.lo + BM < end ? t.lo + BM : end;
      t.g = g0 + src;
      return true;
    }
    before += w.total();
    g0 += 64;
    if (g0 >= a.groups) return false;
    w.load(a, g0);
  }
}
template <int BM>
__device__ __forceinline__ u32 ring_count_tiles(const RingArgs &a, const RingGroups<BM> &first) {
  if (!a.offsets) return (u32)((a.n_rows + BM - 1) / BM);
  u32 n = first.total();
  for (int g0 = 64; g0 < a.groups; g0 += 64) {
    RingGroups<BM> more;
    more.load(a, g0);
    n += more.total();
  }
  return n < (u32)a.row_tiles ? n : (u32)a.row_tiles;   // groups that overlap, which none may, could have more than the grid
}

// The tile of a workgroup.  Workgroups go round the 8 XCDs, each with an L2 of its own; what runs on an XCD at one time should
// share rows and weights, so each has a contiguous piece of the order "16 output tiles across, row tiles down", of the row tiles
// that the groups have.  (Four across reads rows four times over where they come from memory: 8192 x 4096 x 4096 with two shares
// 1.97 ms against 1.91.  Row tiles dealt out to the XCDs one by one leave up to a row of tiles more on one of them: 777 x 1023 x 515
// in three parts 30 us.)
__device__ __forceinline__ bool ring_block(const RingArgs &a, u32 row_tiles, int &ot, u32 &rt) {
  constexpr u32 kAcross = 16;
  const u32 out_tiles = (u32)a.out_tiles, total = out_tiles * row_tiles, per = (total + 7) / 8;
  const u32 q = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
  if ((blockIdx.x >> 3) >= per || q >= total) return false;
  const u32 panel = q / (kAcross * row_tiles), rest = q - panel * kAcross * row_tiles;
  const u32 wide = out_tiles - panel * kAcross < kAcross ? out_tiles - panel * kAcross : kAcross;
  rt = rest / wide, ot = (int)(panel * kAcross + rest % wide);
  return true;
}

// the row of x that row r reads, or -1 (an index outside [0, n_tokens) reads as a row of zeros)
__device__ __forceinline__ long long ring_token(const RingArgs &a, size_t r) {
  const long long t = a.rows ? a.rows[r] : (long long)r;
  return t >= 0 && t < (long long)a.n_tokens ? t : -1;
}

// rows that no group has, in the columns [n0, n1): zeros, where the caller asked for them; workgroup `part` of `parts` on them
__device__ __forceinline__ void ring_zero_rest(const RingArgs &a, int n0, int n1, u32 part, u32 parts) {
  if (!a.zero_rest || !a.offsets) return;
  const long long n = (long long)a.n_rows;
  long long b = a.offsets[0], e = a.offsets[a.groups];
  b = b < 0 ? 0 : b > n ? n : b, e = e < b ? b : e > n ? n : e;
  n1 = n1 < a.n_out ? n1 : a.n_out;
  for (long long i = part; i < n - (e - b); i += parts) {
    u64 *p = a.out + (size_t)(i < b ? i : i + (e - b)) * a.ldo;
    for (int c = n0 + (int)threadIdx.x; c < n1; c += blockDim.x) p[c] = 0;
  }
}

struct __attribute__((packed, aligned(8))) Words2 {   // 16-byte accesses to 8-byte aligned words
  u64 v[2];
};
__device__ __forceinline__ void ring_load4(const u64 *p, u64 (&v)[4]) {
  const Words2 t = reinterpret_cast<const Words2 *>(p)[0], u = reinterpret_cast<const Words2 *>(p)[1];
  v[0] = t.v[0], v[1] = t.v[1], v[2] = u.v[0], v[3] = u.v[1];
}
__device__ __forceinline__ void ring_store4(u64 *p, const u64 (&v)[4]) {
  reinterpret_cast<Words2 *>(p)[0] = Words2{{v[0], v[1]}};
  reinterpret_cast<Words2 *>(p)[1] = Words2{{v[2], v[3]}};
}
// bytes e[0..3].b -> one dword per byte place: a 4 x 4 byte transposition
__device__ __forceinline__ void transpose4(u32 e0, u32 e1, u32 e2, u32 e3, u32 (&d)[4]) {
  const u32 l0 = __builtin_amdgcn_perm(e1, e0, 0x05010400), h0 = __builtin_amdgcn_perm(e1, e0, 0x07030602);
  const u32 l1 = __builtin_amdgcn_perm(e3, e2, 0x05010400), h1 = __builtin_amdgcn_perm(e3, e2, 0x07030602);
  d[0] = __builtin_amdgcn_perm(l1, l0, 0x05040100), d[1] = __builtin_amdgcn_perm(l1, l0, 0x07060302);
  d[2] = __builtin_amdgcn_perm(h1, h0, 0x05040100), d[3] = __builtin_amdgcn_perm(h1, h0, 0x07060302);
}
constexpr u64 kDigitBias = 0x8080808080808080ull;
// digits of four words: dig[i] holds digit i of each
template <int NX>
__device__ __forceinline__ void ring_digits4(const u64 (&v)[4], u32 (&dig)[8]) {
  u64 t[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) t[e] = v[e] + kDigitBias;
  u32 d[4];
  transpose4(lo32(t[0]), lo32(t[1]), lo32(t[2]), lo32(t[3]), d);
#pragma unroll
  for (int i = 0; i < 4; ++i) dig[i] = d[i] ^ 0x80808080u;
  if (NX > 4) {
    transpose4(hi32(t[0]), hi32(t[1]), hi32(t[2]), hi32(t[3]), d);
#pragma unroll
    for (int i = 0; i < 4; ++i) dig[4 + i] = d[i] ^ 0x80808080u;
  }
}

__device__ __forceinline__ v4i as_v4i(const uint4 &t) { return v4i{(int)t.x, (int)t.y, (int)t.z, (int)t.w}; }
// sum_s 256^s acc_s mod 2^64: what lies at 2^32 and above in 32-bit arithmetic
template <int NX, typename T>
__device__ __forceinline__ u64 ring_value(const T (&acc)[NX], int e) {
  u64 v = (u64)(long long)acc[0][e];
#pragma unroll
  for (int s = 1; s < NX && s < 4; ++s) v += (u64)((long long)acc[s][e] * (1 << 8 * s));
  u32 h = hi32(v);
#pragma unroll
  for (int s = 4; s < NX; ++s) h += (u32)acc[s][e] << (8 * (s - 4));
  return make64(lo32(v), h);
}

// ---- which columns a step's 64 places hold: the last step ends with the last column, and with fewer than 64 columns so does the
// last piece of four that a lane loads.  Nothing is read past a row's end; weights at places whose column an earlier place has
// (or that there is none for) are laid out as zeros.
__device__ __forceinline__ int ring_step_column(int cols, int c) {
  const int k = c * 64;
  return k + 64 <= cols ? k : cols < 64 ? 0 : cols - 64;
}
__device__ __forceinline__ int ring_piece(int cols, int place) { return cols < 64 && place + 4 > cols ? cols - 4 : place; }

// Fewer than 4 columns: 64-bit products, one output a lane.
__global__ __launch_bounds__(256) void ring_narrow_kernel(RingArgs a, int nw) {
  ring_zero_rest(a, (int)blockIdx.x * 256, (int)blockIdx.x * 256 + 256, blockIdx.y, gridDim.y);
  RingGroups<32> groups;
  RingTile tile;
  if (a.offsets) groups.load(a, 0);
  if (!ring_find_tile(a, groups, blockIdx.y, tile)) return;
  const int n = (int)(blockIdx.x * 256 + threadIdx.x);
  if (n >= a.n_out) return;
  u64 w[3];
  for (int k = 0; k < a.cols; ++k) {
    w[k] = 0;
    for (int j = 0; j < nw; ++j)
      w[k] += (u64)(long long)a.w[(((size_t)tile.g * a.out32 + (n >> 5)) * a.k32 * nw + j) * 1024 + (n & 31) * 16 + k] << (8 * j);
  }
  for (size_t row = tile.lo; row < tile.hi; ++row) {
    const long long t = ring_token(a, row);
    u64 v = a.add ? a.add[row * a.ldadd + n] : 0;
    for (int k = 0; k < a.cols && t >= 0; ++k)
      v += (a.x[(size_t)t * a.ldx + k] + (a.x1 ? a.x1[(size_t)t * a.ldx1 + k] : 0)) * w[k];
    a.out[row * a.ldo + n] = v & a.mask;
  }
}

// Up to 8 rows: a workgroup computes them for 16 outputs, its 16 waves split k in steps of 64 columns and join their 64-bit sums
// through LDS.  Bound by latency: everything a wave needs of its first steps is asked for at once (kAhead steps), and it cuts
// its own digits into LDS of its own, so the loop has no barrier.  16 x 16 products (v_mfma_i32_16x16x64_i8), of whose rows 8
// stay zero: their rate does not matter here, their few registers do.  4 columns or more.
// us by rows, 64 bits and two-byte weights, calls back to back in a graph (a kernel trace reads 0.3 to 0.8 more), against the tile
// kernel with k split and its second launch:
//   2048 -> 1001: 1 row 5.0 (11.3), 4 5.5 (11.5), 8 7.4 (11.5);  4096 -> 4096: 1 row 7.4 (15.0; 33.5 MB of digits = 4.5 TB/s),
//   8 12.4 (15.7);  8192 -> 1024: 1 row 9.0 (19.1), 8 19.3 (18.9).  16 rows would read twice the words per workgroup.
// Eight digits of both operands with a second share spill 36 registers; no other variant spills.
template <int NX, int NW, bool TWO>
__global__ __launch_bounds__(1024) void ring_few_kernel(RingArgs a) {
  constexpr int W = 16, kAhead = NW <= 2 && !TWO ? 2 : 1;
  __shared__ uint4 lds[W][NX * 64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int ot = (int)blockIdx.x;   // 16 outputs
  ring_zero_rest(a, ot * 16, ot * 16 + 16, blockIdx.y, gridDim.y);
  RingGroups<8> groups;
  RingTile tile;
  if (a.offsets) groups.load(a, 0);
  if (!ring_find_tile(a, groups, blockIdx.y, tile)) return;
  const int g = tile.g;
  const size_t lo = tile.lo, hi = tile.hi;
  // a lane cuts four words of rows lane % 4 and, with more than four rows, lane % 4 + 4
  const int r = lane & 3, k4 = lane >> 2;
  const bool eight = hi - lo > 4;
  const u64 *px[2], *px1[2];
#pragma unroll
  for (int b = 0; b < 2; ++b) {
    const size_t row = lo + 4 * b + r;
    const long long t = row < hi ? ring_token(a, row) : -1;
    const size_t token = t < 0 ? 0 : (size_t)t;   // any row will do: its sums are not used
    const int piece = ring_piece(a.cols, k4 * 4);
    px[b] = a.x + token * a.ldx + piece, px1[b] = TWO ? a.x1 + token * a.ldx1 + piece : nullptr;
  }
  // 16 outputs x 64 columns of a step's two fragments: lane (quarter, output) reads 16 columns
  const int8_t *pw = a.w + ((size_t)g * a.out32 + (ot >> 1)) * a.k32 * (NW * 1024) + (lane >> 5) * (NW * 1024) +
                     (lane >> 4 & 1) * 512 + ((ot & 1) * 16 + (lane & 15)) * 16;
  const int last = a.k32 / 2 - 1;
  struct Step {
    v4i w[NW];
    u64 x[2][4], x1[TWO ? 2 : 1][4];
  } s[kAhead];
  auto load = [&](Step &v, int c) {
    c = c < last ? c : last;
    const int k = ring_step_column(a.cols, c);
#pragma unroll
    for (int j = 0; j < NW; ++j) v.w[j] = *reinterpret_cast<const v4i *>(pw + ((size_t)2 * c * NW + j) * 1024);
#pragma unroll
    for (int b = 0; b < 2; ++b)
      if (b == 0 || eight) {
        ring_load4(px[b] + k, v.x[b]);
        if constexpr (TWO) ring_load4(px1[b] + k, v.x1[b]);
      }
  };
#pragma unroll
  for (int i = 0; i < kAhead; ++i) load(s[i], wave + i * W);
#pragma unroll
  for (int i = 0; i < NX; ++i) lds[wave][i * 64 + lane] = make_uint4(0, 0, 0, 0);
  v4i acc[NX];
#pragma unroll
  for (int i = 0; i < NX; ++i) acc[i] = v4i{0, 0, 0, 0};
  auto step = [&](Step &v, int c) {
#pragma unroll
    for (int b = 0; b < 2; ++b)
      if (b == 0 || eight) {
        u64 t[4];
        u32 dig[8];
#pragma unroll
        for (int e = 0; e < 4; ++e) t[e] = TWO ? v.x[b][e] + v.x1[TWO ? b : 0][e] : v.x[b][e];
        ring_digits4<NX>(t, dig);
#pragma unroll
        for (int d = 0; d < NX; ++d) reinterpret_cast<u32 *>(&lds[wave][d * 64 + (k4 >> 2) * 16 + 4 * b + r])[k4 & 3] = dig[d];
      }
    v4i w[NW];
#pragma unroll
    for (int j = 0; j < NW; ++j) w[j] = v.w[j];
    if (c + kAhead * W <= last) load(v, c + kAhead * W);
#pragma unroll
    for (int i = 0; i < NX; ++i) {
      const v4i x = as_v4i(lds[wave][i * 64 + lane]);
#pragma unroll
      for (int j = 0; j < NW; ++j)
        if (i + j < NX) acc[i + j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[j], x, acc[i + j], 0, 0, 0);
    }
  };
  for (int c = wave; c <= last; c += kAhead * W)
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
      if (c + i * W <= last) step(s[i], c + i * W);
  // element e of a lane: row lane % 16, output 4 * (lane / 16) + e
  __syncthreads();
  u64 *part = reinterpret_cast<u64 *>(&lds[0][0]);   // [wave][row][output]
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if ((lane & 15) < 8) part[(wave * 8 + (lane & 15)) * 16 + (lane >> 4) * 4 + e] = ring_value<NX>(acc, e);
  }
  __syncthreads();
  const int i = (int)threadIdx.x, row = i >> 4, n = ot * 16 + (i & 15);
  if (i >= 128 || lo + row >= hi || n >= a.n_out) return;
  u64 v = a.add ? a.add[(lo + row) * a.ldadd + n] : 0;
  if (ring_token(a, lo + row) >= 0)
#pragma unroll
    for (int k = 0; k < W; ++k) v += part[(k * 8 + row) * 16 + (i & 15)];
  a.out[(lo + row) * a.ldo + n] = v & a.mask;
}

// Large products: a workgroup of 8 waves computes 32 rows x 256*OT outputs in steps of 64 columns.  The rows' digits are cut
// once per workgroup into LDS (three buffers, one barrier per step); the weights' fragments come straight from L2 in the order
// they were laid out in.  Words and weights are loaded into registers two steps before they are used; nothing in the loop
// branches.  4 columns or more.
template <int NX, int NW, int OT, bool TWO>
__global__ __launch_bounds__(512, 2) void ring_tile_kernel(RingArgs a) {
  __shared__ uint4 xs[3][2 * NX * 64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int r = lane & 15, sub = lane >> 4;
  RingGroups<32> groups;
  if (a.offsets) groups.load(a, 0);
  if (!a.ws) {   // the grid has a workgroup for each output tile, at least
    const u32 parts = gridDim.x / a.out_tiles, part = blockIdx.x / a.out_tiles, t = blockIdx.x - part * a.out_tiles;
    if (part < parts) ring_zero_rest(a, t * 256 * OT, (t + 1) * 256 * OT, part, parts);
  }
  const int last = a.k32 / 2 - 1;
  const int first = (int)((long long)(last + 1) * blockIdx.y / gridDim.y);
  const int end = (int)((long long)(last + 1) * (blockIdx.y + 1) / gridDim.y);

  u32 rt;
  RingTile tile;
  if (!ring_block(a, ring_count_tiles(a, groups), tile.ot, rt)) return;
  if (!ring_find_tile(a, groups, rt, tile)) return;
  const size_t lo = tile.lo, hi = tile.hi;
  const int ot0 = (tile.ot * 8 + wave) * OT;
  // this wave cuts the 16 x 16 block (row half wave % 2, column quarter wave / 2) of every step
  const size_t my_row = lo + (wave & 1) * 16 + r;
  const long long my_token = my_row < hi ? ring_token(a, my_row) : -1;
  const size_t token = my_token < 0 ? 0 : (size_t)my_token;   // any row will do: its sums are not used
  const int in_step = ring_piece(a.cols, (wave >> 1) * 16 + sub * 4);
  const u64 *px = a.x + token * a.ldx + in_step, *px1 = TWO ? a.x1 + token * a.ldx1 + in_step : nullptr;
  const int8_t *pw[OT];
#pragma unroll
  for (int o = 0; o < OT; ++o) {
    const int n = ot0 + o < a.out32 ? ot0 + o : a.out32 - 1;
    pw[o] = a.w + ((size_t)tile.g * a.out32 + n) * a.k32 * (NW * 1024);
  }

  struct Words {
    u64 x[4], x1[TWO ? 4 : 1];
  };
  Words words[2];
  auto load_x = [&](Words &v, int c) {
    c = c < last ? c : last;
    const int k = ring_step_column(a.cols, c);
    ring_load4(px + k, v.x);
    if constexpr (TWO) ring_load4(px1 + k, v.x1);
  };
  // half 0: digits 0 .. 3, half 1: the others
  auto store_x = [&](const Words &v, int buf, int half) {
    u32 d[4];
    u64 t[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) t[e] = (TWO ? v.x[e] + v.x1[TWO ? e : 0] : v.x[e]) + kDigitBias;
    if (half == 0) transpose4(lo32(t[0]), lo32(t[1]), lo32(t[2]), lo32(t[3]), d);
    else transpose4(hi32(t[0]), hi32(t[1]), hi32(t[2]), hi32(t[3]), d);
    uint4 *frag = xs[buf] + (wave >> 2) * (NX * 64) + (wave >> 1 & 1) * 32 + (wave & 1) * 16 + r;
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (4 * half + k < NX) reinterpret_cast<u32 *>(frag + (4 * half + k) * 64)[sub] = d[k] ^ lo32(kDigitBias);
  };
  constexpr int kSets = NW <= (OT == 1 ? 4 : 5 - NX) ? 2 : 1;   // weights are loaded this many steps before their use (registers)
  v4i w[kSets][2][OT][NW];
  v16i acc[OT][NX];
  auto load_w = [&](int p, int h, int c) {
    c = c < last ? c : last;
#pragma unroll
    for (int o = 0; o < OT; ++o)
#pragma unroll
      for (int j = 0; j < NW; ++j) w[p % kSets][h][o][j] = reinterpret_cast<const v4i *>(pw[o] + ((size_t)(2 * c + h) * NW + j) * 1024)[lane];
  };
  // fragment t of a step (column half t / NX, digit t % NX) is read from LDS D products' places ahead of its use
  constexpr int D = NX == 5 ? 4 : 3;
  static_assert(2 * NX % (D + 1) == 0, "a step leaves the ring of fragments where it found it");
  v4i f[D + 1];
  // the barrier orders LDS alone: loads from memory stay in flight across it
  auto barrier = [] { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); };
  // Step c: products from buffer rd, digits of step c + 2 into wr, words and weights of set p.  All waves have read the last of
  // wr, the buffer of step c - 1, when they reach this step's barrier, so it is written behind it; the next step's barrier
  // publishes the digits, before the end of that step starts to read them.
  constexpr int kBarrier = NX / 2, kCut = kBarrier + 1;
  static_assert(kCut + 2 < 2 * NX && kBarrier < 2 * NX - D, "cut within the step, read ahead behind the barrier");
  int rd = 0, nx = 1, wr = 2;
  // Products, reads and the cutting of digits are kept in this order (sched_barrier): moved together, the cutting would wait
  // for words that were only just asked for, and reads for products.
  auto step = [&](int p, int c) {
#pragma unroll
    for (int t = 0; t < 2 * NX; ++t) {
      const int n = t + D, i = t % NX, h = t / NX;
      f[n % (D + 1)] = as_v4i(n < 2 * NX ? xs[rd][n * 64 + lane] : xs[nx][(n - 2 * NX) * 64 + lane]);
#pragma unroll
      for (int o = 0; o < OT; ++o)
#pragma unroll
        for (int j = 0; j < NW; ++j)
          if (i + j < NX)
            acc[o][i + j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(w[p % kSets][h][o][j], f[t % (D + 1)], acc[o][i + j], 0, 0, 0);
      if (t == kBarrier) barrier();
      if (t == kCut) store_x(words[p], wr, 0);
      if (NX > 4 && t == kCut + 2) store_x(words[p], wr, 1);
      if (t == NX - 1) load_w(p, 0, c + kSets);
      __builtin_amdgcn_sched_barrier(0x4);   // scalar arithmetic may cross
    }
    load_x(words[p], c + 4);
    load_w(p, 1, c + kSets);
    const int t = rd;
    rd = nx, nx = wr, wr = t;
    __builtin_amdgcn_sched_barrier(0x4);
  };
  constexpr int kFlush = 131071 / NW / 64;   // steps whose sums fit 32 bits
  for (int c0 = first; c0 < end; c0 += kFlush) {
    const int c1 = c0 + kFlush < end ? c0 + kFlush : end;
    Words one, two;
    load_x(one, c0);
    load_x(two, c0 + 1);
#pragma unroll
    for (int p = 0; p < kSets; ++p) load_w(p, 0, c0 + p), load_w(p, 1, c0 + p);
    load_x(words[0], c0 + 2);
    load_x(words[1], c0 + 3);
    barrier();   // the last segment's digits have been read
#pragma unroll
    for (int half = 0; half < (NX > 4 ? 2 : 1); ++half) store_x(one, rd, half), store_x(two, nx, half);
#pragma unroll
    for (int o = 0; o < OT; ++o)
#pragma unroll
      for (int s = 0; s < NX; ++s)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[o][s][e] = 0;
    barrier();
#pragma unroll
    for (int t = 0; t < D; ++t) f[t] = as_v4i(xs[rd][t * 64 + lane]);
    int c = c0;
    for (; c + 1 < c1; c += 2) step(0, c), step(1, c + 1);
    if (c < c1) step(0, c);
    // element e of a lane: row lane % 32, output e % 4 + 8 * (e / 4) + 4 * (lane / 32)
    const size_t row = lo + (lane & 31);
    if (row < hi) {
      const bool none = ring_token(a, row) < 0;
      u64 *dst = a.ws ? a.ws + ((size_t)blockIdx.y * a.n_rows + row) * a.n_out : a.out + row * a.ldo;
      const u64 *base = c0 > first ? dst : a.add && !a.ws ? a.add + row * a.ldadd : nullptr;
#pragma unroll
      for (int o = 0; o < OT; ++o)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int n = (ot0 + o) * 32 + q * 8 + (lane >> 5) * 4;
          u64 v[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            v[e] = none ? 0 : ring_value<NX>(acc[o], q * 4 + e);
            if (base && n + e < a.n_out) v[e] += base[n + e];
            v[e] &= a.mask;
          }
          if (n + 4 <= a.n_out) ring_store4(dst + n, v);
          else
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (n + e < a.n_out) dst[n + e] = v[e];
        }
    }
  }
}

// the parts of k that several workgroups summed: out = add + sum of the parts, two outputs a lane, four parts asked for at once
__global__ __launch_bounds__(256) void ring_join_kernel(RingArgs a, int parts) {
  const int n = (int)(blockIdx.x * 256 + threadIdx.x) * 2;
  if (n >= a.n_out) return;
  const bool pair = n + 1 < a.n_out;
  const size_t stride = a.n_rows * a.n_out;
  for (size_t row = blockIdx.y; row < a.n_rows; row += gridDim.y) {
    u64 v[2] = {0, 0};
    if (a.offsets && ((long long)row < a.offsets[0] || (long long)row >= a.offsets[a.groups])) {
      if (!a.zero_rest) continue;
    } else {
      const u64 *ws = a.ws + row * a.n_out + n;
      for (int p = 0; p < parts; p += 4) {
        u64 u[4][2];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const u64 *q = ws + (p + i < parts ? p + i : p) * stride;
          u[i][0] = q[0], u[i][1] = q[pair];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (p + i < parts) v[0] += u[i][0], v[1] += u[i][1];
      }
      if (a.add) v[0] += a.add[row * a.ldadd + n], v[1] += a.add[row * a.ldadd + n + pair];
    }
    u64 *out = a.out + row * a.ldo + n;
    out[0] = v[0] & a.mask;
    if (pair) out[1] = v[1] & a.mask;
  }
}

// ---- weights: how many digits the widest needs, then the layout
template <typename T>
__device__ __forceinline__ long long ring_weight(const T *w, size_t i, int bw) {
  const long long v = (long long)w[i];
  return bw < 64 ? (long long)((u64)v << (64 - bw)) >> (64 - bw) : v;   // the representative next to zero
}
template <typename T>
__global__ __launch_bounds__(256) void ring_weight_digits_kernel(const T *__restrict__ w, size_t n, int bw, int *need) {
  int m = 1;
  for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (size_t)gridDim.x * 256) {
    const long long v = ring_weight(w, i, bw);
    // v has d balanced digits when v + 0x80..80 (d bytes) lies in [0, 256^d)
    while (m < 8 && ((u64)v + (0x8080808080808080ull >> (64 - 8 * m))) >> (8 * m)) ++m;
  }
#pragma unroll
  for (int d = 32; d; d >>= 1) m = max(m, __shfl_xor(m, d));
  __shared__ int waves[4];
  if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = m;
  __syncthreads();
  m = max(max(waves[0], waves[1]), max(waves[2], waves[3]));
  if (threadIdx.x == 0 && *(volatile int *)need < m) atomicMax(need, m);
}
template <typename T>
__global__ __launch_bounds__(256) void ring_weight_layout_kernel(const T *__restrict__ w, size_t rows, size_t cols, int bw,
                                                                 size_t out32, size_t k32, int nw, size_t n_units,
                                                                 int8_t *__restrict__ out) {
  // u: (group, out32, k32, half, output), 16 columns of a row
  for (size_t u = (size_t)blockIdx.x * 256 + threadIdx.x; u < n_units; u += (size_t)gridDim.x * 256) {
    const size_t frag = u >> 6, c = frag % k32, ot = frag / k32 % out32, g = frag / k32 / out32;
    const size_t step = c >> 1, o = ot * 32 + (u & 31), place = (c & 1) * 32 + (u >> 5 & 1) * 16;
    u64 t[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const size_t piece = (place + e) & ~size_t(3);
      const size_t k = cols < 4 ? place + e : ring_step_column((int)cols, (int)step) + ring_piece((int)cols, (int)piece) + (e & 3);
      const bool in = o < rows && k < cols && k >= step * 64 && (cols >= 64 || k >= piece);
      const u64 C = 0x8080808080808080ull;
      t[e] = ((u64)(in ? ring_weight(w, (g * rows + o) * cols + k, bw) : 0) + C) ^ C;
    }
    for (int j = 0; j < nw; ++j) {
      u32 d[4] = {0, 0, 0, 0};
#pragma unroll
      for (int e = 0; e < 16; ++e) d[e >> 2] |= (u32)(t[e] >> (8 * j) & 0xff) << (8 * (e & 3));
      *reinterpret_cast<uint4 *>(out + (frag * nw + j) * 1024 + (u & 63) * 16) = make_uint4(d[0], d[1], d[2], d[3]);
    }
  }
}

template <typename T>
static void ring_launch_digits(const void *w, size_t n, int bw, int *need, hipStream_t s) {
  hipLaunchKernelGGL(ring_weight_digits_kernel<T>, dim3((unsigned)std::min<size_t>((n + 255) / 256, 2048)), dim3(256), 0, s,
                     (const T *)w, n, bw, need);
}
template <typename T>
static void ring_launch_layout(const void *w, const mmh_ring_weights *h, hipStream_t s) {
  const size_t units = h->groups * h->out32 * h->k32 * 64;
  hipLaunchKernelGGL(ring_weight_layout_kernel<T>, dim3((unsigned)std::min<size_t>((units + 255) / 256, 65536)), dim3(256), 0, s,
                     (const T *)w, h->rows, h->cols, h->bw, h->out32, h->k32, h->nw, units, h->d);
}

// Parts of k, by which few tiles fill the chip (48 x 4096 x 4096 72 -> 28 us, 200 x 4096 x 1024 72 -> 26, 64 x 1024 x 1024 23 -> 13),
// by a model of the tile kernel's time (us): rounds of workgroups on the 32 compute units of each XCD, each round its steps and 5
// us for its start and its results; the second launch and 16 bytes of traffic per part and output.  A step of 30 products takes
// 1.05 us on a few compute units and 1.45 with all of them busy, one of a few products no less than 0.9.
static int ring_parts(size_t tiles, size_t steps, int products, size_t outputs) {
  auto time = [&](int p) {
    const double busy = std::min(1.0, (double)(tiles * p) / 256), step = std::max(0.9, products * (0.035 + 0.0133 * busy));
    const double rounds = (double)(((tiles + 7) / 8 * p + 31) / 32);
    return rounds * ((double)((steps + p - 1) / p) * step + 5) + (p > 1 ? 2.5 + p * (double)outputs * 16 / 2.8e6 : 0);
  };
  int best = 1;
  double least = 0.95 * time(1);   // one launch unless two are faster
  for (int p = 2; p <= 16 && (size_t)p * 2 <= steps; ++p)
    if (time(p) < least) best = p, least = time(p);
  return best;
}
// up to 8 rows in all go to ring_few_kernel, whose waves must not sum more columns than fit 32 bits and whose grid, 1024 lanes for
// 16 outputs, has to stay below 2^32 lanes
static bool ring_few(size_t n_rows, size_t rows, size_t cols, int nw) {
  return n_rows <= 8 && (cols / 64 / 16 + 1) * 64 * nw <= 131071 && (rows + 15) / 16 < (size_t(1) << 22);
}
static constexpr int ring_products(int nx, int nw) { return 2 * (nx * nw - nw * (nw - 1) / 2); }   // of a 64-column step
// 32-output tiles a wave computes.  Two halve the reads of digits from LDS, which bound the product when there are few digits;
// their sums take 32 nx registers of a lane's 256.  4 x 1, 4 x 2 and 5 x 1 digits fit; 5 x 1 with a second share spills 2 registers,
// 5 x 2 10 and 6 x 1 14, and all of them keep some 80 scalars in vector registers.  They pay nevertheless when the chip has work
// enough: 4096 x 2048 x 2048 with digits 4 x 1 135 -> 80 us, 4 x 2 135 -> 114, 5 x 1 121 -> 90, 6 x 1 121 -> 101, 5 x 2 155 -> 138,
// but 1024 rows 35 -> 39 us (5 x 1), 40 -> 52 us (5 x 2).  Of the tiles of one, 8 x 4 (8) and 8 x 8 (6) with a second share spill.
static constexpr bool ring_wide_fits(int nx, int nw, bool two) { return nx + nw <= 6 || (!two && nx + nw <= 7 && nw <= 2); }
static size_t ring_out_tiles(size_t out32, int ot) { return (out32 + 8 * ot - 1) / (8 * ot); }
static bool ring_wide(int nx, int nw, bool two, size_t out32, size_t row_tiles) {
  return ring_wide_fits(nx, nw, two) && ring_out_tiles(out32, 2) * row_tiles >= 256;
}
// parts of k of a call (1: the tile kernel writes the result itself)
static int ring_call_parts(int nx, int nw, bool two, size_t out32, size_t row_tiles, size_t steps, size_t outputs) {
  const int ot = ring_wide(nx, nw, two, out32, row_tiles) ? 2 : 1;
  return ring_parts(ring_out_tiles(out32, ot) * row_tiles, steps, ot * ring_products(nx, nw), outputs);
}

template <int NX, int NW, int OT, bool TWO>
static void ring_launch_tiles(RingArgs a, hipStream_t s, int parts) {
  a.out_tiles = (int)ring_out_tiles(a.out32, OT);
  const dim3 grid((a.row_tiles * a.out_tiles + 7) / 8 * 8, parts);
  hipLaunchKernelGGL((ring_tile_kernel<NX, NW, OT, TWO>), grid, dim3(512), 0, s, a);
}
template <int NX, int NW, bool TWO>
static void ring_launch(RingArgs a, hipStream_t s) {
  if (ring_few(a.n_rows, a.n_out, a.cols, NW)) {
    const dim3 grid((a.n_out + 15) / 16, a.offsets ? std::min<unsigned>(a.groups, a.n_rows) : 1);
    hipLaunchKernelGGL((ring_few_kernel<NX, NW, TWO>), grid, dim3(1024), 0, s, a);
    return;
  }
  const int parts = a.ws ? ring_call_parts(NX, NW, TWO, a.out32, a.row_tiles, a.k32 / 2, a.n_rows * a.n_out) : 1;
  if (parts == 1) a.ws = nullptr;
  const u64 mask = a.mask;
  if (a.ws) a.mask = ~u64(0);
  if constexpr (ring_wide_fits(NX, NW, TWO)) {
    if (ring_wide(NX, NW, TWO, a.out32, a.row_tiles)) ring_launch_tiles<NX, NW, 2, TWO>(a, s, parts);
    else ring_launch_tiles<NX, NW, 1, TWO>(a, s, parts);
  } else {
    ring_launch_tiles<NX, NW, 1, TWO>(a, s, parts);
  }
  a.mask = mask;
  if (a.ws)
    hipLaunchKernelGGL(ring_join_kernel, dim3((a.n_out + 511) / 512, (unsigned)std::min<size_t>(a.n_rows, 65535)), dim3(256), 0,
                       s, a, parts);
}
// digits of x and of the weights that kernels exist for (x: what the ring needs, rounded up; weights: 1..4 or all)
static int ring_digits_x(int bw) { return bw <= 32 ? 4 : bw <= 40 ? 5 : bw <= 48 ? 6 : 8; }
static int ring_digits_w(int need, int nx) { return need <= 4 && need < nx ? need : nx; }
template <int NX, bool TWO>
static bool ring_dispatch_w(int nw, const RingArgs &a, hipStream_t s) {
  if (nw == 1) ring_launch<NX, 1, TWO>(a, s);
  else if (nw == 2) ring_launch<NX, 2, TWO>(a, s);
  else if (nw == 3) ring_launch<NX, 3, TWO>(a, s);
  else if (nw == 4) ring_launch<NX, 4, TWO>(a, s);
  else if (nw == NX) ring_launch<NX, NX, TWO>(a, s);
  else return false;
  return true;
}
template <bool TWO>
static bool ring_dispatch(int nx, int nw, const RingArgs &a, hipStream_t s) {
  if (nx == 4) return ring_dispatch_w<4, TWO>(nw, a, s);
  if (nx == 5) return ring_dispatch_w<5, TWO>(nw, a, s);
  if (nx == 6) return ring_dispatch_w<6, TWO>(nw, a, s);
  return nx == 8 && ring_dispatch_w<8, TWO>(nw, a, s);
}
}  // namespace mmh

using namespace mmh;

extern "C" int mmh_ring_weights_create(const void *d_w, int elem_bytes, size_t n_groups, size_t rows, size_t cols, int ring_bw,
                                       void *stream, mmh_ring_weights **out) {
  MMH_REQUIRE(out, MMH_ERR_NULL_POINTER);
  *out = nullptr;
  MMH_REQUIRE(d_w, MMH_ERR_NULL_POINTER);
  MMH_REQUIRE(elem_bytes == 1 || elem_bytes == 2 || elem_bytes == 4 || elem_bytes == 8, MMH_ERR_INVALID_ARG);
  MMH_REQUIRE(ring_bw >= 2 && ring_bw <= 64, MMH_ERR_INVALID_ARG);
  MMH_REQUIRE(n_groups >= 1 && rows >= 1 && cols >= 1, MMH_ERR_DIM_MISMATCH);
  MMH_REQUIRE(n_groups <= kRingGroups && rows < (size_t(1) << 30) && cols < (size_t(1) << 30), MMH_ERR_OUT_BOUND);
  hipStream_t s = (hipStream_t)stream;
  hipStreamCaptureStatus cap = hipStreamCaptureStatusNone;
  (void)hipGetLastError();
  MMH_HIP(hipStreamIsCapturing(s, &cap));
  MMH_REQUIRE(cap == hipStreamCaptureStatusNone, MMH_ERR_INVALID_ARG);   // allocates and waits: not under capture
  mmh_ring_weights *h = new (std::nothrow) mmh_ring_weights;
  MMH_REQUIRE(h, MMH_ERR_MEMORY);
  h->groups = n_groups, h->rows = rows, h->cols = cols, h->bw = ring_bw;
  h->nx = ring_digits_x(ring_bw);
  h->k32 = (cols + 63) / 64 * 2, h->out32 = (rows + 31) / 32;
  const size_t frags = n_groups * h->out32 * h->k32;
  int need = 0, *d_need = nullptr;
  auto fail = [&](int code, const char *what, hipError_t e) {
    (void)hipGetLastError();
    if (d_need) (void)hipFree(d_need);
    if (h->d) (void)hipFree(h->d);
    delete h;
    set_error(std::string("mmh_ring_weights_create: ") + what + (e == hipSuccess ? "" : std::string(": ") + hipGetErrorString(e)));
    return code;
  };
  hipError_t e = hipGetDevice(&h->device);
  if (e != hipSuccess) return fail(MMH_ERR_INTERNAL, "hipGetDevice", e);
  if (frags / n_groups / h->out32 != h->k32 || frags >= (size_t(1) << 31) || n_groups * rows * cols / rows / cols != n_groups)
    return fail(MMH_ERR_OUT_BOUND, "too many weights", hipSuccess);
  e = hipMalloc((void **)&d_need, sizeof(int));
  if (e != hipSuccess) return fail(MMH_ERR_MEMORY, "hipMalloc", e);
  const size_t n = n_groups * rows * cols;
  e = hipMemcpyAsync(d_need, &need, sizeof need, hipMemcpyHostToDevice, s);
  if (e != hipSuccess) return fail(MMH_ERR_INTERNAL, "hipMemcpyAsync", e);
  if (elem_bytes == 1) ring_launch_digits<int8_t>(d_w, n, ring_bw, d_need, s);
  else if (elem_bytes == 2) ring_launch_digits<int16_t>(d_w, n, ring_bw, d_need, s);
  else if (elem_bytes == 4) ring_launch_digits<int32_t>(d_w, n, ring_bw, d_need, s);
  else ring_launch_digits<int64_t>(d_w, n, ring_bw, d_need, s);
  e = hipGetLastError();
  if (e == hipSuccess) e = hipMemcpyAsync(&need, d_need, sizeof need, hipMemcpyDeviceToHost, s);
  if (e == hipSuccess) e = hipStreamSynchronize(s);
  if (e != hipSuccess) return fail(MMH_ERR_INTERNAL, "reading the weights", e);
  h->nw = ring_digits_w(need, h->nx);
  e = hipMalloc((void **)&h->d, frags * h->nw * 1024);
  if (e != hipSuccess) return fail(MMH_ERR_MEMORY, "hipMalloc", e);
  if (elem_bytes == 1) ring_launch_layout<int8_t>(d_w, h, s);
  else if (elem_bytes == 2) ring_launch_layout<int16_t>(d_w, h, s);
  else if (elem_bytes == 4) ring_launch_layout<int32_t>(d_w, h, s);
  else ring_launch_layout<int64_t>(d_w, h, s);
  e = hipGetLastError();
  if (e == hipSuccess) e = hipStreamSynchronize(s);   // usable on any stream from here on
  if (e != hipSuccess) return fail(MMH_ERR_INTERNAL, "laying out the weights", e);
  (void)hipFree(d_need);
  *out = h;
  return MMH_OK;
}
extern "C" int mmh_ring_weights_destroy(mmh_ring_weights *w) {
  if (!w) return MMH_OK;
  DeviceScope scope(w->device);
  if (w->d) (void)hipFree(w->d);   // waits for kernels that still read it
  delete w;
  return MMH_OK;
}
extern "C" int mmh_ring_weights_info(const mmh_ring_weights *w, size_t *n_groups, size_t *rows, size_t *cols, int *ring_bw,
                                     int *digits) {
  MMH_REQUIRE(w, MMH_ERR_NULL_POINTER);
  if (n_groups) *n_groups = w->groups;
  if (rows) *rows = w->rows;
  if (cols) *cols = w->cols;
  if (ring_bw) *ring_bw = w->bw;
  if (digits) *digits = w->nw;
  return MMH_OK;
}
namespace mmh {
// row tiles of 32 rows that the groups can have: each nonempty group has at most one that is not full
static size_t ring_row_tiles(const mmh_ring_weights *w, size_t n_rows, bool offsets) {
  return offsets ? n_rows / 32 + std::min(w->groups, n_rows) : (n_rows + 31) / 32;
}
static size_t ring_ws_words(const mmh_ring_weights *w, size_t n_rows, size_t row_tiles, bool two) {
  if (w->cols < 4 || ring_few(n_rows, w->rows, w->cols, w->nw)) return 0;
  const int parts = ring_call_parts(w->nx, w->nw, two, w->out32, row_tiles, w->k32 / 2, n_rows * w->rows);
  return parts > 1 ? parts * n_rows * w->rows : 0;
}
// a dimension of a grid holds fewer than 2^32 lanes: below 2^23 workgroups of the tile kernel
static bool ring_grid_fits(const mmh_ring_weights *w, size_t n_rows, size_t row_tiles, bool two) {
  if (w->cols < 4 || ring_few(n_rows, w->rows, w->cols, w->nw)) return true;
  const int ot = ring_wide(w->nx, w->nw, two, w->out32, row_tiles) ? 2 : 1;
  return row_tiles * ring_out_tiles(w->out32, ot) + 7 < (size_t(1) << 23);
}
}  // namespace mmh
extern "C" int mmh_ring_matmul_workspace(const mmh_ring_weights *w, size_t n_rows, size_t *words) {
  MMH_REQUIRE(w && words, MMH_ERR_NULL_POINTER);
  *words = 0;   // the most of what calls with or without offsets and a second share take
  for (int i = 0; i < 4; ++i) *words = std::max(*words, ring_ws_words(w, n_rows, ring_row_tiles(w, n_rows, i & 1), i & 2));
  return MMH_OK;
}
extern "C" int mmh_ring_matmul(const mmh_ring_weights *w, const uint64_t *d_x, size_t ldx, const uint64_t *d_x1, size_t ldx1,
                               size_t n_tokens, const int64_t *d_rows, const int64_t *d_offsets, size_t n_rows,
                               const uint64_t *d_add, size_t ldadd, uint64_t *d_out, size_t ldo, int zero_rest,
                               uint64_t *d_ws, size_t ws_words, void *stream) {
  MMH_REQUIRE(w, MMH_ERR_NULL_POINTER);
  DeviceScope scope(w->device);
  if (scope.rc) MMH_FAIL(scope.rc, "cannot make the weights' device current");
  if (n_rows == 0) return MMH_OK;
  MMH_REQUIRE(d_out && d_x, MMH_ERR_NULL_POINTER);
  MMH_REQUIRE(d_offsets || w->groups == 1, MMH_ERR_NULL_POINTER);
  MMH_REQUIRE(n_tokens >= 1 && (d_rows || n_rows <= n_tokens), MMH_ERR_DIM_MISMATCH);
  MMH_REQUIRE((ldx == 0 || ldx >= w->cols) && (!d_x1 || ldx1 == 0 || ldx1 >= w->cols), MMH_ERR_DIM_MISMATCH);
  MMH_REQUIRE(ldo >= w->rows, MMH_ERR_DIM_MISMATCH);
  MMH_REQUIRE(!d_add || ldadd == 0 || ldadd >= w->rows, MMH_ERR_DIM_MISMATCH);
  // row tiles are the second dimension of a grid, which the hardware counts in 16 bits, and with the output tiles the first
  MMH_REQUIRE(n_rows <= (size_t(1) << 19), MMH_ERR_OUT_BOUND);
  MMH_REQUIRE((n_rows / 32 + w->groups + 8) * (w->out32 + 8) < (size_t(1) << 31), MMH_ERR_OUT_BOUND);
  const size_t row_tiles = ring_row_tiles(w, n_rows, d_offsets != nullptr);
  MMH_REQUIRE(ring_grid_fits(w, n_rows, row_tiles, d_x1 != nullptr), MMH_ERR_OUT_BOUND);
  RingArgs a;
  a.w = w->d, a.x = d_x, a.x1 = d_x1, a.add = d_add, a.rows = d_rows, a.offsets = d_offsets, a.out = d_out;
  a.ldx = ldx, a.ldx1 = ldx1, a.ldadd = ldadd, a.ldo = ldo, a.n_tokens = n_tokens, a.n_rows = n_rows;
  a.ws = nullptr, a.out_tiles = 0, a.zero_rest = zero_rest;
  a.groups = (int)w->groups, a.cols = (int)w->cols, a.n_out = (int)w->rows, a.k32 = (int)w->k32, a.out32 = (int)w->out32;
  a.mask = w->bw >= 64 ? ~u64(0) : (u64(1) << w->bw) - 1;
  a.row_tiles = (int)row_tiles;
  a.ws = d_ws && ws_words >= ring_ws_words(w, n_rows, a.row_tiles, d_x1 != nullptr) ? d_ws : nullptr;
  hipStream_t s = (hipStream_t)stream;
  bool ok = w->cols < 4;
  if (ok) hipLaunchKernelGGL(ring_narrow_kernel, dim3((a.n_out + 255) / 256, a.row_tiles), dim3(256), 0, s, a, w->nw);
  else ok = d_x1 ? ring_dispatch<true>(w->nx, w->nw, a, s) : ring_dispatch<false>(w->nx, w->nw, a, s);
  MMH_REQUIRE(ok, MMH_ERR_INTERNAL);
  MMH_HIP(hipGetLastError());
  return MMH_OK;
}
