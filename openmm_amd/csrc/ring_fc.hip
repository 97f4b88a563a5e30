// Products of secret shares with cleartext weights in Z_{2^l}, grouped by expert:
//   out[r][o] = add[r][o] + sum_k (x[t][k] + x1[t][k]) * w[g][o][k]  mod 2^l,   t = rows[r], offsets[g] <= r < offsets[g+1]
//
// Mathematics.  Both operands are written in balanced base-256 digits, x = sum x_i 256^i and w = sum w_j 256^j with
// digits in [-128, 127]: with C = 0x80...80, the digits of v are the bytes of (v + C) ^ C (adding C makes every byte
// digit + 128, the exclusive or takes the 128 off again as a signed byte).  l bits need nx = ceil(l/8) digits of x (what
// lies above is a multiple of 2^l), a weight as many as its size asks for, found when the weights are laid out.  The
// product modulo 2^l is then sum over s < nx of 256^s * sum_{i+j=s} x_i w_j, every inner sum an exact i8 x i8 -> i32
// matrix product (v_mfma_i32_16x16x64_i8), nx accumulators per output.  |x_i w_j| <= 2^14 and at most nw products share
// an accumulator, so up to (2^17 - 1) / nw terms of k cannot overflow; longer k is added up in 64-bit pieces.
// Everything is exact: the result does not depend on the order of the sums.
#include <algorithm>
#include <new>

#include "common.hpp"
#include "convert_device.hpp"

struct mmh_ring_weights {
  int device = 0;
  size_t groups = 0, rows = 0, cols = 0;
  int bw = 0, nx = 0, nw = 0;   // nw: digits stored per weight (a width the product kernels exist for)
  size_t k64 = 0, out16 = 0;
  int8_t *d = nullptr;          // [group][out16][k64][digit][4][16 outputs][16 columns]: 1 KiB matrix-core fragments
};

namespace mmh {
typedef int v4i __attribute__((ext_vector_type(4)));

struct RingArgs {
  const int8_t *w;
  const u64 *x, *x1, *add;
  const int64_t *rows, *offsets;
  u64 *out;
  size_t ldx, ldx1, ldadd, ldo, n_tokens, n_rows;
  int groups, cols, n_out, k64, out16;
  u64 mask;
  int vec_x, vec_out;   // 16-byte accesses are aligned
};

// The rows of row tile `tile` (BM rows, tiles do not cross groups).  Every wave finds it by itself: 64 groups at a time,
// a prefix sum of their tile counts.  Offsets are clamped to [0, n_rows], so nothing they hold leads out of bounds.
template <int BM>
__device__ __forceinline__ bool ring_find_tile(const RingArgs &a, u32 tile, int &g, size_t &lo, size_t &hi) {
  if (!a.offsets) {
    g = 0, lo = (size_t)tile * BM;
    hi = lo + BM < a.n_rows ? lo + BM : a.n_rows;
    return lo < a.n_rows;
  }
  const int lane = threadIdx.x & 63;
  u32 before = 0;
  for (int g0 = 0; g0 < a.groups; g0 += 64) {
    long long s = 0, e = 0;
    if (g0 + lane < a.groups) {
      const long long n = (long long)a.n_rows;
      s = a.offsets[g0 + lane], e = a.offsets[g0 + lane + 1];
      s = s < 0 ? 0 : s > n ? n : s;
      e = e < s ? s : e > n ? n : e;
    }
    const u32 tiles = (u32)((e - s + BM - 1) / BM);
    u32 sum = tiles;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const u32 t = __shfl_up(sum, d);
      if (lane >= d) sum += t;
    }
    const unsigned long long past = __ballot(before + sum > tile);
    if (past) {
      const int src = __ffsll(past) - 1;
      const u32 first = before + (u32)__shfl((int)(sum - tiles), src);
      lo = (size_t)__shfl(s, src) + (size_t)(tile - first) * BM;
      const size_t end = (size_t)__shfl(e, src);
      hi = lo + BM < end ? lo + BM : end;
      g = g0 + src;
      return true;
    }
    before += (u32)__shfl((int)sum, 63);
  }
  return false;
}

// the row of x that row r reads, or -1 (an index outside [0, n_tokens) reads as a row of zeros)
__device__ __forceinline__ long long ring_token(const RingArgs &a, size_t r) {
  const long long t = a.rows ? a.rows[r] : (long long)r;
  return t >= 0 && t < (long long)a.n_tokens ? t : -1;
}

// four words of a row from column k on (zeros past the end), plus the second share's
__device__ __forceinline__ void ring_load4(const u64 *p, int k, int cols, int vec, u64 (&v)[4]) {
  if (vec && k + 4 <= cols) {
    const ulonglong2 t = *reinterpret_cast<const ulonglong2 *>(p + k), u = *reinterpret_cast<const ulonglong2 *>(p + k + 2);
    v[0] = t.x, v[1] = t.y, v[2] = u.x, v[3] = u.y;
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = k + e < cols ? p[k + e] : 0;
  }
}
// bytes e[0..3].b -> one dword per byte place: a 4 x 4 byte transposition
__device__ __forceinline__ void transpose4(u32 e0, u32 e1, u32 e2, u32 e3, u32 (&d)[4]) {
  const u32 l0 = __builtin_amdgcn_perm(e1, e0, 0x05010400), h0 = __builtin_amdgcn_perm(e1, e0, 0x07030602);
  const u32 l1 = __builtin_amdgcn_perm(e3, e2, 0x05010400), h1 = __builtin_amdgcn_perm(e3, e2, 0x07030602);
  d[0] = __builtin_amdgcn_perm(l1, l0, 0x05040100), d[1] = __builtin_amdgcn_perm(l1, l0, 0x07060302);
  d[2] = __builtin_amdgcn_perm(h1, h0, 0x05040100), d[3] = __builtin_amdgcn_perm(h1, h0, 0x07060302);
}
// digits of four words: dig[i] holds digit i of each
template <int NX>
__device__ __forceinline__ void ring_digits4(const u64 (&v)[4], u32 (&dig)[8]) {
  constexpr u64 C = 0x8080808080808080ull;
  u64 t[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) t[e] = v[e] + C;
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

// Few rows: one workgroup per 16 rows x 16*OT outputs, its WK waves split k and join their 64-bit sums through LDS.
// Bound: the weights' bytes.  A lane reads the 16 words of its fragment itself and cuts them to digits in registers, so
// the loop has no LDS access and no barrier.
template <int NX, int NW, int OT, int WK>
__global__ __launch_bounds__(64 * WK) void ring_rows_kernel(RingArgs a) {
  __shared__ u64 part[WK][OT][16][17];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  int g;
  size_t lo, hi;
  if (!ring_find_tile<16>(a, blockIdx.y, g, lo, hi)) return;
  const int ot0 = (int)blockIdx.x * OT, r = lane & 15, kq = lane >> 4;
  const long long t = lo + r < hi ? ring_token(a, lo + r) : -1;
  const u64 *px = t < 0 ? nullptr : a.x + (size_t)t * a.ldx;
  const u64 *px1 = t < 0 || !a.x1 ? nullptr : a.x1 + (size_t)t * a.ldx1;
  constexpr int kFlush = 131071 / NW / 64;   // chunks whose sums fit 32 bits
  u64 total[OT][4] = {};
  v4i acc[OT][NX];
#pragma unroll
  for (int o = 0; o < OT; ++o)
#pragma unroll
    for (int s = 0; s < NX; ++s) acc[o][s] = v4i{0, 0, 0, 0};
  auto fold = [&] {
#pragma unroll
    for (int o = 0; o < OT; ++o) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        u64 v = 0;
#pragma unroll
        for (int s = NX - 1; s >= 0; --s) v = (v << 8) + (u64)(long long)acc[o][s][e];
        total[o][e] += v;
      }
#pragma unroll
      for (int s = 0; s < NX; ++s) acc[o][s] = v4i{0, 0, 0, 0};
    }
  };
  int since = 0;
  for (int c = wave; c < a.k64; c += WK) {
    v4i w[OT][NW];
#pragma unroll
    for (int o = 0; o < OT; ++o) {
      const int ot = ot0 + o < a.out16 ? ot0 + o : a.out16 - 1;
      const int8_t *p = a.w + (((size_t)g * a.out16 + ot) * a.k64 + c) * (NW * 1024) + lane * 16;
#pragma unroll
      for (int j = 0; j < NW; ++j) w[o][j] = *reinterpret_cast<const v4i *>(p + j * 1024);
    }
    u64 v[4][4] = {};
    if (px) {
      const int k = c * 64 + kq * 16;
#pragma unroll
      for (int e = 0; e < 4; ++e) ring_load4(px, k + 4 * e, a.cols, a.vec_x, v[e]);
      if (px1) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          u64 u[4];
          ring_load4(px1, k + 4 * e, a.cols, a.vec_x, u);
#pragma unroll
          for (int i = 0; i < 4; ++i) v[e][i] += u[i];
        }
      }
    }
    v4i x[8];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      u32 dig[8];
      ring_digits4<NX>(v[e], dig);
#pragma unroll
      for (int i = 0; i < NX; ++i) x[i][e] = (int)dig[i];
    }
#pragma unroll
    for (int o = 0; o < OT; ++o)
#pragma unroll
      for (int j = 0; j < NW; ++j)
#pragma unroll
        for (int i = 0; i < NX; ++i)
          if (i + j < NX) acc[o][i + j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[o][j], x[i], acc[o][i + j], 0, 0, 0);
    if (++since == kFlush) fold(), since = 0;
  }
  fold();
  // a lane holds outputs 4*(lane/16) .. +3 of row lane%16
#pragma unroll
  for (int o = 0; o < OT; ++o)
#pragma unroll
    for (int e = 0; e < 4; ++e) part[wave][o][r][kq * 4 + e] = total[o][e];
  __syncthreads();
  for (int i = (int)threadIdx.x; i < OT * 256; i += 64 * WK) {
    const int col = i & 15, o = (i >> 4) % OT, row = i / (16 * OT);
    const int n = (ot0 + o) * 16 + col;
    if (lo + row >= hi || n >= a.n_out) continue;
    u64 v = a.add ? a.add[(lo + row) * a.ldadd + n] : 0;
#pragma unroll
    for (int w = 0; w < WK; ++w) v += part[w][o][row][col];
    a.out[(lo + row) * a.ldo + n] = v & a.mask;
  }
}

// Many rows: a workgroup of WR x WO waves computes 16*RT*WR rows x 16*OT*WO outputs.  The rows' digits of one 64-column
// step are cut once per workgroup into LDS (two buffers, one barrier per step); the weights' fragments come straight from
// L2 in the order they were laid out in.
template <int NX, int NW, int RT, int OT, int WR, int WO>
__global__ __launch_bounds__(64 * WR * WO) void ring_tile_kernel(RingArgs a) {
  constexpr int BM = 16 * RT * WR, W = WR * WO, kBlocks = BM / 16 * 4, kPer = (kBlocks + W - 1) / W;
  static_assert(kBlocks % W == 0, "every wave cuts the same number of 16 x 16 blocks");
  __shared__ uint4 xs[2][BM / 16][NX][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  int g;
  size_t lo, hi;
  if (!ring_find_tile<BM>(a, blockIdx.y, g, lo, hi)) return;
  const int wr = wave % WR, wo = wave / WR, ot0 = ((int)blockIdx.x * WO + wo) * OT;
  const int r = lane & 15, sub = lane >> 4;
  // block b of the step: row tile b / 4, columns 16 * (b % 4) ..; a lane cuts four words of one row
  const u64 *px[kPer], *px1[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const size_t row = lo + (size_t)((i * W + wave) / 4) * 16 + r;
    const long long t = row < hi ? ring_token(a, row) : -1;
    px[i] = t < 0 ? nullptr : a.x + (size_t)t * a.ldx;
    px1[i] = t < 0 || !a.x1 ? nullptr : a.x1 + (size_t)t * a.ldx1;
  }
  u64 xv[kPer][4], xu[kPer][4];
  auto load_x = [&](int c) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int k = c * 64 + ((i * W + wave) & 3) * 16 + sub * 4;
#pragma unroll
      for (int e = 0; e < 4; ++e) xv[i][e] = 0, xu[i][e] = 0;
      if (px[i]) ring_load4(px[i], k, a.cols, a.vec_x, xv[i]);
      if (px1[i]) ring_load4(px1[i], k, a.cols, a.vec_x, xu[i]);
    }
  };
  auto store_x = [&](int buf) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int b = i * W + wave;
      u64 v[4];
      u32 dig[8];
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = xv[i][e] + xu[i][e];
      ring_digits4<NX>(v, dig);
#pragma unroll
      for (int d = 0; d < NX; ++d) reinterpret_cast<u32 *>(&xs[buf][b >> 2][d][(b & 3) * 16 + r])[sub] = dig[d];
    }
  };
  const int8_t *pw[OT];
#pragma unroll
  for (int o = 0; o < OT; ++o) {
    const int ot = ot0 + o < a.out16 ? ot0 + o : a.out16 - 1;
    pw[o] = a.w + ((size_t)g * a.out16 + ot) * a.k64 * (NW * 1024) + lane * 16;
  }
  v4i wn[OT][NW], wc[OT][NW], acc[RT][OT][NX];
  auto load_w = [&](int c) {
#pragma unroll
    for (int o = 0; o < OT; ++o)
#pragma unroll
      for (int j = 0; j < NW; ++j) wn[o][j] = *reinterpret_cast<const v4i *>(pw[o] + (size_t)c * (NW * 1024) + j * 1024);
  };
  constexpr int kFlush = 131071 / NW / 64;
  for (int c0 = 0; c0 < a.k64; c0 += kFlush) {
    const int c1 = c0 + kFlush < a.k64 ? c0 + kFlush : a.k64;
#pragma unroll
    for (int m = 0; m < RT; ++m)
#pragma unroll
      for (int o = 0; o < OT; ++o)
#pragma unroll
        for (int s = 0; s < NX; ++s) acc[m][o][s] = v4i{0, 0, 0, 0};
    load_x(c0);
    load_w(c0);
    store_x(0);
    __syncthreads();
    int buf = 0;
    for (int c = c0; c < c1; ++c) {
#pragma unroll
      for (int o = 0; o < OT; ++o)
#pragma unroll
        for (int j = 0; j < NW; ++j) wc[o][j] = wn[o][j];
      const bool more = c + 1 < c1;
      if (more) load_x(c + 1), load_w(c + 1);
#pragma unroll
      for (int m = 0; m < RT; ++m)
#pragma unroll
        for (int i = 0; i < NX; ++i) {
          const uint4 t = xs[buf][wr * RT + m][i][lane];
          const v4i x = v4i{(int)t.x, (int)t.y, (int)t.z, (int)t.w};
#pragma unroll
          for (int o = 0; o < OT; ++o)
#pragma unroll
            for (int j = 0; j < NW; ++j)
              if (i + j < NX)
                acc[m][o][i + j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wc[o][j], x, acc[m][o][i + j], 0, 0, 0);
        }
      if (more) store_x(buf ^ 1);
      __syncthreads();
      buf ^= 1;
    }
    // a lane holds outputs 4*(lane/16) .. +3 of row lane%16 of each tile
#pragma unroll
    for (int m = 0; m < RT; ++m) {
      const size_t row = lo + (size_t)(wr * RT + m) * 16 + r;
      if (row >= hi) continue;
      const u64 *base = c0 ? a.out + row * a.ldo : a.add ? a.add + row * a.ldadd : nullptr;
#pragma unroll
      for (int o = 0; o < OT; ++o) {
        const int n = (ot0 + o) * 16 + sub * 4;
        u64 v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          v[e] = 0;
#pragma unroll
          for (int s = NX - 1; s >= 0; --s) v[e] = (v[e] << 8) + (u64)(long long)acc[m][o][s][e];
          if (base && n + e < a.n_out) v[e] += base[n + e];
          v[e] &= a.mask;
        }
        u64 *p = a.out + row * a.ldo + n;
        if (a.vec_out && n + 4 <= a.n_out) {
          reinterpret_cast<ulonglong2 *>(p)[0] = make_ulonglong2(v[0], v[1]);
          reinterpret_cast<ulonglong2 *>(p)[1] = make_ulonglong2(v[2], v[3]);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (n + e < a.n_out) p[e] = v[e];
        }
      }
    }
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
  if ((threadIdx.x & 63) == 0) atomicMax(need, m);
}
template <typename T>
__global__ __launch_bounds__(256) void ring_weight_layout_kernel(const T *__restrict__ w, size_t rows, size_t cols, int bw,
                                                                 size_t out16, size_t k64, int nw, size_t n_units,
                                                                 int8_t *__restrict__ out) {
  const size_t u = (size_t)blockIdx.x * 256 + threadIdx.x;   // (group, out16, k64, quarter, output): 16 columns of a row
  if (u >= n_units) return;
  const size_t frag = u >> 6, c = frag % k64, ot = frag / k64 % out16, g = frag / k64 / out16;
  const size_t o = ot * 16 + (u & 15), k = c * 64 + (u >> 4 & 3) * 16;
  u64 t[16];
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    const bool in = o < rows && k + e < cols;
    const u64 C = 0x8080808080808080ull;
    t[e] = ((u64)(in ? ring_weight(w, (g * rows + o) * cols + k + e, bw) : 0) + C) ^ C;
  }
  for (int j = 0; j < nw; ++j) {
    u32 d[4] = {0, 0, 0, 0};
#pragma unroll
    for (int e = 0; e < 16; ++e) d[e >> 2] |= (u32)(t[e] >> (8 * j) & 0xff) << (8 * (e & 3));
    *reinterpret_cast<uint4 *>(out + (frag * nw + j) * 1024 + (u & 63) * 16) = make_uint4(d[0], d[1], d[2], d[3]);
  }
}

template <typename T>
static void ring_launch_digits(const void *w, size_t n, int bw, int *need, hipStream_t s) {
  hipLaunchKernelGGL(ring_weight_digits_kernel<T>, dim3((unsigned)std::min<size_t>((n + 255) / 256, 4096)), dim3(256), 0, s,
                     (const T *)w, n, bw, need);
}
template <typename T>
static void ring_launch_layout(const void *w, const mmh_ring_weights *h, hipStream_t s) {
  const size_t units = h->groups * h->out16 * h->k64 * 64;
  hipLaunchKernelGGL(ring_weight_layout_kernel<T>, dim3((unsigned)((units + 255) / 256)), dim3(256), 0, s, (const T *)w,
                     h->rows, h->cols, h->bw, h->out16, h->k64, h->nw, units, h->d);
}

template <int NX, int NW>
static void ring_launch(const RingArgs &a, hipStream_t s) {
  // row tiles of BM rows that the groups can have: each nonempty group has at most one that is not full
  auto tiles = [&](size_t bm) { return a.offsets ? a.n_rows / bm + std::min<size_t>((size_t)a.groups, a.n_rows) : (a.n_rows + bm - 1) / bm; };
  if (a.n_rows <= 16 * (size_t)a.groups) {
    constexpr int OT = 1, WK = 8;
    hipLaunchKernelGGL((ring_rows_kernel<NX, NW, OT, WK>), dim3((a.out16 + OT - 1) / OT, (unsigned)tiles(16)), dim3(64 * WK),
                       0, s, a);
  } else {
    constexpr int RT = 2, OT = 2, WR = 1, WO = 4;
    hipLaunchKernelGGL((ring_tile_kernel<NX, NW, RT, OT, WR, WO>),
                       dim3((a.out16 + OT * WO - 1) / (OT * WO), (unsigned)tiles(16 * RT * WR)), dim3(64 * WR * WO), 0, s, a);
  }
}
// digits of x and of the weights that kernels exist for (x: what the ring needs, rounded up; weights: 1..4 or all)
static int ring_digits_x(int bw) { return bw <= 32 ? 4 : bw <= 40 ? 5 : bw <= 48 ? 6 : 8; }
static int ring_digits_w(int need, int nx) { return need <= 4 && need < nx ? need : nx; }
template <int NX>
static bool ring_dispatch_w(int nw, const RingArgs &a, hipStream_t s) {
  if (nw == 1) ring_launch<NX, 1>(a, s);
  else if (nw == 2) ring_launch<NX, 2>(a, s);
  else if (nw == 3) ring_launch<NX, 3>(a, s);
  else if (nw == 4) ring_launch<NX, 4>(a, s);
  else if (nw == NX) ring_launch<NX, NX>(a, s);
  else return false;
  return true;
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
  MMH_REQUIRE(n_groups < (size_t(1) << 24) && rows < (size_t(1) << 30) && cols < (size_t(1) << 30), MMH_ERR_OUT_BOUND);
  hipStream_t s = (hipStream_t)stream;
  hipStreamCaptureStatus cap = hipStreamCaptureStatusNone;
  (void)hipGetLastError();
  MMH_HIP(hipStreamIsCapturing(s, &cap));
  MMH_REQUIRE(cap == hipStreamCaptureStatusNone, MMH_ERR_INVALID_ARG);   // allocates and waits: not under capture
  mmh_ring_weights *h = new (std::nothrow) mmh_ring_weights;
  MMH_REQUIRE(h, MMH_ERR_MEMORY);
  h->groups = n_groups, h->rows = rows, h->cols = cols, h->bw = ring_bw;
  h->nx = ring_digits_x(ring_bw);
  h->k64 = (cols + 63) / 64, h->out16 = (rows + 15) / 16;
  const size_t frags = n_groups * h->out16 * h->k64;
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
  if (frags / n_groups / h->out16 != h->k64 || frags >= (size_t(1) << 31) || n_groups * rows * cols / rows / cols != n_groups)
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
extern "C" int mmh_ring_matmul(const mmh_ring_weights *w, const uint64_t *d_x, size_t ldx, const uint64_t *d_x1, size_t ldx1,
                               size_t n_tokens, const int64_t *d_rows, const int64_t *d_offsets, size_t n_rows,
                               const uint64_t *d_add, size_t ldadd, uint64_t *d_out, size_t ldo, void *stream) {
  MMH_REQUIRE(w, MMH_ERR_NULL_POINTER);
  DeviceScope scope(w->device);
  if (scope.rc) MMH_FAIL(scope.rc, "cannot make the weights' device current");
  if (n_rows == 0) return MMH_OK;
  MMH_REQUIRE(d_out && (d_x || n_tokens == 0), MMH_ERR_NULL_POINTER);
  MMH_REQUIRE(d_offsets || w->groups == 1, MMH_ERR_NULL_POINTER);
  MMH_REQUIRE(d_rows || n_rows <= n_tokens, MMH_ERR_DIM_MISMATCH);
  MMH_REQUIRE(ldx >= w->cols && (!d_x1 || ldx1 >= w->cols) && ldo >= w->rows, MMH_ERR_DIM_MISMATCH);
  MMH_REQUIRE(!d_add || ldadd == 0 || ldadd >= w->rows, MMH_ERR_DIM_MISMATCH);
  // row tiles are the second dimension of the grid, which the hardware counts in 16 bits
  MMH_REQUIRE(n_rows <= (size_t(1) << 19) && w->groups <= 32767, MMH_ERR_OUT_BOUND);
  RingArgs a;
  a.w = w->d, a.x = d_x, a.x1 = d_x1, a.add = d_add, a.rows = d_rows, a.offsets = d_offsets, a.out = d_out;
  a.ldx = ldx, a.ldx1 = ldx1, a.ldadd = ldadd, a.ldo = ldo, a.n_tokens = n_tokens, a.n_rows = n_rows;
  a.groups = (int)w->groups, a.cols = (int)w->cols, a.n_out = (int)w->rows, a.k64 = (int)w->k64, a.out16 = (int)w->out16;
  a.mask = w->bw >= 64 ? ~u64(0) : (u64(1) << w->bw) - 1;
  auto aligned = [](const void *p, size_t ld) { return ((uintptr_t)p & 15) == 0 && (ld & 1) == 0; };
  a.vec_x = aligned(d_x, ldx) && (!d_x1 || aligned(d_x1, ldx1));
  a.vec_out = aligned(d_out, ldo);
  hipStream_t s = (hipStream_t)stream;
  bool ok = false;
  if (w->nx == 4) ok = ring_dispatch_w<4>(w->nw, a, s);
  else if (w->nx == 5) ok = ring_dispatch_w<5>(w->nw, a, s);
  else if (w->nx == 6) ok = ring_dispatch_w<6>(w->nw, a, s);
  else if (w->nx == 8) ok = ring_dispatch_w<8>(w->nw, a, s);
  MMH_REQUIRE(ok, MMH_ERR_INTERNAL);
  MMH_HIP(hipGetLastError());
  return MMH_OK;
}
