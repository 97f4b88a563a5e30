// Rotary positions on secret shares in Z_{2^l}: the turn's coefficients are public, so each party turns its own share.
//   (a, b) -> (a c - b s, b c + a s) mod 2^l,   c = round(A cos(2 pi p f / 2^64)), s = round(A sin(...)), A = amplitude 2^frac
// p is the token's position, f the pair's phase step as a 64-bit fraction of a turn: p f mod 2^64 is the phase exactly, at
// any position, because whole turns are multiples of 2^64.  The parties' coefficients have to agree to the last bit (a
// share times c1 - c0 is noise as large as the ring), so they are computed by a fixed sequence of IEEE double operations
// (no table, no library function): the phase is reduced to an eighth of a turn around a quadrant in integers, sine and
// cosine there are their Taylor sums (terms to x^15 and x^16: the first one left out is below 2^-53), rounded to the
// nearest integer, ties to even.  Elements beyond the turned part are multiplied by 2^frac, so that one truncation by
// frac (or by frac and the scale of the product before) serves the whole head.
//
// Bound: HBM, 8 B read and 8 B written per element (16 with the comparison's operand).  A workgroup computes the coefficients of
// its tokens once, into LDS, and applies them to all their heads; a lane takes two neighbouring words per access where rows are
// 16-byte aligned.  Calls back to back in a graph: 16384 tokens x 40 heads x 128 252 us = 5.3 TB/s (torch's copy of as many
// bytes: 4.7); one token 2.4 us, of which a launch is 1.6 (a kernel trace reads 3.1).  Out of the last-level cache, which holds
// all of these: 2048 tokens 27 us = 6.3 TB/s, 6000 x 13 x 42 11.2 us = 4.7, words at 8 modulo 16, 6000 x 13 x 43, 12.8 us = 4.2.
#include <algorithm>

#include "common.hpp"
#include "convert_device.hpp"

namespace mmh {
struct RotaryArgs {
  const u64 *x, *phase;
  const int64_t *pos;
  u64 *out, *cmp;
  size_t xs_token, xs_head, os_token, os_head, n_tokens;   // cmp is laid out like out
  int heads, dim, half;        // half = turned pairs per head
  int frac, heads_per_block, tokens_per_block;
  double scale;
  u64 mask, offset, cmp_flip;  // out = (turned + offset) & mask, cmp = out ^ cmp_flip (all ones below l: mask - out)
};

__device__ __forceinline__ int2 rotary_coefficients(u64 turn, double scale) {
  const u64 quad = (turn + (u64(1) << 61)) >> 62;
  const double x = (double)(long long)(turn - (quad << 62)) * 0x1.921fb54442d18p-62;   // 2 pi / 2^64
  const double z = x * x;
  double s = -1.0 / 1307674368000.0, c = 1.0 / 20922789888000.0;
  s = __builtin_fma(s, z, 1.0 / 6227020800.0), c = __builtin_fma(c, z, -1.0 / 87178291200.0);
  s = __builtin_fma(s, z, -1.0 / 39916800.0), c = __builtin_fma(c, z, 1.0 / 479001600.0);
  s = __builtin_fma(s, z, 1.0 / 362880.0), c = __builtin_fma(c, z, -1.0 / 3628800.0);
  s = __builtin_fma(s, z, -1.0 / 5040.0), c = __builtin_fma(c, z, 1.0 / 40320.0);
  s = __builtin_fma(s, z, 1.0 / 120.0), c = __builtin_fma(c, z, -1.0 / 720.0);
  s = __builtin_fma(s, z, -1.0 / 6.0), c = __builtin_fma(c, z, 1.0 / 24.0);
  const double xz = x * z;
  s = __builtin_fma(xz, s, x), c = __builtin_fma(c, z, -0.5);
  c = __builtin_fma(c, z, 1.0);
  const int is = (int)__builtin_rint(s * scale), ic = (int)__builtin_rint(c * scale);
  const int q = (int)(quad & 3);
  const int a = q & 1 ? is : ic, b = q & 1 ? ic : is;     // quadrant 1: (-s, c), 2: (-c, -s), 3: (s, -c)
  return make_int2(q == 1 || q == 2 ? -a : a, q >= 2 ? -b : b);
}

// V = 2: two neighbouring words per access.  INTER: pairs are neighbours (2i, 2i+1), else (i, i + half).
template <int V, bool INTER>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryArgs a) {
  extern __shared__ int2 coef[];   // [tokens_per_block][half]
  const size_t t0 = (size_t)blockIdx.x * a.tokens_per_block;
  const int nt = (int)(a.n_tokens - t0 < (size_t)a.tokens_per_block ? a.n_tokens - t0 : (size_t)a.tokens_per_block);
  const int h0 = (int)blockIdx.y * a.heads_per_block, nh = a.heads - h0 < a.heads_per_block ? a.heads - h0 : a.heads_per_block;
  for (int i = (int)threadIdx.x; i < nt * a.half; i += 256) {
    const int t = i / a.half, f = i - t * a.half;
    coef[i] = rotary_coefficients((u64)a.pos[t0 + t] * a.phase[f], a.scale);
  }
  __syncthreads();
  // units of a head: the turned pairs (V of them in the split layout), then the V-word pieces that are only scaled
  const int turned = INTER ? a.half : a.half / V, rest = (a.dim - 2 * a.half) / V, units = turned + rest;
  const int rows = nt * nh, dq = 256 / units, dr = 256 - dq * units;
  int row = (int)threadIdx.x / units, u = (int)threadIdx.x - row * units;
  for (; row < rows;) {
    const int t = row / nh, h = h0 + row - t * nh;
    const u64 *px = a.x + (t0 + t) * a.xs_token + (size_t)h * a.xs_head;
    const size_t at = (t0 + t) * a.os_token + (size_t)h * a.os_head;
    auto put = [&](int k, u64 v0, u64 v1) {
      v0 = (v0 + a.offset) & a.mask, v1 = (v1 + a.offset) & a.mask;
      if (V == 2) *reinterpret_cast<ulonglong2 *>(a.out + at + k) = make_ulonglong2(v0, v1);
      else a.out[at + k] = v0;
      if (!a.cmp) return;
      if (V == 2) *reinterpret_cast<ulonglong2 *>(a.cmp + at + k) = make_ulonglong2(v0 ^ a.cmp_flip, v1 ^ a.cmp_flip);
      else a.cmp[at + k] = v0 ^ a.cmp_flip;
    };
    auto get = [&](int k, u64 (&v)[2]) {
      if (V == 2) {
        const ulonglong2 w = *reinterpret_cast<const ulonglong2 *>(px + k);
        v[0] = w.x, v[1] = w.y;
      } else {
        v[0] = px[k], v[1] = 0;
      }
    };
    u64 p[2], q[2];
    if (u >= turned) {
      const int k = 2 * a.half + (u - turned) * V;
      get(k, p);
      put(k, p[0] << a.frac, p[1] << a.frac);
    } else if (INTER) {
      const int2 c = coef[t * a.half + u];
      const u64 cc = (u64)(long long)c.x, ss = (u64)(long long)c.y;
      if (V == 2) {
        get(2 * u, p);
        put(2 * u, p[0] * cc - p[1] * ss, p[1] * cc + p[0] * ss);
      } else {
        get(2 * u, p);
        get(2 * u + 1, q);
        put(2 * u, p[0] * cc - q[0] * ss, 0);
        put(2 * u + 1, q[0] * cc + p[0] * ss, 0);
      }
    } else {
      get(u * V, p);
      get(a.half + u * V, q);
      u64 o[2] = {0, 0}, w[2] = {0, 0};
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const int2 c = coef[t * a.half + u * V + e];
        const u64 cc = (u64)(long long)c.x, ss = (u64)(long long)c.y;
        o[e] = p[e] * cc - q[e] * ss, w[e] = q[e] * cc + p[e] * ss;
      }
      put(u * V, o[0], o[1]);
      put(a.half + u * V, w[0], w[1]);
    }
    row += dq, u += dr;
    if (u >= units) u -= units, ++row;
  }
}

static u64 bw_mask_host(int bw) { return bw >= 64 ? ~u64(0) : (u64(1) << bw) - 1; }

// Tokens and heads of a workgroup.  Small heads: several tokens, up to 4096 words and 2048 pairs of coefficients (16384 x 1 x 16:
// 3.0 us, a token each 12.9).  Few tokens: the heads over several workgroups, each of 512 words or more, until there are 512 of
// them (1 x 40 x 128: 2.4 us, in one 3.8).
static void rotary_blocks(size_t tokens, size_t heads, size_t dim, int half, int &per_tokens, int &per_heads) {
  const size_t words = heads * dim;
  size_t t = std::min<size_t>(4096 / words, 2048 / std::max(half, 1));
  t = std::max<size_t>(1, std::min(t, tokens / 512));
  size_t split = std::max<size_t>(1, std::min({512 / ((tokens + t - 1) / t), words / 512, heads}));
  per_tokens = (int)t, per_heads = (int)((heads + split - 1) / split);
}

static int rotary_call(const uint64_t *d_x, size_t xs_token, size_t xs_head, size_t n_tokens, size_t n_heads, size_t head_dim,
                       const int64_t *d_pos, const uint64_t *d_phase, size_t rot_dim, int interleaved, double amplitude,
                       int frac_bits, int bw, u64 offset, u64 cmp_flip, uint64_t *d_out, uint64_t *d_cmp, size_t os_token,
                       size_t os_head, void *stream) {
  MMH_REQUIRE(bw >= 2 && bw <= 64 && frac_bits >= 0 && frac_bits <= 24, MMH_ERR_INVALID_ARG);
  MMH_REQUIRE(amplitude > 0 && amplitude <= 16, MMH_ERR_INVALID_ARG);   // also false for a NaN
  MMH_REQUIRE(head_dim >= 1 && rot_dim % 2 == 0 && rot_dim <= head_dim, MMH_ERR_DIM_MISMATCH);
  MMH_REQUIRE(head_dim <= 4096 && n_heads <= (size_t(1) << 16) && n_tokens < (size_t(1) << 31), MMH_ERR_OUT_BOUND);
  if (n_tokens == 0 || n_heads == 0) return MMH_OK;
  MMH_REQUIRE(d_x && d_out && d_pos && (d_phase || rot_dim == 0), MMH_ERR_NULL_POINTER);
  // rows of the result must not overlap: of the two strides the smaller holds a row, the larger all rows at the smaller
  const size_t far = std::max(n_tokens > 1 ? os_token : 0, n_heads > 1 ? os_head : 0);
  const bool tokens_far = n_tokens > 1 && os_token == far;
  const size_t near = tokens_far ? os_head : os_token, n_near = tokens_far ? n_heads : n_tokens;
  MMH_REQUIRE((n_near == 1 || near >= head_dim) && (far == 0 || far >= near * (n_near - 1) + head_dim) &&
              (n_heads * n_tokens == 1 || far > 0), MMH_ERR_DIM_MISMATCH);
  RotaryArgs a;
  a.x = d_x, a.phase = d_phase, a.pos = d_pos, a.out = d_out, a.cmp = d_cmp;
  a.xs_token = xs_token, a.xs_head = xs_head, a.os_token = os_token, a.os_head = os_head, a.n_tokens = n_tokens;
  a.heads = (int)n_heads, a.dim = (int)head_dim, a.half = (int)rot_dim / 2, a.frac = frac_bits;
  a.scale = amplitude * (double)(u64(1) << frac_bits);
  a.mask = bw_mask_host(bw), a.offset = offset, a.cmp_flip = cmp_flip;
  rotary_blocks(n_tokens, n_heads, head_dim, a.half, a.tokens_per_block, a.heads_per_block);
  // a dimension of a grid holds fewer than 2^32 lanes
  MMH_REQUIRE((n_tokens + a.tokens_per_block - 1) / a.tokens_per_block < (size_t(1) << 24), MMH_ERR_OUT_BOUND);
  const dim3 grid((unsigned)((n_tokens + a.tokens_per_block - 1) / a.tokens_per_block),
                  (unsigned)((n_heads + a.heads_per_block - 1) / a.heads_per_block));
  const size_t lds = (size_t)std::max(1, a.tokens_per_block * a.half) * sizeof(int2);
  auto even = [](const void *p, size_t st, size_t sh) { return !p || (((uintptr_t)p & 15) == 0 && st % 2 == 0 && sh % 2 == 0); };
  const bool pairs = even(d_x, xs_token, xs_head) && even(d_out, os_token, os_head) && even(d_cmp, os_token, os_head) &&
                     head_dim % 2 == 0 && (interleaved || a.half % 2 == 0);
  hipStream_t s = (hipStream_t)stream;
  (void)hipGetLastError();
  if (interleaved) {
    if (pairs) hipLaunchKernelGGL((rotary_kernel<2, true>), grid, dim3(256), lds, s, a);
    else hipLaunchKernelGGL((rotary_kernel<1, true>), grid, dim3(256), lds, s, a);
  } else {
    if (pairs) hipLaunchKernelGGL((rotary_kernel<2, false>), grid, dim3(256), lds, s, a);
    else hipLaunchKernelGGL((rotary_kernel<1, false>), grid, dim3(256), lds, s, a);
  }
  MMH_HIP(hipGetLastError());
  return MMH_OK;
}
}  // namespace mmh

using namespace mmh;

extern "C" int mmh_rotary(const uint64_t *d_x, size_t xs_token, size_t xs_head, size_t n_tokens, size_t n_heads,
                          size_t head_dim, const int64_t *d_pos, const uint64_t *d_phase, size_t rot_dim, int interleaved,
                          double amplitude, int frac_bits, int ring_bw, uint64_t *d_out, size_t os_token, size_t os_head,
                          void *stream) {
  return rotary_call(d_x, xs_token, xs_head, n_tokens, n_heads, head_dim, d_pos, d_phase, rot_dim, interleaved, amplitude,
                     frac_bits, ring_bw, 0, 0, d_out, nullptr, os_token, os_head, stream);
}
extern "C" int mmh_rotary_trunc_pre(int party, const uint64_t *d_x, size_t xs_token, size_t xs_head, size_t n_tokens,
                                    size_t n_heads, size_t head_dim, const int64_t *d_pos, const uint64_t *d_phase,
                                    size_t rot_dim, int interleaved, double amplitude, int frac_bits, int ring_bw,
                                    int signed_arith, int heuristic, uint64_t *d_adj, uint64_t *d_cmp, void *stream) {
  MMH_REQUIRE(party == 1 || party == 2, MMH_ERR_INVALID_ARG);
  MMH_REQUIRE(ring_bw >= (heuristic ? 4 : 2) && ring_bw <= 64, MMH_ERR_INVALID_ARG);
  // the offsets of trunc_pre_kernel (convert.hip); BOB's comparison operand is mask - v, which is v with every bit of the
  // ring flipped
  u64 offset = 0;
  if (heuristic && party != kAlice) offset += u64(1) << (ring_bw - 3);
  if (signed_arith && party == kAlice) offset += u64(1) << (ring_bw - 1);
  return rotary_call(d_x, xs_token, xs_head, n_tokens, n_heads, head_dim, d_pos, d_phase, rot_dim, interleaved, amplitude,
                     frac_bits, ring_bw, offset, party == kAlice ? u64(0) : bw_mask_host(ring_bw), d_adj, d_cmp,
                     n_heads * head_dim, head_dim, stream);
}
