// Write of new tokens into the 8-bit cache: code = round(x / s), s the scale of the token's 64-token block
// and KV head, a power of two that covers the largest value of the block so far.
//
// Powers of two: dividing by the scale, and rescaling the codes of a block whose scale grows, are exact for
// e4m3 (a floating-point code loses nothing by a scale that is up to twice the tightest one) short of its
// subnormal range; int8 loses at most one bit of its seven and rounds a second time, by half a step of
// the larger scale, when a block's scale grows.  In return the codes of a block depend on the values alone, not
// on the arithmetic's last bit.
//
// What bounds it: 2 bytes read and 1 written per element: HBM for prompts, the chain slot -> scale so far -> codes for a
// decode step.  A CTA takes the runs (tokens of one block, consecutive rows) that begin among its CHUNK entries of the
// slot list, for `items` of the 2 Hkv (head, K or V) pairs.  A few long runs are done by the whole CTA one after the
// other: the values of a run stay in registers between the maximum and the rounding (one read), and those of the next
// one are on their way meanwhile.  Many short ones, the tokens of a decode step, are done by a warp each.
#pragma once
#include "common.cuh"
#include "decode8.cuh"

namespace kvb {

constexpr int W8_THREADS = 256;
constexpr int W8_WARPS = W8_THREADS / 32;
constexpr int W8_COOP = 2;             // runs of a chunk up to which the whole CTA works on one run
constexpr float W8_MIN_SCALE = 7.888609052210118e-31f;   // 2^-100

// Largest magnitude of the 16-bit floats of a 16-byte group and m, two at a time (magnitudes order like their bits).
__device__ __forceinline__ uint32_t w8_top(uint32_t m, const uint4 w) {
  m = __vmaxu2(m, w.x & 0x7fff7fffu);
  m = __vmaxu2(m, w.y & 0x7fff7fffu);
  m = __vmaxu2(m, w.z & 0x7fff7fffu);
  return __vmaxu2(m, w.w & 0x7fff7fffu);
}
// The same of the finite ones alone.
__device__ __forceinline__ uint32_t w8_top_finite(uint32_t m, const uint4 w, const uint32_t inf) {
  const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t a = v[i] & 0x7fffu, b = (v[i] >> 16) & 0x7fffu;
    m = __vmaxu2(m, (a < inf ? a : 0u) | (b < inf ? b << 16 : 0u));
  }
  return m;
}
template <bool F16>
__device__ __forceinline__ float2 w8_pair(const uint32_t w) {
  return F16 ? unpack_f16(w) : make_float2(bf_lo(w), bf_hi(w));
}
// Smallest power of two s >= 2^-100 with top <= qmax s; top: bits of a finite 16-bit float.
template <int KIND, bool F16>
__device__ __forceinline__ float w8_scale(const uint32_t top) {
  const float x = F16 ? __half2float(__ushort_as_half(static_cast<unsigned short>(top))) : __uint_as_float(top << 16);
  const uint32_t bits = __float_as_uint(x);
  // qmax = 1.75 * 2^8 or 1.984375 * 2^6
  const int e = static_cast<int>(bits >> 23) - 127 -
                (KIND == KVSKIP_KIND_E4M3 ? 8 : 6) + ((bits & 0x7fffffu) > (KIND == KVSKIP_KIND_E4M3 ? 0x600000u : 0x7e0000u));
  return __uint_as_float(static_cast<uint32_t>(max(e, -100) + 127) << 23);
}
// 1 / s where that is exact (s a power of two in range), else 0
__device__ __forceinline__ float w8_inverse(const float s) {
  const uint32_t bits = __float_as_uint(s);
  return (bits & 0x7fffffu) == 0 && (bits >> 23) <= 250u ? __uint_as_float((254u - (bits >> 23)) << 23) : 0.f;
}
// four values (in units of the scale) -> four codes
template <int KIND>
__device__ __forceinline__ uint32_t w8_codes(const float a, const float b, const float c, const float d) {
  if constexpr (KIND == KVSKIP_KIND_E4M3) {
    uint16_t lo, hi;      // rounds to nearest even, saturates, keeps a NaN
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
    return lo | (static_cast<uint32_t>(hi) << 16);
  } else {
    auto one = [](const float x) -> uint32_t {      // (the conversion of a NaN gives 0)
      return static_cast<uint32_t>(max(-127, min(127, __float2int_rn(x)))) & 0xffu;
    };
    return one(a) | (one(b) << 8) | (one(c) << 16) | (one(d) << 24);
  }
}
// Eight values x / s, exactly rounded, as codes.  EXACT: by the reciprocal `f` of a power of two, else by s = f itself
// (a scale that the cache had from elsewhere).
template <int KIND, bool F16, bool EXACT>
__device__ __forceinline__ uint2 w8_codes8(const uint4 w, const float f) {
  const float2 a = w8_pair<F16>(w.x), b = w8_pair<F16>(w.y), c = w8_pair<F16>(w.z), d = w8_pair<F16>(w.w);
  auto q = [f](const float x) { return EXACT ? x * f : __fdiv_rn(x, f); };
  return make_uint2(w8_codes<KIND>(q(a.x), q(a.y), q(b.x), q(b.y)), w8_codes<KIND>(q(c.x), q(c.y), q(d.x), q(d.y)));
}
// four codes times r, rounded again
template <int KIND>
__device__ __forceinline__ uint32_t w8_again(const uint32_t w, const float r) {
  uint32_t x, y;
  codes_to_f16<KIND, 0>(w, x, y);
  const float2 a = unpack_f16(x), b = unpack_f16(y);
  return w8_codes<KIND>(a.x * r, a.y * r, b.x * r, b.y * r);
}

template <int KIND, int D, int CHUNK, bool F16>
__global__ void __launch_bounds__(W8_THREADS, 4)
write8_kernel(const __grid_constant__ kvskip_write8_params p, const int items) {
  constexpr int LPR = D / 8;                        // lanes of a row, 8 values each
  constexpr int RPC = W8_THREADS / LPR, RPW = 32 / LPR;   // rows of a pass of the CTA / a warp
  constexpr int PASSES = TILE / RPC;
  constexpr int SPAN = CHUNK + TILE;                // slots looked at: the chunk and what a run may reach behind it
  static_assert(SPAN < W8_THREADS, "one slot a thread");
  __shared__ int64_t slot[SPAN + 1];                // [0]: the one before the chunk
  __shared__ uint32_t brk[(SPAN + 31) / 32];        // bit i: slot i does not continue the run of slot i - 1
  __shared__ int lead[CHUNK], n_lead, longest;
  __shared__ uint32_t wtop[2][W8_WARPS];
  __shared__ float wold[2];

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  // Blocks of one chunk follow one another, K heads first: the 2 D bytes that a pair reads of a token lie beside those of
  // its neighbours, and DRAM pages are opened once for all of them.
  const int groups = (2 * p.Hkv + items - 1) / items;
  const int i0 = blockIdx.x / groups * CHUNK, n = static_cast<int>(p.n);
  const int c0 = blockIdx.x % groups * items, c1 = min(c0 + items, 2 * p.Hkv);     // pairs: K heads, then V heads
  const bool first = c0 == 0;
  constexpr uint32_t inf = F16 ? 0x7c00u : 0x7f80u;
  pdl_wait_prior();
  pdl_launch_dependents();

  // values of token i (of this chunk's slots), eight channels
  auto value = [&](const int i, const int c, const int ch) -> uint4 {
    const uint32_t at = i0 + i, inner = static_cast<uint32_t>(p.inner);
    const uint32_t o = p.inner == p.n ? 0u : at / inner;
    const bool v = c >= p.Hkv;
    const int64_t so = v ? p.vn_so : p.kn_so, si = v ? p.vn_si : p.kn_si, sh = v ? p.vn_sh : p.kn_sh;
    return __ldg(reinterpret_cast<const uint4*>((v ? p.v_new : p.k_new) + o * so + (at - o * inner) * si + (v ? c - p.Hkv : c) * sh + 8 * ch));
  };
  if (tid == 0) n_lead = longest = 0;
  if (tid <= SPAN) {
    const int at = i0 + tid - 1;
    int64_t s = -1;
    if (at >= 0 && at < n) {
      s = p.slots[at];
      // outside the cache: a slot too large, or a row that the contiguous form has no room for
      bool out = s >= p.num_blocks * TILE;
      if (p.blocks > 1 || p.tokens < TILE) out |= s >= 0 && (s / TILE) % p.blocks * TILE + s % TILE >= p.tokens;
      if (out) {
        if (first) atomicCAS(&g_status, 0u, 0x302u);
        s = -1;
      }
    }
    slot[tid] = s;
  }
  __syncthreads();
  if (tid < ((SPAN + 31) & ~31)) {
    const bool in = tid < SPAN;
    const int64_t s = in ? slot[tid + 1] : -1, before = in ? slot[tid] : -1;
    const bool cont = s >= 0 && before >= 0 && s == before + 1 && (s & (TILE - 1)) != 0;
    const uint32_t bits = __ballot_sync(0xffffffffu, !cont);
    if (lane == 0) brk[warp] = bits;
    if (in && tid < CHUNK && s >= 0 && !cont) {
      if (before >= 0 && (s >> 6) == (before >> 6)) {      // a second run of the same block
        if (first) atomicCAS(&g_status, 0u, 0x303u);
      } else {
        lead[atomicAdd(&n_lead, 1)] = tid;                 // (the order of the runs does not matter)
      }
    }
  }
  __syncthreads();

  auto length = [&](const int i) -> int {                  // tokens of the run that begins at i
    int j = i + 1;
    while (j < SPAN) {
      const uint32_t w = brk[j >> 5] >> (j & 31);
      if (w) return min(j + __ffs(w) - 1, SPAN) - i;
      j = (j | 31) + 1;
    }
    return SPAN - i;                                       // (runs end at the block's last row: at most 64)
  };
  struct Run {
    int i, n, row;
    int64_t seq, blk;    // sequence (page) and block in it
  };
  auto open = [&](const int i) -> Run {
    Run r;
    r.i = i;
    r.n = length(i);
    const int64_t s = slot[i + 1];
    r.row = static_cast<int>(s & (TILE - 1));
    r.seq = s >> 6, r.blk = 0;
    if (p.blocks > 1) r.blk = r.seq % p.blocks, r.seq /= p.blocks;
    return r;
  };
  auto codes = [&](const Run& r, const int c) -> uint8_t* {
    return c >= p.Hkv ? p.v + r.seq * p.v_sb + (c - p.Hkv) * p.v_sh + (r.blk * TILE + r.row) * p.v_st
                      : p.k + r.seq * p.k_sb + c * p.k_sh + (r.blk * TILE + r.row) * p.k_st;
  };
  auto scale = [&](const Run& r, const int c) -> float* {
    return c >= p.Hkv ? p.v_scale + r.seq * p.vs_sb + (c - p.Hkv) * p.vs_sh + r.blk * p.vs_st
                      : p.k_scale + r.seq * p.ks_sb + c * p.ks_sh + r.blk * p.ks_st;
  };
  auto before = [&](const Run& r, const int c) -> float {  // scale of the rows before the run
    if (r.row == 0) return W8_MIN_SCALE;
    const float o = *scale(r, c);
    return o > 0.f && o <= 3.402823466e38f ? o : W8_MIN_SCALE;
  };
  // rows before the run, rounded to the larger scale
  auto again = [&](const Run& r, const int c, const float ratio, const int ch, const int r0, const int step) {
    const int64_t st = c >= p.Hkv ? p.v_st : p.k_st;
    for (int row = r0 - r.row; row < 0; row += step) {
      uint2* y = reinterpret_cast<uint2*>(codes(r, c) + row * st + 8 * ch);
      const uint2 w = *y;
      *y = make_uint2(w8_again<KIND>(w.x, ratio), w8_again<KIND>(w.y, ratio));
    }
  };

  if (n_lead <= W8_COOP) {
    if (tid < n_lead) atomicMax(&longest, length(lead[tid]));
    __syncthreads();
  }
  if (n_lead <= W8_COOP && longest > 2 * RPW) {
    const int ch = tid % LPR, r0 = tid / LPR;
    const Run run0 = open(lead[0]), run1 = open(lead[n_lead - 1]);
    const int jobs = (c1 - c0) * n_lead;
    // (a run that goes on in the next row of a padded list has no one stride)
    const uint32_t inner = static_cast<uint32_t>(p.inner);
    auto fetch = [&](const int j, uint4 (&x)[PASSES], float& old) {
      const Run& r = j % n_lead ? run1 : run0;
      const int c = c0 + j / n_lead;
      const uint32_t at = i0 + r.i, o = inner == static_cast<uint32_t>(n) ? 0u : at / inner, in = at - o * inner;
      if (in + r.n <= inner) {
        const bool v = c >= p.Hkv;
        const int64_t si = v ? p.vn_si : p.kn_si;
        const uint16_t* src = v ? p.v_new + o * p.vn_so + (c - p.Hkv) * p.vn_sh : p.k_new + o * p.kn_so + c * p.kn_sh;
        src += (in + r0) * si + 8 * ch;
#pragma unroll
        for (int q = 0; q < PASSES; ++q) {
          x[q] = make_uint4(0u, 0u, 0u, 0u);
          if (q * RPC + r0 < r.n) x[q] = __ldg(reinterpret_cast<const uint4*>(src + q * RPC * si));
        }
      } else {
#pragma unroll
        for (int q = 0; q < PASSES; ++q) {
          x[q] = make_uint4(0u, 0u, 0u, 0u);
          if (q * RPC + r0 < r.n) x[q] = value(r.i + q * RPC + r0, c, ch);
        }
      }
      if (tid == 0) old = before(r, c);
    };
    auto work = [&](const int j, const uint4 (&x)[PASSES], const float old) {
      const Run& r = j % n_lead ? run1 : run0;
      const int c = c0 + j / n_lead;
      uint32_t top = 0;
#pragma unroll
      for (int q = 0; q < PASSES; ++q) top = w8_top(top, x[q]);
      if (max(top & 0xffffu, top >> 16) >= inf) {
        top = 0;
#pragma unroll
        for (int q = 0; q < PASSES; ++q) top = w8_top_finite(top, x[q], inf);
      }
      top = __reduce_max_sync(0xffffffffu, max(top & 0xffffu, top >> 16));
      if (lane == 0) wtop[j & 1][warp] = top;
      if (tid == 0) wold[j & 1] = old;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < W8_WARPS; ++w) top = max(top, wtop[j & 1][w]);
      const float was = wold[j & 1], s = fmaxf(was, w8_scale<KIND, F16>(top));
      const float inv = w8_inverse(s);
      const int64_t st = c >= p.Hkv ? p.v_st : p.k_st;
      uint8_t* y = codes(r, c) + r0 * st + 8 * ch;
      if (inv != 0.f) {
#pragma unroll
        for (int q = 0; q < PASSES; ++q)
          if (q * RPC + r0 < r.n) *reinterpret_cast<uint2*>(y + q * RPC * st) = w8_codes8<KIND, F16, true>(x[q], inv);
      } else {
#pragma unroll
        for (int q = 0; q < PASSES; ++q)
          if (q * RPC + r0 < r.n) *reinterpret_cast<uint2*>(y + q * RPC * st) = w8_codes8<KIND, F16, false>(x[q], s);
      }
      if (r.row > 0 && s > was) again(r, c, __fdiv_rn(was, s), ch, r0, RPC);
      if (tid == 0) *scale(r, c) = s;
    };
    uint4 x[PASSES], y[PASSES];
    float ox = 0.f, oy = 0.f;
    fetch(0, x, ox);
    for (int j = 0; j < jobs; j += 2) {
      if (j + 1 < jobs) fetch(j + 1, y, oy);
      work(j, x, ox);
      if (j + 1 == jobs) break;
      if (j + 2 < jobs) fetch(j + 2, x, ox);
      work(j + 1, y, oy);
    }
    return;
  }
  for (int k = warp; k < n_lead; k += W8_WARPS) {
    const Run r = open(lead[k]);
    const int ch = lane % LPR, r0 = lane / LPR;
    for (int c = c0; c < c1; ++c) {
      const float was = before(r, c);
      uint32_t top = 0;
      for (int q = r0; q < r.n; q += RPW) top = w8_top_finite(top, value(r.i + q, c, ch), inf);
      top = __reduce_max_sync(0xffffffffu, max(top & 0xffffu, top >> 16));
      const float s = fmaxf(was, w8_scale<KIND, F16>(top));
      const float inv = w8_inverse(s);
      uint8_t* y = codes(r, c) + 8 * ch;
      const int64_t st = c >= p.Hkv ? p.v_st : p.k_st;
      for (int q = r0; q < r.n; q += RPW) {
        const uint4 x = value(r.i + q, c, ch);
        *reinterpret_cast<uint2*>(y + q * st) = inv != 0.f ? w8_codes8<KIND, F16, true>(x, inv) : w8_codes8<KIND, F16, false>(x, s);
      }
      if (r.row > 0 && s > was) again(r, c, __fdiv_rn(was, s), ch, r0, RPW);
      __syncwarp();                        // (every lane has read the old scale)
      if (lane == 0) *scale(r, c) = s;
    }
  }
}

}  // namespace kvb
