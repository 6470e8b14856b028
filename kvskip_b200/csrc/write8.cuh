// Write of new tokens into the 8-bit cache: code = round(x / s), s the scale of the token's 64-token block
// and KV head, a power of two that covers the largest value of the block so far.
//
// Powers of two: dividing by the scale, and rescaling the codes of a block whose scale grows, are exact for
// e4m3 (a floating-point code loses nothing by a scale that is up to twice the tightest one) short of its
// subnormal range; int8 loses at most one bit of its seven and rounds a second time, by half a step of
// the larger scale, when a block's scale grows.  In return the codes of a block depend on the values alone, not
// on the arithmetic's last bit.
//
// What bounds it: 2 bytes read and 1 written per element: HBM for prompts, the chain slot -> row, old scale
// -> codes for a decode step.  A CTA takes the runs (tokens of one block, consecutive rows) that begin among
// its CHUNK entries of the slot list, for one head and one of K and V.  A few long runs are done by the whole
// CTA one after the other, the values staying in registers between the maximum and the rounding (one read); many
// short ones by a warp each.
#pragma once
#include "common.cuh"
#include "decode8.cuh"

namespace kvb {

constexpr int W8_THREADS = 256;
constexpr int W8_WARPS = W8_THREADS / 32;
constexpr int W8_COOP = 2;             // runs of a chunk up to which the whole CTA works on one run
constexpr float W8_MIN_SCALE = 7.888609052210118e-31f;   // 2^-100

// Largest finite magnitude of two 16-bit floats' bits and m (magnitudes order like their bits).
__device__ __forceinline__ uint32_t w8_top(uint32_t m, const uint32_t w, const uint32_t inf) {
  const uint32_t a = w & 0x7fffu, b = (w >> 16) & 0x7fffu;
  if (a < inf) m = max(m, a);
  if (b < inf) m = max(m, b);
  return m;
}
__device__ __forceinline__ float2 w8_pair(const uint32_t w, const bool f16) {
  return f16 ? unpack_f16(w) : make_float2(bf_lo(w), bf_hi(w));
}
// Smallest power of two s >= 2^-100 with top <= qmax s; top: bits of a finite 16-bit float.
template <int KIND>
__device__ __forceinline__ float w8_scale(const uint32_t top, const bool f16) {
  const float x = f16 ? __half2float(__ushort_as_half(static_cast<unsigned short>(top))) : __uint_as_float(top << 16);
  const uint32_t bits = __float_as_uint(x);
  // qmax = 1.75 * 2^8 or 1.984375 * 2^6
  const int e = static_cast<int>(bits >> 23) - 127 -
                (KIND == KVSKIP_KIND_E4M3 ? 8 : 6) + ((bits & 0x7fffffu) > (KIND == KVSKIP_KIND_E4M3 ? 0x600000u : 0x7e0000u));
  return __uint_as_float(static_cast<uint32_t>(max(e, -100) + 127) << 23);
}
// x / s, exactly rounded: a product with the reciprocal where s is a power of two (uniform in a run)
struct W8Div {
  float s, inv;
  __device__ __forceinline__ explicit W8Div(const float s_) : s(s_), inv(0.f) {
    const uint32_t bits = __float_as_uint(s_);
    if ((bits & 0x7fffffu) == 0 && (bits >> 23) <= 250u) inv = __uint_as_float((254u - (bits >> 23)) << 23);
  }
  __device__ __forceinline__ float operator()(const float x) const { return inv != 0.f ? x * inv : __fdiv_rn(x, s); }
};
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
template <int KIND>
__device__ __forceinline__ uint2 w8_codes8(const uint4 w, const W8Div& div, const bool f16) {
  const float2 a = w8_pair(w.x, f16), b = w8_pair(w.y, f16), c = w8_pair(w.z, f16), d = w8_pair(w.w, f16);
  return make_uint2(w8_codes<KIND>(div(a.x), div(a.y), div(b.x), div(b.y)),
                    w8_codes<KIND>(div(c.x), div(c.y), div(d.x), div(d.y)));
}
// four codes times r, rounded again
template <int KIND>
__device__ __forceinline__ uint32_t w8_again(const uint32_t w, const float r) {
  uint32_t x, y;
  codes_to_f16<KIND, 0>(w, x, y);
  const float2 a = unpack_f16(x), b = unpack_f16(y);
  return w8_codes<KIND>(a.x * r, a.y * r, b.x * r, b.y * r);
}

// One tensor of the call: K or V.
struct W8Side {
  const uint16_t* x;
  int64_t so, si, sh;
  uint8_t* y;
  int64_t sb, sth, st;
  float* scale;
  int64_t cb, ch, ct;
};

template <int KIND, int D, int CHUNK>
__global__ void __launch_bounds__(W8_THREADS) write8_kernel(const __grid_constant__ kvskip_write8_params p) {
  constexpr int LPR = D / 8;                        // lanes of a row, 8 values each
  constexpr int RPC = W8_THREADS / LPR, RPW = 32 / LPR;   // rows of a pass of the CTA / a warp
  constexpr int PASSES = TILE / RPC;
  constexpr int SPAN = CHUNK + TILE;                // slots looked at: the chunk and what a run may reach behind it
  __shared__ int64_t slot[SPAN + 1];                // [0]: the one before the chunk
  __shared__ uint32_t brk[(SPAN + 31) / 32];        // bit i: slot i does not continue the run of slot i - 1
  __shared__ int lead[CHUNK], n_lead;
  __shared__ uint32_t wtop[2][W8_WARPS];

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int h = blockIdx.y;
  const int64_t i0 = static_cast<int64_t>(blockIdx.x) * CHUNK;
  const bool f16 = p.x_f16 != 0;
  const uint32_t inf = f16 ? 0x7c00u : 0x7f80u;
  W8Side t;
  if (blockIdx.z == 0) t = {p.k_new, p.kn_so, p.kn_si, p.kn_sh, p.k, p.k_sb, p.k_sh, p.k_st, p.k_scale, p.ks_sb, p.ks_sh, p.ks_st};
  else t = {p.v_new, p.vn_so, p.vn_si, p.vn_sh, p.v, p.v_sb, p.v_sh, p.v_st, p.v_scale, p.vs_sb, p.vs_sh, p.vs_st};
  const int64_t cap = p.num_blocks * TILE;
  pdl_wait_prior();
  pdl_launch_dependents();

  if (tid == 0) n_lead = 0;
  for (int i = tid; i <= SPAN; i += W8_THREADS) {
    const int64_t at = i0 + i - 1;
    int64_t s = -1;
    if (at >= 0 && at < p.n) {
      s = p.slots[at];
      // outside the cache: a slot too large, or a row that the contiguous form has no room for
      if (s >= cap || (s >= 0 && (s / TILE) % p.blocks * TILE + s % TILE >= p.tokens)) {
        if (h == 0 && blockIdx.z == 0) atomicCAS(&g_status, 0u, 0x302u);
        s = -1;
      }
    }
    slot[i] = s;
  }
  __syncthreads();
  static_assert(SPAN <= W8_THREADS, "one slot a thread");
  if (tid < ((SPAN + 31) & ~31)) {
    const bool in = tid < SPAN;
    const int64_t s = in ? slot[tid + 1] : -1, before = in ? slot[tid] : -1;
    const bool cont = s >= 0 && before >= 0 && s == before + 1 && (s % TILE) != 0;
    const uint32_t bits = __ballot_sync(0xffffffffu, !cont);
    if (lane == 0) brk[warp] = bits;
    if (in && tid < CHUNK && s >= 0 && !cont) {
      if (before >= 0 && s / TILE == before / TILE) {      // a second run of the same block
        if (h == 0 && blockIdx.z == 0) atomicCAS(&g_status, 0u, 0x303u);
      } else {
        lead[atomicAdd(&n_lead, 1)] = tid;                 // (the order of the runs does not matter)
      }
    }
  }
  __syncthreads();

  // values of token i (of this chunk's slots), this thread's eight channels
  auto value = [&](const int i, const int ch) -> uint4 {
    const int64_t at = i0 + i, o = at / p.inner;
    return *reinterpret_cast<const uint4*>(t.x + o * t.so + (at - o * p.inner) * t.si + h * t.sh + 8 * ch);
  };
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
    uint8_t* y;      // the block's codes
    float* scale;
    float old;       // scale of the rows before the run (2^-100 where there are none)
  };
  auto open = [&](const int i) -> Run {
    Run r;
    r.i = i;
    r.n = length(i);
    const int64_t s = slot[i + 1], blk = s / TILE, seq = blk / p.blocks, j = blk - seq * p.blocks;
    r.row = static_cast<int>(s - blk * TILE);
    r.y = t.y + seq * t.sb + h * t.sth + j * TILE * t.st;
    r.scale = t.scale + seq * t.cb + h * t.ch + j * t.ct;
    r.old = W8_MIN_SCALE;
    if (r.row > 0) {
      const float o = *r.scale;
      if (o > 0.f && o <= 3.402823466e38f) r.old = o;
    }
    return r;
  };

  if (n_lead <= W8_COOP) {
    for (int k = 0; k < n_lead; ++k) {
      const Run r = open(lead[k]);
      const int ch = tid % LPR, r0 = tid / LPR;
      uint4 x[PASSES];
      uint32_t top = 0;
#pragma unroll
      for (int q = 0; q < PASSES; ++q) {
        x[q] = make_uint4(0u, 0u, 0u, 0u);
        if (q * RPC + r0 < r.n) x[q] = value(r.i + q * RPC + r0, ch);
      }
#pragma unroll
      for (int q = 0; q < PASSES; ++q)
        top = w8_top(w8_top(w8_top(w8_top(top, x[q].x, inf), x[q].y, inf), x[q].z, inf), x[q].w, inf);
      top = __reduce_max_sync(0xffffffffu, top);
      if (lane == 0) wtop[k & 1][warp] = top;
      __syncthreads();                     // (also: everyone has read the old scale)
#pragma unroll
      for (int w = 0; w < W8_WARPS; ++w) top = max(top, wtop[k & 1][w]);
      const float s = fmaxf(r.old, w8_scale<KIND>(top, f16));
      const W8Div div(s);
#pragma unroll
      for (int q = 0; q < PASSES; ++q)
        if (q * RPC + r0 < r.n)
          *reinterpret_cast<uint2*>(r.y + (r.row + q * RPC + r0) * t.st + 8 * ch) = w8_codes8<KIND>(x[q], div, f16);
      if (r.row > 0 && s > r.old) {
        const float ratio = __fdiv_rn(r.old, s);
        for (int row = r0; row < r.row; row += RPC) {
          uint2* y = reinterpret_cast<uint2*>(r.y + row * t.st + 8 * ch);
          const uint2 w = *y;
          *y = make_uint2(w8_again<KIND>(w.x, ratio), w8_again<KIND>(w.y, ratio));
        }
      }
      if (tid == 0) *r.scale = s;
    }
    return;
  }
  for (int k = warp; k < n_lead; k += W8_WARPS) {
    const Run r = open(lead[k]);
    const int ch = lane % LPR, r0 = lane / LPR;
    uint32_t top = 0;
    for (int q = r0; q < r.n; q += RPW) {
      const uint4 x = value(r.i + q, ch);
      top = w8_top(w8_top(w8_top(w8_top(top, x.x, inf), x.y, inf), x.z, inf), x.w, inf);
    }
    top = __reduce_max_sync(0xffffffffu, top);
    const float s = fmaxf(r.old, w8_scale<KIND>(top, f16));
    const W8Div div(s);
    for (int q = r0; q < r.n; q += RPW)
      *reinterpret_cast<uint2*>(r.y + (r.row + q) * t.st + 8 * ch) = w8_codes8<KIND>(value(r.i + q, ch), div, f16);
    if (r.row > 0 && s > r.old) {
      const float ratio = __fdiv_rn(r.old, s);
      for (int row = r0; row < r.row; row += RPW) {
        uint2* y = reinterpret_cast<uint2*>(r.y + row * t.st + 8 * ch);
        const uint2 w = *y;
        *y = make_uint2(w8_again<KIND>(w.x, ratio), w8_again<KIND>(w.y, ratio));
      }
    }
    if (lane == 0) *r.scale = s;
  }
}

}  // namespace kvb
