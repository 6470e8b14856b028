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
// decode step.  A warp takes the runs (tokens of one block, consecutive rows) that begin among CHUNK entries of the
// slot list, for one of the 2 Hkv (head, K or V) pairs, and needs no other warp: it looks at the slots with ballots,
// brings a run's values into its own 64 rows of shared memory with TMA, reads them there once for the maximum and
// once for the codes.  Runs of one token, those of a decode step, are read from global memory directly, two or four an
// instruction and four or eight at once.
#pragma once
#include "common.cuh"
#include "decode8.cuh"

namespace kvb {

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
// Eight values x / s, exactly rounded, as codes: by the reciprocal `inv` of a power of two, or (a scale that the cache had
// from elsewhere; out of the way of the usual code) by a division.
template <int KIND, bool F16>
__device__ __forceinline__ uint2 w8_codes8(const uint4 w, const float inv) {
  const float2 a = w8_pair<F16>(w.x), b = w8_pair<F16>(w.y), c = w8_pair<F16>(w.z), d = w8_pair<F16>(w.w);
  return make_uint2(w8_codes<KIND>(a.x * inv, a.y * inv, b.x * inv, b.y * inv),
                    w8_codes<KIND>(c.x * inv, c.y * inv, d.x * inv, d.y * inv));
}
template <int KIND, bool F16>
__device__ __noinline__ uint2 w8_codes8_div(const uint4 w, const float s) {
  const float2 a = w8_pair<F16>(w.x), b = w8_pair<F16>(w.y), c = w8_pair<F16>(w.z), d = w8_pair<F16>(w.w);
  return make_uint2(w8_codes<KIND>(__fdiv_rn(a.x, s), __fdiv_rn(a.y, s), __fdiv_rn(b.x, s), __fdiv_rn(b.y, s)),
                    w8_codes<KIND>(__fdiv_rn(c.x, s), __fdiv_rn(c.y, s), __fdiv_rn(d.x, s), __fdiv_rn(d.y, s)));
}
// Rows of a block whose scale has grown, rounded to it: eight codes a lane, rows [row, end) in steps of `rows`.
template <int KIND>
__device__ __noinline__ void w8_again(uint8_t* y, const int64_t st, int row, const int end, const int rows, const float ratio) {
  auto four = [ratio](const uint32_t w) {
    uint32_t x, z;
    codes_to_f16<KIND, 0>(w, x, z);
    const float2 a = unpack_f16(x), b = unpack_f16(z);
    return w8_codes<KIND>(a.x * ratio, a.y * ratio, b.x * ratio, b.y * ratio);
  };
#pragma unroll 4
  for (; row < end; row += rows) {
    uint2* at = reinterpret_cast<uint2*>(y + row * st);
    const uint2 w = *at;
    *at = make_uint2(four(w.x), four(w.y));
  }
}

struct W8Maps {
  CUtensorMap k, v;                      // (D, inner, Hkv, outer) of the new tokens; a box is 16 rows of one head
};
template <int D, int CHUNK>
struct W8Cfg {
  static constexpr int kWarps = CHUNK == 4 ? 2 : 12;
  static constexpr int kBatch = CHUNK == 4 ? 4 : 8;          // runs of one token that a warp has in flight
  static constexpr int kThreads = kWarps * 32;
  static constexpr int kStage = TILE * D * 2;                // a run's values
  static constexpr int kSmem = kWarps * kStage + 128;
};

// tma: the tensor maps are valid (all strides positive); jobs: chunks of the slot list times pairs.
template <int KIND, int D, int CHUNK, bool F16>
__global__ void __launch_bounds__(W8Cfg<D, CHUNK>::kThreads, 1)
write8_kernel(const __grid_constant__ kvskip_write8_params p, const __grid_constant__ W8Maps maps, const int jobs,
              const int tma) {
  using Cfg = W8Cfg<D, CHUNK>;
  constexpr int NW = Cfg::kWarps;
  constexpr int LPR = D / 8, RPW = 32 / LPR;        // lanes of a row, 8 values each; rows of an instruction
  constexpr int WORDS = CHUNK / 32 + (CHUNK % 32 != 0) + 2;   // 32 slots each: the chunk and what a run may reach behind it
  constexpr uint32_t inf = F16 ? 0x7c00u : 0x7f80u;
  extern __shared__ unsigned char smem_raw[];
  __shared__ uint64_t bars[NW];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  unsigned char* stage = smem_raw + ((128 - (smem_u32(smem_raw) & 127)) & 127) + warp * Cfg::kStage;
  uint64_t* bar = &bars[warp];
  if (lane == 0) mbar_init(bar, 1);
  mbar_fence_init();
  __syncwarp();
  pdl_wait_prior();
  pdl_launch_dependents();

  const int n = static_cast<int>(p.n), pairs = 2 * p.Hkv;
  const uint32_t inner = static_cast<uint32_t>(p.inner);
  const int ch = lane % LPR, r0 = lane / LPR;
  uint32_t phase = 0;
  auto read_slots = [&](const int job, int64_t (&s)[WORDS], int64_t& prev) {
    const int i0 = job / pairs * CHUNK;
    prev = -1;
    if (lane == 0 && i0 > 0) prev = p.slots[i0 - 1];
#pragma unroll
    for (int k = 0; k < WORDS; ++k) {
      const int at = i0 + k * 32 + lane;
      s[k] = -1;
      if (k * 32 + lane < CHUNK + TILE && at < n) s[k] = p.slots[at];
    }
  };
  const int step = NW * gridDim.x;
  int job = blockIdx.x * NW + warp;      // (neighbouring warps: the pairs of one chunk, whose values lie side by side)
  int64_t ahead[WORDS], ahead_prev = -1;
  if (job < jobs) read_slots(job, ahead, ahead_prev);

  for (; job < jobs; job += step) {
    const int i0 = job / pairs * CHUNK;
    const int c = job % pairs;             // K heads, then V heads
    const bool v = c >= p.Hkv;
    int64_t slot[WORDS], last = ahead_prev;
#pragma unroll
    for (int k = 0; k < WORDS; ++k) slot[k] = ahead[k];
    if (job + step < jobs) read_slots(job + step, ahead, ahead_prev);

    // ---- the runs: bit i of brk: slot i does not continue the run of slot i - 1; of lead: a run begins there
    uint32_t brk[WORDS + 1], lead[WORDS], single[WORDS];
    auto outside = [&](const int64_t s) {           // a slot too large, or a row the contiguous form has no room for
      bool out = s >= p.num_blocks * TILE;
      if (p.blocks > 1 || p.tokens < TILE) out |= s >= 0 && (s / TILE) % p.blocks * TILE + s % TILE >= p.tokens;
      return out;
    };
    if (outside(last)) last = -1;
#pragma unroll
    for (int k = 0; k < WORDS; ++k) {
      const bool in = k * 32 + lane < CHUNK;
      if (outside(slot[k])) {
        if (in && c == 0) atomicCAS(&g_status, 0u, 0x302u);
        slot[k] = -1;
      }
      int64_t before = __shfl_up_sync(0xffffffffu, slot[k], 1);
      if (lane == 0) before = last;
      last = __shfl_sync(0xffffffffu, slot[k], 31);
      const bool some = slot[k] >= 0;
      const bool cont = some && before >= 0 && slot[k] == before + 1 && (slot[k] & (TILE - 1)) != 0;
      const bool twice = some && !cont && before >= 0 && (slot[k] >> 6) == (before >> 6);   // a second run of the block
      if (twice && in && c == 0) atomicCAS(&g_status, 0u, 0x303u);
      brk[k] = __ballot_sync(0xffffffffu, !cont);
      lead[k] = __ballot_sync(0xffffffffu, some && !cont && !twice && in);
    }
    brk[WORDS] = 0xffffffffu;
#pragma unroll
    for (int k = 0; k < WORDS; ++k) single[k] = lead[k] & __funnelshift_r(brk[k], brk[k + 1], 1);   // the next slot breaks too
    struct Run {
      int i, n, row;
      int64_t seq, blk;    // sequence (page) and block in it
    };
    auto open = [&](const int k, const int bit) -> Run {
      Run r;
      r.i = k * 32 + bit;
      r.n = 0;
      int64_t s = 0;
#pragma unroll
      for (int x = 0; x < WORDS; ++x) {
        const int64_t v = __shfl_sync(0xffffffffu, slot[x], bit);
        if (x == k) s = v;
        // tokens up to the next break (a run ends with its block, at most 64 tokens on)
        const uint32_t w = x < k ? 0u : x == k ? brk[x] & ~((2u << bit) - 1u) : brk[x];
        if (r.n == 0 && w) r.n = x * 32 + __ffs(w) - 1 - r.i;
      }
      if (r.n == 0) r.n = WORDS * 32 - r.i;
      r.row = static_cast<int>(s & (TILE - 1));
      r.seq = s >> 6, r.blk = 0;
      if (p.blocks > 1) r.blk = r.seq % p.blocks, r.seq /= p.blocks;
      return r;
    };
    auto source = [&](const uint32_t at) -> const uint16_t* {    // values of one token
      const uint32_t o = inner == static_cast<uint32_t>(n) ? 0u : at / inner, in = at - o * inner;
      return v ? p.v_new + o * p.vn_so + in * p.vn_si + (c - p.Hkv) * p.vn_sh : p.k_new + o * p.kn_so + in * p.kn_si + c * p.kn_sh;
    };
    auto codes = [&](const Run& r) -> uint8_t* {
      return v ? p.v + r.seq * p.v_sb + (c - p.Hkv) * p.v_sh + (r.blk * TILE + r.row) * p.v_st
               : p.k + r.seq * p.k_sb + c * p.k_sh + (r.blk * TILE + r.row) * p.k_st;
    };
    auto scale = [&](const Run& r) -> float* {
      return v ? p.v_scale + r.seq * p.vs_sb + (c - p.Hkv) * p.vs_sh + r.blk * p.vs_st
               : p.k_scale + r.seq * p.ks_sb + c * p.ks_sh + r.blk * p.ks_st;
    };
    auto usable = [](const float o) { return o > 0.f && o <= 3.402823466e38f ? o : W8_MIN_SCALE; };
    // rows before the run, rounded to the larger scale
    const int64_t st = v ? p.v_st : p.k_st;
    auto again = [&](const Run& r, const float ratio, const int row0, const int rows) {
      w8_again<KIND>(codes(r) - r.row * st + 8 * ch, st, row0, r.row, rows, ratio);
    };
    auto put = [&](uint8_t* y, const uint4 x, const float s, const float inv) {
      *reinterpret_cast<uint2*>(y) = inv != 0.f ? w8_codes8<KIND, F16>(x, inv) : w8_codes8_div<KIND, F16>(x, s);
    };

    // ---- runs of several tokens
#pragma unroll
    for (int k = 0; k < (CHUNK + 31) / 32; ++k)
      for (uint32_t rest = lead[k] & ~single[k]; rest; rest &= rest - 1) {
        const Run r = open(k, __ffs(rest) - 1);
        const uint32_t at = i0 + r.i, o = inner == static_cast<uint32_t>(n) ? 0u : at / inner, in = at - o * inner;
        const bool staged = tma && in + r.n <= inner;      // (a run may go on in the next row of a padded list)
        float was = W8_MIN_SCALE;
        if (r.row > 0) was = *scale(r);
        if (staged && lane == 0) {
          const int boxes = (r.n + 15) / 16;
          mbar_expect_tx(bar, boxes * 16 * D * 2);
          for (int x = 0; x < boxes; ++x)
            tma_load_4d(stage + x * 16 * D * 2, v ? &maps.v : &maps.k, bar, 0, in + 16 * x, v ? c - p.Hkv : c, o);
        }
        was = usable(was);
        uint32_t top = 0;
        const uint4* mine = reinterpret_cast<const uint4*>(stage) + lane;     // row r0, then every RPW-th
        if (staged) {
          if (!mbar_wait_warp(bar, phase, 0x740u + warp)) return;
          phase ^= 1;
          const int full = r.n / RPW;
          int q = 0;
          for (; q + 8 <= full; q += 8)
#pragma unroll
            for (int u = 0; u < 8; ++u) top = w8_top(top, mine[(q + u) * 32]);
          for (; q * RPW + r0 < r.n; ++q) top = w8_top(top, mine[q * 32]);
          if (__any_sync(0xffffffffu, max(top & 0xffffu, top >> 16) >= inf)) {
            top = 0;
            for (q = 0; q * RPW + r0 < r.n; ++q) top = w8_top_finite(top, mine[q * 32], inf);
          }
        } else {
          for (int q = r0; q < r.n; q += RPW)
            top = w8_top_finite(top, *reinterpret_cast<const uint4*>(source(at + q) + 8 * ch), inf);
        }
        top = __reduce_max_sync(0xffffffffu, max(top & 0xffffu, top >> 16));
        const float s = fmaxf(was, w8_scale<KIND, F16>(top)), inv = w8_inverse(s);
        uint8_t* y = codes(r) + r0 * st + 8 * ch;
        if (staged && inv != 0.f) {
          const int full = r.n / RPW;
          int q = 0;
          for (; q + 4 <= full; q += 4, y += 4 * RPW * st)
#pragma unroll
            for (int u = 0; u < 4; ++u) *reinterpret_cast<uint2*>(y + u * RPW * st) = w8_codes8<KIND, F16>(mine[(q + u) * 32], inv);
          for (; q * RPW + r0 < r.n; ++q, y += RPW * st) *reinterpret_cast<uint2*>(y) = w8_codes8<KIND, F16>(mine[q * 32], inv);
        } else {
          for (int q = r0; q < r.n; q += RPW, y += RPW * st)
            put(y, staged ? mine[(q - r0) / RPW * 32] : *reinterpret_cast<const uint4*>(source(at + q) + 8 * ch), s, inv);
        }
        if (r.row > 0 && s > was) again(r, __fdiv_rn(was, s), r0, RPW);
        __syncwarp();                    // the stage has been read, and the old scale by every lane
        if (lane == 0) *scale(r) = s;
      }

    // ---- runs of one token: lanes r0 = 0 .. RPW - 1 take one each, kBatch / RPW of them at once
    constexpr int U = Cfg::kBatch / RPW;
#pragma unroll
    for (int k = 0; k < (CHUNK + 31) / 32; ++k)
      for (uint32_t rest = single[k]; rest;) {
        Run r[U];
        uint4 x[U];
        float was[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          r[u].i = -1;
#pragma unroll
          for (int m = 0; m < RPW; ++m) {
            const int bit = rest ? __ffs(rest) - 1 : 0;
            const int64_t s = __shfl_sync(0xffffffffu, slot[k], bit);
            if (m == r0 && rest) {
              r[u].i = k * 32 + bit, r[u].n = 1;
              r[u].row = static_cast<int>(s & (TILE - 1));
              r[u].seq = s >> 6, r[u].blk = 0;
              if (p.blocks > 1) r[u].blk = r[u].seq % p.blocks, r[u].seq /= p.blocks;
            }
            rest &= rest - 1;
          }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          x[u] = make_uint4(0u, 0u, 0u, 0u);
          was[u] = W8_MIN_SCALE;
          if (r[u].i >= 0) {
            x[u] = *reinterpret_cast<const uint4*>(source(i0 + r[u].i) + 8 * ch);
            if (r[u].row > 0) was[u] = *scale(r[u]);
          }
        }
        __syncwarp();                    // every lane of a row has the old scale before one of them stores the new one
#pragma unroll
        for (int u = 0; u < U; ++u) {
          uint32_t top = w8_top_finite(0u, x[u], inf);
          top = max(top & 0xffffu, top >> 16);
#pragma unroll
          for (int d = LPR / 2; d > 0; d >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, d));
          if (r[u].i >= 0) {
            const float old = usable(was[u]), s = fmaxf(old, w8_scale<KIND, F16>(top));
            put(codes(r[u]) + 8 * ch, x[u], s, w8_inverse(s));
            if (r[u].row > 0 && s > old) again(r[u], __fdiv_rn(old, s), 0, 1);
            if (ch == 0) *scale(r[u]) = s;
          }
        }
      }
  }
}

}  // namespace kvb
