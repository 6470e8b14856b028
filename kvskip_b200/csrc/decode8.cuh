// Attention of one token per sequence over a cache of 8-bit codes with a scale per 64-token block and
// KV head:   s_t = scale * ks[blk(t)] * q . k8[t],   out = sum_t softmax(s)_t * vs[blk(t)] * v8[t].
//
// What bounds it: 2 D bytes per token and KV head against 4 G D operations, at most 32 operations a byte
// for G = 16: HBM, as long as the arithmetic stays out of the way.  The codes go to the tensor cores as
// fp16, which holds every e4m3 and int8 value exactly (converting q to 8 bits instead would lose what the
// codes keep); q is held in fp16 relative to a power of two of its own row, so nothing of a bf16 q is
// lost that could show in an fp32 sum.  M is the token (scores) or the channel (output) axis and the G
// query heads of a KV head are the 8 columns of mma.m16n8k16: the tcgen05 shapes start at 64 x 8 per
// instruction but take A from shared memory or TMEM in fp16, so the converted codes would have to be
// written back there first, which costs more than the products do.
//
// Work split: the (sequence, head, block) items of the whole launch are one list, ordered by sequence,
// head and block; CTA c of C takes the items [W c / C, W (c+1) / C), its warps contiguous parts of those.
// So requests of any mixture of lengths keep every SM busy to the end without the host knowing a length.
// A warp keeps the running maximum, sum and output of the head it is in and has its own ring of
// stages (a K and a V tile with an mbarrier each): no barrier between warps inside the loop.  A head that a
// warp starts and ends is written out by that warp; the other pieces (at most two per warp) are joined in shared
// memory in item order, and what then still is a part of a head (at most two per CTA) goes to `work` and is
// joined by decode8_merge_kernel.  Everything is added in a fixed order: results do not depend on timing.
//
// P (0..1 relative to its block's maximum) goes to the tensor cores as fp16 high + low parts, which hold
// 22 bits of it: with G <= 4 the two parts share one instruction (columns 0-3 high, 4-7 low; the scores of a
// head are computed in both, which costs nothing), else they are two instructions.  P is scaled by 2^13,
// so that weights down to 2^-27 of the block's maximum are normal fp16 numbers.
#pragma once
#include "common.cuh"
#include "mma.cuh"

namespace kvb {

struct D8Maps {
  CUtensorMap k, v;
};

// MODE 0: G <= 4, one column tile with high and low parts; 1: G <= 8, one tile; 2: G <= 16, two tiles.
template <int D, int MODE>
struct D8Cfg {
  static constexpr int kCols = MODE == 0 ? 4 : MODE == 1 ? 8 : 16;   // query heads there is room for
  static constexpr int kTiles = MODE == 2 ? 2 : 1;
  static constexpr int kParts = MODE == 0 ? 1 : 2;                   // MMA instructions per P fragment
  static constexpr int kWarps = MODE == 0 ? 12 : MODE == 1 ? 10 : 8;
  static constexpr int kThreads = kWarps * 32;
  static constexpr int kStages = D == 128 ? 1 : 2;                   // per warp
  static constexpr int kTile = TILE * D;                             // bytes of a K or V tile
  static constexpr int kRing = kWarps * kStages * 2 * kTile;
  static constexpr int kPiece = kCols * (D + 2);                     // floats of a piece: acc, m, l
  static constexpr int kFirst = kWarps * kPiece * 4;                 // pieces that begin before their warp's part
  static constexpr int kSmem = kRing + kFirst + 1024;
  static_assert(kPiece * 4 <= kStages * 2 * kTile, "a warp's last piece fits into its ring");
};

constexpr float D8_PSCALE = 13.f;   // log2 of the scaling of P
constexpr int D8_MAX_CTAS = 160;    // bound on the grid that `work` is sized for (148 SMs)

__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
               "{%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float2 unpack_f16(uint32_t x) {
  return __half22float2(*reinterpret_cast<const __half2*>(&x));
}
__device__ __forceinline__ uint32_t sub_f16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// Four codes of a register -> two fp16 pairs, exactly.  PAIRS 0: (b0, b1) and (b2, b3); 1: (b0, b2) and
// (b1, b3).  int8: 1024 + (code + 128) is the fp16 number 0x64uu with uu = code ^ 0x80.
template <int KIND, int PAIRS>
__device__ __forceinline__ void codes_to_f16(uint32_t w, uint32_t& x, uint32_t& y) {
  if constexpr (KIND == KVSKIP_KIND_E4M3) {
    if constexpr (PAIRS == 1) w = __byte_perm(w, 0u, 0x3120);
    asm("{\n.reg .b16 l, h;\nmov.b32 {l, h}, %2;\ncvt.rn.f16x2.e4m3x2 %0, l;\ncvt.rn.f16x2.e4m3x2 %1, h;\n}"
        : "=r"(x), "=r"(y) : "r"(w));
  } else {
    w ^= 0x80808080u;
    x = sub_f16x2(__byte_perm(w, 0x64646464u, PAIRS == 0 ? 0x4140 : 0x4240), 0x64806480u);
    y = sub_f16x2(__byte_perm(w, 0x64646464u, PAIRS == 0 ? 0x4342 : 0x4341), 0x64806480u);
  }
}

// One block of the work list, held by one lane.
struct D8Item {
  int bh, blk, page;   // sequence * Hkv + head; block; page (paged form) or sequence
  int info;            // valid tokens | first of its head << 8 | last of its head << 9
  int left;            // items of the head behind this one
  float ks, vs;
};

// Items of one unit of the list: a sequence (all heads, every block) or, with block lists, a (sequence, head).
__device__ __forceinline__ int d8_len(const kvskip_decode8_params& p, int b) {
  return p.lens ? max(0, min(p.lens[b], p.T)) : p.T;
}
__device__ __forceinline__ int d8_count(const kvskip_decode8_params& p, int u) {
  if (p.block_idx) return max(0, min(p.block_cnt[u], p.max_blocks));
  return (d8_len(p, u) + TILE - 1) / TILE;
}

// Item x of the list; pref[t]: items before the units of thread t's share.
template <int THREADS>
__device__ __forceinline__ D8Item d8_item(const kvskip_decode8_params& p, const int* pref, const int per, const int x) {
  D8Item it;
  int lo = 0, hi = THREADS - 1;          // last t with pref[t] <= x
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (pref[mid] <= x) lo = mid; else hi = mid - 1;
  }
  const int mul = p.block_idx ? 1 : p.Hkv;
  int rem = x - pref[lo], u = lo * per, cnt = d8_count(p, u);
  while (rem >= cnt * mul) {
    rem -= cnt * mul;
    cnt = d8_count(p, ++u);
  }
  int b, h, j;
  if (p.block_idx) {
    b = u / p.Hkv, h = u - b * p.Hkv, j = rem;
    it.blk = p.block_idx[static_cast<int64_t>(u) * p.max_blocks + j];
  } else {
    b = u, h = rem / cnt, j = rem - h * cnt;
    it.blk = j;
  }
  it.bh = b * p.Hkv + h;
  const bool in = it.blk >= 0 && it.blk < p.nb;
  const int tok = in ? max(0, min(TILE, d8_len(p, b) - it.blk * TILE)) : 0;
  it.info = tok | (j == 0 ? 256 : 0) | (j == cnt - 1 ? 512 : 0);
  it.left = cnt - 1 - j;
  it.ks = it.vs = 0.f;
  it.page = b;
  if (p.page_table) {
    it.page = in ? p.page_table[static_cast<int64_t>(b) * p.max_pages + it.blk] : -1;
    if (it.page >= 0 && it.page < p.num_pages) {
      it.ks = p.k_scale[it.page * p.ks_sb + h * p.ks_sh];
      it.vs = p.v_scale[it.page * p.vs_sb + h * p.vs_sh];
    } else {
      it.page = -1;                      // out of bounds for the tensor map: reads as zeros
    }
  } else if (in) {
    it.ks = p.k_scale[b * p.ks_sb + h * p.ks_sh + it.blk * p.ks_st];
    it.vs = p.v_scale[b * p.vs_sb + h * p.vs_sh + it.blk * p.vs_st];
  }
  if (tok == 0) it.ks = it.vs = 0.f;     // a listed block behind the length: its scale may be anything
  return it;
}

// Output rows: o[head][d0], [d0 + 1] of query head hq.
__device__ __forceinline__ void d8_store(const kvskip_decode8_params& p, const int64_t hq, const int d0, float a, float b) {
  uint32_t w;
  if (p.q_f16) w = pack_f16(a, b);
  else w = pack_bf16(a, b);
  *reinterpret_cast<uint32_t*>(p.out + hq * p.D + d0) = w;
  if (p.out_f32) *reinterpret_cast<float2*>(p.out_f32 + hq * p.D + d0) = make_float2(a, b);
}
__device__ __forceinline__ float d8_lse(float m, float l) {
  return l == 0.f ? -INFINITY : (m + log2f(l) - D8_PSCALE) * LN2;   // (a NaN sum stays one)
}
__device__ __forceinline__ float d8_safe(float m) { return m == -INFINITY ? 0.f : m; }

template <int KIND, int D, int MODE>
__global__ void __launch_bounds__(D8Cfg<D, MODE>::kThreads, 1)
decode8_kernel(const __grid_constant__ kvskip_decode8_params p, const __grid_constant__ D8Maps maps, const int min_items) {
  using Cfg = D8Cfg<D, MODE>;
  constexpr int NW = Cfg::kWarps, NT = Cfg::kThreads, ST = Cfg::kStages, KS = D / 16;
  constexpr int CT = Cfg::kTiles, PT = Cfg::kParts, COLS = Cfg::kCols;

  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ uint64_t bars[NW * ST * 2];
  __shared__ int pref[NT];
  __shared__ int wsum[NW];
  __shared__ int piece_bh[2 * NW], piece_flag[2 * NW], piece_end[2 * NW];

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int c = blockIdx.x;
  const int G = p.Hq / p.Hkv;
  const int g = lane >> 2, q4 = lane & 3;
  if (tid == 0) {
    tma_prefetch_desc(&maps.k);
    tma_prefetch_desc(&maps.v);
  }
  if (tid < NW * ST * 2) mbar_init(&bars[tid], 1);
  if (tid < 2 * NW) piece_bh[tid] = -1;
  mbar_fence_init();
  pdl_wait_prior();
  pdl_launch_dependents();

  // ---- the work list: items before every thread's share of the units, and all of them
  const int units = p.block_idx ? p.B * p.Hkv : p.B;
  const int mul = p.block_idx ? 1 : p.Hkv;
  const int per = (units + NT - 1) / NT;
  int mine = 0;
  for (int u = tid * per; u < min(units, (tid + 1) * per); ++u) mine += d8_count(p, u) * mul;
  int incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) wsum[warp] = incl;
  __syncthreads();
  int before = 0, W = 0;
#pragma unroll
  for (int w = 0; w < NW; ++w) {
    if (w < warp) before += wsum[w];
    W += wsum[w];
  }
  pref[tid] = before + incl - mine;
  __syncthreads();

  const int C = max(1, min(static_cast<int>(gridDim.x), (W + min_items - 1) / min_items));
  float* work = static_cast<float*>(p.work);
  int* meta = reinterpret_cast<int*>(work + 2 * static_cast<int64_t>(gridDim.x) * Cfg::kPiece);
  const int c0 = c < C ? static_cast<int>(static_cast<int64_t>(W) * c / C) : 0;
  const int c1 = c < C ? static_cast<int>(static_cast<int64_t>(W) * (c + 1) / C) : 0;
  const int w0 = c0 + static_cast<int>(static_cast<int64_t>(c1 - c0) * warp / NW);
  const int n = c0 + static_cast<int>(static_cast<int64_t>(c1 - c0) * (warp + 1) / NW) - w0;

  float* first_piece = reinterpret_cast<float*>(smem + Cfg::kRing) + warp * Cfg::kPiece;
  float* last_piece = reinterpret_cast<float*>(smem + warp * ST * 2 * Cfg::kTile);   // on top of the warp's ring

  if (n > 0) {
    unsigned char* ring = smem + warp * ST * 2 * Cfg::kTile;
    uint64_t* bar = bars + warp * ST * 2;      // [stage][K, V]
    // items 32 i .. 32 i + 31 of this warp are in the lanes of `now`, the 32 behind them in `next`
    D8Item now = d8_item<NT>(p, pref, per, w0 + min(lane, n - 1));
    D8Item next = now;

    auto load = [&](const int i, const int base, const bool is_v) {   // item i -> its stage
      const bool far = (i >> 5) != base;
      const int bh = __shfl_sync(0xffffffffu, far ? next.bh : now.bh, i & 31);
      const int blk = __shfl_sync(0xffffffffu, far ? next.blk : now.blk, i & 31);
      const int page = __shfl_sync(0xffffffffu, far ? next.page : now.page, i & 31);
      if (lane == 0) {
        const int s = i % ST;
        uint64_t* b = &bar[2 * s + is_v];
        mbar_expect_tx(b, Cfg::kTile);
        tma_load_4d(ring + (2 * s + is_v) * Cfg::kTile, is_v ? &maps.v : &maps.k, b, 0, p.page_table ? 0 : blk * TILE,
                    bh % p.Hkv, page);
      }
    };
#pragma unroll
    for (int i = 0; i < ST; ++i)
      if (i < n) {
        load(i, 0, false);
        load(i, 0, true);
      }
    if (n > 32) next = d8_item<NT>(p, pref, per, w0 + min(32 + lane, n - 1));

    uint32_t bq[CT][KS][2];
    float cm[CT][2];                       // softmax scale / row scale of q of this thread's two columns
    float m_run[CT][2], l_run[CT][2], acc[KS][CT][4];
    int cur = -1, began = 0;

    // the piece of head `cur`: written out if it is the whole head, else kept for the join
    auto flush = [&](const bool ends, const int end_item) {
      float l[CT][2];
#pragma unroll
      for (int t = 0; t < CT; ++t)
#pragma unroll
        for (int e = 0; e < 2; ++e) l[t][e] = quadcol_sum(l_run[t][e]);
      const int64_t hq0 = static_cast<int64_t>(cur / p.Hkv) * p.Hq + (cur % p.Hkv) * G;
      if (MODE == 0) {
#pragma unroll
        for (int mt = 0; mt < KS; ++mt)
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[mt][0][i] += __shfl_xor_sync(0xffffffffu, acc[mt][0][i], 2);
      }
      float* dst = began ? last_piece : first_piece;
      if (MODE == 0 && q4 >= 2) {
        // (the columns of the low parts: their sums are in the other half)
      } else {
#pragma unroll
        for (int t = 0; t < CT; ++t)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int head = 8 * t + 2 * q4 + e;
            if (head >= G) continue;
            if (began && ends) {
              const float inv = l[t][e] == 0.f ? 0.f : __fdividef(1.f, l[t][e]);
#pragma unroll
              for (int mt = 0; mt < KS; ++mt) {
                const float a = l[t][e] == 0.f ? 0.f : acc[mt][t][e] * inv, b = l[t][e] == 0.f ? 0.f : acc[mt][t][e + 2] * inv;
                d8_store(p, hq0 + head, mt * 16 + 2 * g, a, b);
              }
              if (g == 0) p.lse[hq0 + head] = d8_lse(m_run[t][e], l[t][e]);
            } else {
#pragma unroll
              for (int mt = 0; mt < KS; ++mt)
                *reinterpret_cast<float2*>(dst + head * D + mt * 16 + 2 * g) = make_float2(acc[mt][t][e], acc[mt][t][e + 2]);
              if (g == 0) {
                dst[COLS * D + head] = m_run[t][e];
                dst[COLS * D + COLS + head] = l[t][e];
              }
            }
          }
      }
      if (!(began && ends) && lane == 0) {
        piece_bh[2 * warp + began] = cur;
        piece_flag[2 * warp + began] = began | (ends ? 2 : 0);
        piece_end[2 * warp + began] = end_item;
      }
    };

    for (int i = 0; i < n; ++i) {
      const int li = i & 31, base = i >> 5;
      if (li == 0 && i > 0) {
        now = next;
        if (i + 32 < n) next = d8_item<NT>(p, pref, per, w0 + min(i + 32 + lane, n - 1));
      }
      const int bh = __shfl_sync(0xffffffffu, now.bh, li);
      const int blk = __shfl_sync(0xffffffffu, now.blk, li);
      const int info = __shfl_sync(0xffffffffu, now.info, li);
      const int left = __shfl_sync(0xffffffffu, now.left, li);
      const float ks = __shfl_sync(0xffffffffu, now.ks, li);
      const float vs = __shfl_sync(0xffffffffu, now.vs, li);
      const int b = bh / p.Hkv, h = bh - b * p.Hkv, tok = info & 255;
      const int64_t hq0 = static_cast<int64_t>(b) * p.Hq + h * G;

      if (bh != cur) {
        cur = bh;
        began = (info >> 8) & 1;
        // Q^T as the B operand: column n = lane / 4; row k = 2 c, 2 c + 1 (+8) of a 16-step is channel
        // 4 c + 0..3 of it, the order in which ldmatrix hands a lane the codes of a K row
        float inv[CT];
#pragma unroll
        for (int t = 0; t < CT; ++t) {
          const int head = MODE == 0 ? (g & 3) : 8 * t + g;
          uint2 w[KS];
          const uint16_t* qp = p.q + b * p.q_sb + (static_cast<int64_t>(h) * G + min(head, G - 1)) * p.q_sh + 4 * q4;
#pragma unroll
          for (int s = 0; s < KS; ++s) w[s] = *reinterpret_cast<const uint2*>(qp + 16 * s);
          float x[KS][4], top = 0.f;
#pragma unroll
          for (int s = 0; s < KS; ++s) {
            if (p.q_f16) {
              const float2 lo = unpack_f16(w[s].x), hi = unpack_f16(w[s].y);
              x[s][0] = lo.x, x[s][1] = lo.y, x[s][2] = hi.x, x[s][3] = hi.y;
            } else {
              x[s][0] = bf_lo(w[s].x), x[s][1] = bf_hi(w[s].x), x[s][2] = bf_lo(w[s].y), x[s][3] = bf_hi(w[s].y);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) top = fmaxf(top, fabsf(x[s][e]));
          }
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
          // 2^k that puts the row's largest value into [2^13, 2^14); 1 for a row of zeros
          int k = top > 0.f ? 140 - static_cast<int>(__float_as_uint(top) >> 23) : 0;
          k = max(-120, min(120, k));
          const float mulq = __uint_as_float(static_cast<uint32_t>(127 + k) << 23);
          inv[t] = __uint_as_float(static_cast<uint32_t>(127 - k) << 23);
#pragma unroll
          for (int s = 0; s < KS; ++s) {
            bq[t][s][0] = head < G ? pack_f16(x[s][0] * mulq, x[s][1] * mulq) : 0u;
            bq[t][s][1] = head < G ? pack_f16(x[s][2] * mulq, x[s][3] * mulq) : 0u;
          }
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            cm[t][e] = p.scale_log2 * __shfl_sync(0xffffffffu, inv[t], (2 * q4 + e) * 4);
            m_run[t][e] = -INFINITY;
            l_run[t][e] = 0.f;
          }
#pragma unroll
          for (int mt = 0; mt < KS; ++mt)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[mt][t][e] = 0.f;
        }
      }
      if (p.blk_max) {
        // statistics of blocks that are not read: up to the previous item of the head, and behind its last one
        int prev = blk - 1, stop = blk;
        if (p.block_idx)
          prev = (info & 256) ? -1 : p.block_idx[static_cast<int64_t>(bh) * p.max_blocks + d8_count(p, bh) - left - 2];
        if (info & 512) stop = p.nb;
        for (int x = max(0, prev + 1) + lane; x < min(stop, p.nb); x += 32)
          if (x != blk)
            for (int e = 0; e < G; ++e) {
              p.blk_max[(hq0 + e) * p.nb + x] = -INFINITY;
              p.blk_sum[(hq0 + e) * p.nb + x] = 0.f;
            }
      }

      const int s = i % ST;
      const uint32_t kt = smem_u32(ring + 2 * s * Cfg::kTile), vt = kt + Cfg::kTile;
      // 16-byte chunk `ch` of row r: the tiles are swizzled over 128 bytes (D = 128) or 64 (D = 64)
      auto at = [&](const uint32_t tile, const int r, const int ch) -> uint32_t {
        if constexpr (D == 128) return tile + r * 128 + ((ch ^ (r & 7)) << 4);
        else return tile + r * 64 + ((ch ^ ((r >> 1) & 3)) << 4);
      };
      const int lrow = lane & 7, lmat = lane >> 3;

      if (!mbar_wait(&bar[2 * s], (i / ST) & 1, 0x600u + warp)) break;
      // ---- S^T = K Q^T: 4 tiles of 16 tokens x 8 columns
      float sc[CT][4][4];
#pragma unroll
      for (int t = 0; t < CT; ++t)
#pragma unroll
        for (int mt = 0; mt < 4; ++mt)
#pragma unroll
          for (int e = 0; e < 4; ++e) sc[t][mt][e] = 0.f;
#pragma unroll
      for (int s2 = 0; s2 < KS; s2 += 2) {
#pragma unroll
        for (int mt = 0; mt < 4; ++mt) {
          uint32_t r[4], a[2][4];
          ldsm_x4(r, at(kt, mt * 16 + (lmat & 1) * 8 + lrow, s2 + (lmat >> 1)));
          codes_to_f16<KIND, 0>(r[0], a[0][0], a[0][2]);
          codes_to_f16<KIND, 0>(r[1], a[0][1], a[0][3]);
          codes_to_f16<KIND, 0>(r[2], a[1][0], a[1][2]);
          codes_to_f16<KIND, 0>(r[3], a[1][1], a[1][3]);
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int t = 0; t < CT; ++t) mma_f16(sc[t][mt], a[u], bq[t][s2 + u][0], bq[t][s2 + u][1]);
        }
      }
      __syncwarp();
      if (i + ST < n) load(i + ST, base, false);

      // ---- softmax relative to the block's own maximum, joined with the running one
      uint32_t pb[CT][4][PT][2];
      float alpha[CT][2], beta[CT][2];
      bool rescale = false;
#pragma unroll
      for (int t = 0; t < CT; ++t) {
        float f[2], mb[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) f[e] = cm[t][e] * ks;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float v = -INFINITY;
#pragma unroll
          for (int mt = 0; mt < 4; ++mt) {
            float x = sc[t][mt][e] * f[e], y = sc[t][mt][e + 2] * f[e];
            if (tok < TILE) {
              if (mt * 16 + g >= tok) x = -INFINITY;
              if (mt * 16 + g + 8 >= tok) y = -INFINITY;
            }
            sc[t][mt][e] = x, sc[t][mt][e + 2] = y;
            v = fmaxf(v, fmaxf(x, y));
          }
          mb[e] = quadcol_max(v);
          const float m_new = fmaxf(m_run[t][e], mb[e]), mu = d8_safe(m_new);
          alpha[t][e] = ex2(m_run[t][e] - mu);
          beta[t][e] = ex2(mb[e] - mu);
          m_run[t][e] = m_new;
          rescale |= alpha[t][e] != 1.f;
        }
        float ls[2] = {0.f, 0.f};
#pragma unroll
        for (int mt = 0; mt < 4; ++mt) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float x = ex2(sc[t][mt][e] - (d8_safe(mb[e & 1]) - D8_PSCALE));
            sc[t][mt][e] = x;
            ls[e & 1] += x;
          }
          // P as the B operand of the output product
          const uint32_t h0 = pack_f16(sc[t][mt][0], sc[t][mt][1]), h1 = pack_f16(sc[t][mt][2], sc[t][mt][3]);
          const float2 u0 = unpack_f16(h0), u1 = unpack_f16(h1);
          const uint32_t l0 = pack_f16(sc[t][mt][0] - u0.x, sc[t][mt][1] - u0.y);
          const uint32_t l1 = pack_f16(sc[t][mt][2] - u1.x, sc[t][mt][3] - u1.y);
          if constexpr (MODE == 0) {
            pb[t][mt][0][0] = movm_t(q4 < 2 ? h0 : l0);
            pb[t][mt][0][1] = movm_t(q4 < 2 ? h1 : l1);
          } else {
            pb[t][mt][0][0] = movm_t(h0), pb[t][mt][0][1] = movm_t(h1);
            pb[t][mt][PT - 1][0] = movm_t(l0), pb[t][mt][PT - 1][1] = movm_t(l1);
          }
        }
        if (p.blk_max) {
          const float e0 = quadcol_sum(ls[0]), e1 = quadcol_sum(ls[1]);
          const int head = 8 * t + 2 * q4;
          if (g == 0 && blk >= 0 && blk < p.nb && (MODE != 0 || q4 < 2)) {
            const float down = 1.f / 8192.f;
            if (head < G) {
              p.blk_max[(hq0 + head) * p.nb + blk] = mb[0] * LN2;
              p.blk_sum[(hq0 + head) * p.nb + blk] = e0 * down;
            }
            if (head + 1 < G) {
              p.blk_max[(hq0 + head + 1) * p.nb + blk] = mb[1] * LN2;
              p.blk_sum[(hq0 + head + 1) * p.nb + blk] = e1 * down;
            }
          }
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          l_run[t][e] = l_run[t][e] * alpha[t][e] + ls[e] * beta[t][e];
          beta[t][e] *= vs;
        }
      }

      if (!mbar_wait(&bar[2 * s + 1], (i / ST) & 1, 0x620u + warp)) break;
      if (tok < TILE) {
        // V rows behind the length: their weights are zero, but zero times a NaN code is not
        unsigned char* vrow = ring + (2 * s + 1) * Cfg::kTile;
        for (int o = tok * D + lane * 16; o < TILE * D; o += 512) *reinterpret_cast<uint4*>(vrow + o) = make_uint4(0u, 0u, 0u, 0u);
        fence_proxy_async_smem();          // ordered before the next load into this stage
        __syncwarp();
      }
      // ---- O^T = alpha O^T + beta vs V^T P^T: row g of a tile is channel 2 g, row g + 8 channel 2 g + 1
      // (two adjacent codes of a token travel as one 16-bit unit through the transposing ldmatrix)
      rescale = __any_sync(0xffffffffu, rescale);
#pragma unroll
      for (int mt = 0; mt < KS; ++mt) {
        float tmp[CT][4];
#pragma unroll
        for (int t = 0; t < CT; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) tmp[t][e] = 0.f;
#pragma unroll
        for (int th = 0; th < 2; ++th) {
          uint32_t r[4];
          ldsm_x4_t(r, at(vt, th * 32 + lmat * 8 + lrow, mt));
#pragma unroll
          for (int kk = 0; kk < 2; ++kk) {
            uint32_t a[4];
            codes_to_f16<KIND, 1>(r[2 * kk], a[0], a[1]);
            codes_to_f16<KIND, 1>(r[2 * kk + 1], a[2], a[3]);
#pragma unroll
            for (int t = 0; t < CT; ++t)
#pragma unroll
              for (int u = 0; u < PT; ++u) mma_f16(tmp[t], a, pb[t][th * 2 + kk][u][0], pb[t][th * 2 + kk][u][1]);
          }
        }
#pragma unroll
        for (int t = 0; t < CT; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if (rescale) acc[mt][t][e] *= alpha[t][e & 1];
            acc[mt][t][e] += beta[t][e & 1] * tmp[t][e];
          }
      }
      __syncwarp();
      if (i + ST < n) load(i + ST, base, true);

      const bool ends = (info >> 9) & 1;
      if (ends || i + 1 == n) flush(ends, w0 + i + left);
      if (ends) cur = -1;
    }
  }

  // ---- heads without an item: zeros
  for (int bh = c * NW + warp; bh < p.B * p.Hkv; bh += gridDim.x * NW) {
    if (d8_count(p, p.block_idx ? bh : bh / p.Hkv) > 0) continue;
    const int64_t hq0 = static_cast<int64_t>(bh / p.Hkv) * p.Hq + (bh % p.Hkv) * G;
    for (int o = lane; o < G * D / 2; o += 32) d8_store(p, hq0 + o / (D / 2), 2 * (o % (D / 2)), 0.f, 0.f);
    if (lane < G) p.lse[hq0 + lane] = -INFINITY;
    if (p.blk_max)
      for (int o = lane; o < G * p.nb; o += 32) {
        p.blk_max[hq0 * p.nb + o] = -INFINITY;
        p.blk_sum[hq0 * p.nb + o] = 0.f;
      }
  }
  __syncthreads();

  // ---- join of the warps' pieces, in item order
  int next_bh = -1, next_ctas = 0;       // head that goes on in the next CTA
  for (int a = 0; a < 2 * NW;) {
    const int bh = piece_bh[a];
    if (bh < 0) {
      ++a;
      continue;
    }
    int z = a, lastp = a;                // pieces a..lastp belong to the head
    while (++z < 2 * NW) {
      if (piece_bh[z] < 0) continue;
      if (piece_bh[z] != bh) break;
      lastp = z;
    }
    const bool begins = piece_flag[a] & 1, ends = piece_flag[lastp] & 2;
    const int64_t hq0 = static_cast<int64_t>(bh / p.Hkv) * p.Hq + (bh % p.Hkv) * G;
    float* out_piece = work + (2 * static_cast<int64_t>(c) + begins) * Cfg::kPiece;
    for (int o = tid; o < G * D / 2; o += NT) {
      const int head = o / (D / 2), d0 = 2 * (o % (D / 2));
      float m = -INFINITY;
      for (int y = a; y <= lastp; ++y) {
        if (piece_bh[y] < 0) continue;
        const float* src = (y & 1) ? reinterpret_cast<float*>(smem + (y >> 1) * ST * 2 * Cfg::kTile)
                                   : reinterpret_cast<float*>(smem + Cfg::kRing) + (y >> 1) * Cfg::kPiece;
        m = fmaxf(m, src[COLS * D + head]);
      }
      const float mu = d8_safe(m);
      float l = 0.f, x0 = 0.f, x1 = 0.f;
      for (int y = a; y <= lastp; ++y) {
        if (piece_bh[y] < 0) continue;
        const float* src = (y & 1) ? reinterpret_cast<float*>(smem + (y >> 1) * ST * 2 * Cfg::kTile)
                                   : reinterpret_cast<float*>(smem + Cfg::kRing) + (y >> 1) * Cfg::kPiece;
        const float w = ex2(src[COLS * D + head] - mu);
        const float2 v = *reinterpret_cast<const float2*>(src + head * D + d0);
        l += src[COLS * D + COLS + head] * w;
        x0 += v.x * w;
        x1 += v.y * w;
      }
      if (begins && ends) {
        d8_store(p, hq0 + head, d0, l == 0.f ? 0.f : x0 / l, l == 0.f ? 0.f : x1 / l);
        if (d0 == 0) p.lse[hq0 + head] = d8_lse(m, l);
      } else {
        *reinterpret_cast<float2*>(out_piece + head * D + d0) = make_float2(x0, x1);
        if (d0 == 0) {
          out_piece[COLS * D + head] = m;
          out_piece[COLS * D + COLS + head] = l;
        }
      }
    }
    if (begins && !ends) {
      // the CTA that holds item x is the last c' with floor(W c' / C) <= x
      next_bh = bh;
      next_ctas = static_cast<int>(((static_cast<int64_t>(piece_end[lastp]) + 1) * C - 1) / W) - c;
    }
    a = z;
  }
  if (tid == 0) {
    meta[2 * c] = next_bh;
    meta[2 * c + 1] = next_ctas;
  }
}

// Heads that are spread over several CTAs: block c joins the head that begins in CTA c and goes on behind it.
template <int D, int MODE>
__global__ void __launch_bounds__(256) decode8_merge_kernel(const __grid_constant__ kvskip_decode8_params p, const int ctas) {
  using Cfg = D8Cfg<D, MODE>;
  constexpr int COLS = Cfg::kCols;
  pdl_wait_prior();
  pdl_launch_dependents();
  const int c = blockIdx.x, G = p.Hq / p.Hkv;
  const float* work = static_cast<const float*>(p.work);
  const int* meta = reinterpret_cast<const int*>(work + 2 * static_cast<int64_t>(ctas) * Cfg::kPiece);
  const int bh = meta[2 * c], more = meta[2 * c + 1];
  if (bh < 0) return;
  const int64_t hq0 = static_cast<int64_t>(bh / p.Hkv) * p.Hq + (bh % p.Hkv) * G;
  auto piece = [&](int y) { return work + (2 * static_cast<int64_t>(c + y) + (y == 0 ? 1 : 0)) * Cfg::kPiece; };
  for (int o = threadIdx.x; o < G * D / 2; o += blockDim.x) {
    const int head = o / (D / 2), d0 = 2 * (o % (D / 2));
    float m = -INFINITY;
    for (int y = 0; y <= more; ++y) m = fmaxf(m, piece(y)[COLS * D + head]);
    const float mu = d8_safe(m);
    float l = 0.f, x0 = 0.f, x1 = 0.f;
    for (int y = 0; y <= more; ++y) {
      const float* src = piece(y);
      const float w = ex2(src[COLS * D + head] - mu);
      const float2 v = *reinterpret_cast<const float2*>(src + head * D + d0);
      l += src[COLS * D + COLS + head] * w;
      x0 += v.x * w;
      x1 += v.y * w;
    }
    d8_store(p, hq0 + head, d0, l == 0.f ? 0.f : x0 / l, l == 0.f ? 0.f : x1 / l);
    if (d0 == 0) p.lse[hq0 + head] = d8_lse(m, l);
  }
}

}  // namespace kvb
