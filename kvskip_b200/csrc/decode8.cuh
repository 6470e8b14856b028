// Attention of one token per sequence over a cache of 8-bit codes with a scale per 64-token block and
// KV head:   s_t = scale * ks[blk(t)] * q . k8[t],   out = sum_t softmax(s)_t * vs[blk(t)] * v8[t].
//
// What bounds it: 2 D bytes per token and KV head against 4 G D operations, at most 32 operations a byte
// for G = 16: HBM, as long as the arithmetic stays out of the way.  The codes go to the tensor cores as
// fp16, which holds every e4m3 and int8 value exactly (converting q to 8 bits instead would lose what the
// codes keep); q is held in fp16 relative to a power of two of its own row: exactly, bf16 values down to 2^-30 of the row's
// largest, fp16 values down to 2^-27; a smaller one is rounded to a multiple of 2^-38 of it.  M is the token (scores) or the channel (output) axis and the G
// query heads of a KV head are the 8 columns of mma.m16n8k16: the tcgen05 shapes start at 64 x 8 per
// instruction but take A from shared memory or TMEM in fp16, so the converted codes would have to be
// written back there first, which costs more than the products do.
//
// Work split: the (sequence, head, block) items of the whole launch are one list, ordered by sequence,
// head and block, cut evenly into one chunk per warp.  So requests of any mixture of lengths keep every SM busy to the end
// without the host knowing a length.  A warp keeps the running maximum, sum and output of the head it is in and has its own
// stage (a K and a V tile with an mbarrier each, refilled as soon as
// its products are done): no barrier between warps anywhere.  A head that a chunk holds from its first to its last
// block is written out by the warp; other pieces (at most two per chunk) go to `work` and are joined, in item order,
// by decode8_merge_kernel.  Nothing is added in an order that depends on timing.  (Chunks taken from a counter, so that SMs
// which get less of a saturated memory do less, gained nothing: with 8 warps an SM the SMs finish within a few
// per cent of each other, with 12 they differed by a third.)
//
// P (0..1 relative to its block's maximum) goes to the tensor cores as fp16 high + low parts, which hold
// 22 bits of it: with G <= 4 the two parts share one instruction (columns 0-3 high, 4-7 low; the scores of a
// head are computed in both, which costs nothing), else they are two instructions.  P is scaled by 2^13,
// so that weights down to 2^-27 of the block's maximum are normal fp16 numbers; the factor that brings a block's sums to the
// running maximum takes the scaling out again, so that outputs up to the end of fp32 do not overflow on the way.
#pragma once
#include "common.cuh"
#include "mma.cuh"

namespace kvb {

struct D8Maps {
  CUtensorMap k, v;
};

// MODE 0: G <= 4, one column tile with high and low parts; 1: G <= 8, one tile; 2: G <= 16, two tiles.
// Warps: as many as keep the memory busy and no more, since a deeper queue in front of it is shared out unevenly between the
// SMs (batch 16 / 64k in a loop of 0.3 s, under the power cap: 346 us with 7, 330 with 8, 372 with 10, 369 with 12; batch 1 /
// 64k: 29.3, 29.5, 34.8, 40.5).  Fewer warps with two stages each are behind too, with one tile of columns at D 128 (6, 5 and 4
// of them: 349, 375, 388 us for batch 16 / 64k; 34.3, 32.5, 31.9 for batch 1): a warp's own instructions become the bound.
// D 64, whose tiles are half as large: 12 warps and 8 take 197 and 215 us for batch 16 / 64k in a loop (int8; 216 and 239 with 8
// query heads), 22.8 and 21.5 for batch 1 / 64k, 7.1 and 6.6 for batch 1 / 1k.
template <int D, int MODE>
struct D8Cfg {
  static constexpr int kCols = MODE == 0 ? 4 : MODE == 1 ? 8 : 16;   // query heads there is room for
  static constexpr int kTiles = MODE == 2 ? 2 : 1;
  static constexpr int kParts = MODE == 0 ? 1 : 2;                   // MMA instructions per P fragment
  static constexpr int kWarps = D == 64 && MODE < 2 ? 12 : 8;
  static constexpr int kThreads = kWarps * 32;
  static constexpr int kTile = TILE * D;                             // bytes of a K or V tile
  static constexpr int kQRow = 2 * D + 16;                           // bytes of a q row in shared memory, conflict-free
  static constexpr int kSmem = kWarps * (2 * kTile + kCols * kQRow) + 1024;
  static constexpr int kPiece = kCols * (D + 2);                     // floats of a piece: acc, m, l
};

constexpr float D8_PSCALE = 13.f, D8_PUNSCALE = 1.f / 8192.f;   // log2 of the scaling of P, and what undoes it

// The chunks of the work list.  Places in the list are costs: a block counts 4, and where heads are short (64 blocks on
// average) and a warp has at least four blocks, the first block of a head D8_HEAD more (q is read and converted there, and
// the output written at the end: 2.7 us per block of a long head, 3.7 us per head of one block, measured with every warp
// of a B200 at work; a ragged batch of 64 takes 45 us with it, 50 without).  A block belongs to the chunk in which it
// begins; every chunk is at least as long as the longest block, so none is empty.
constexpr int D8_COST = 4, D8_HEAD = 2;
constexpr int D8_HEAD_MIN = 4;       // blocks per warp from which on heads are counted,
constexpr int D8_HEAD_MAX = 64;      // and the mean length of a head up to which they are
struct D8Chunks {
  uint32_t head, all;                // cost of a head's beginning, of everything
  uint32_t count, size, longer;      // chunks; the first `longer` of them have cost size + 1, the others size
  __device__ __forceinline__ D8Chunks(const uint32_t W, const uint32_t heads, const uint32_t warps)
      : head(W / D8_HEAD_MIN >= warps && W / D8_HEAD_MAX < heads ? D8_HEAD : 0), all(W * D8_COST + heads * head),
        count(min(W, warps)), size(count ? all / count : 0), longer(all - size * count) {}
  __device__ __forceinline__ uint32_t edge(const uint32_t i) const { return size * i + min(i, longer); }
  __device__ __forceinline__ uint32_t of(const uint32_t x) const {
    const uint32_t split = longer * (size + 1);
    return x < split ? x / (size + 1) : longer + (x - split) / size;
  }
  // first cost of block j of a head, and the first block that begins at or behind cost r of one
  __device__ __forceinline__ uint32_t at(const uint32_t j) const { return j ? head + j * D8_COST : 0; }
  __device__ __forceinline__ uint32_t block(const uint32_t r) const {
    return r == 0 ? 0 : r <= head + D8_COST ? 1 : (r - head + D8_COST - 1) / D8_COST;
  }
};
// Layout of `work`: blocks and heads before every unit of the list, then the pieces (two per chunk).
__host__ __device__ inline int64_t d8_piece_base(const int64_t units) { return (2 * (units + 1) + 3) / 4 * 4; }

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
__device__ __forceinline__ void cp_async8(const uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_all;" ::: "memory"); }
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
  int b, blk, page;    // sequence; block; page (paged form) or sequence
  int info;            // valid tokens | first of its head << 8 | last of its head << 9 | KV head << 10
  int pos;             // place in the head's blocks
  float ks, vs;
};

// Items of one unit of the list: a sequence (all heads, every block) or, with block lists, a (sequence, head).
__device__ __forceinline__ int d8_len(const kvskip_decode8_params& p, int b) {
  return p.lens ? max(0, min(__ldcg(p.lens + b), p.T)) : p.T;
}
__device__ __forceinline__ int d8_count(const kvskip_decode8_params& p, int u) {
  if (p.block_idx) return max(0, min(__ldcg(p.block_cnt + u), p.max_blocks));
  return (d8_len(p, u) + TILE - 1) / TILE;
}

// pref[t]: blocks (x) and heads (y) before the units of thread t's share; pref[THREADS]: all of them.
// The last t with x * cx + y * cy <= key; the whole warp asks for the same key.
template <int THREADS>
__device__ __forceinline__ int d8_find(const int2* pref, const uint32_t key, const uint32_t cx, const uint32_t cy) {
  constexpr int N = THREADS / 32;
  static_assert(THREADS % 32 == 0 && N <= 32, "two rounds");
  const int lane = threadIdx.x & 31;
  auto below = [&](const int t) { return static_cast<uint32_t>(pref[t].x) * cx + static_cast<uint32_t>(pref[t].y) * cy <= key; };
  const int base = (31 - __clz(__ballot_sync(0xffffffffu, below(lane * N)))) * N;
  return base + 31 - __clz(__ballot_sync(0xffffffffu, lane < N && below(base + lane)));
}
// Number of the first block that begins at or behind cost e.
template <int THREADS>
__device__ __forceinline__ int d8_first(const kvskip_decode8_params& p, const D8Chunks& cut, const int2* pref, const int per,
                                        const uint32_t e) {
  if (cut.head == 0) return static_cast<int>((e + D8_COST - 1) / D8_COST);
  if (e >= cut.all) return pref[THREADS].x;
  const int lo = d8_find<THREADS>(pref, e, D8_COST, cut.head);
  const uint32_t mul = p.block_idx ? 1 : p.Hkv;
  uint32_t rem = e - (static_cast<uint32_t>(pref[lo].x) * D8_COST + static_cast<uint32_t>(pref[lo].y) * cut.head), cnt;
  int first = pref[lo].x;
  if (per == 1) {
    cnt = static_cast<uint32_t>(pref[lo + 1].x - first) / mul;
  } else {
    int u = lo * per;
    for (cnt = d8_count(p, u); rem >= mul * (cnt ? cnt * D8_COST + cut.head : 0); cnt = d8_count(p, ++u)) {
      rem -= mul * (cnt ? cnt * D8_COST + cut.head : 0);
      first += static_cast<int>(mul * cnt);
    }
  }
  const uint32_t one = cnt * D8_COST + cut.head, h = rem / one;
  return first + static_cast<int>(h * cnt + cut.block(rem - h * one));
}
// Block number j of the cnt blocks of KV head h of sequence b.
__device__ __forceinline__ D8Item d8_block(const kvskip_decode8_params& p, const int b, const int h, const int j, const int cnt) {
  D8Item it;
  it.blk = p.block_idx ? p.block_idx[(static_cast<int64_t>(b) * p.Hkv + h) * p.max_blocks + j] : j;
  it.b = b;
  const bool in = it.blk >= 0 && it.blk < p.nb;
  const int tok = in ? max(0, min(TILE, d8_len(p, b) - it.blk * TILE)) : 0;
  it.info = tok | (j == 0 ? 256 : 0) | (j == cnt - 1 ? 512 : 0) | (h << 10);
  it.pos = j;
  it.ks = it.vs = 0.f;
  it.page = b;
  // (a listed block behind the length has no scale: what is there may be anything.  Nothing here uses the
  // scales once they are asked for, so that the loads of the first block need not wait for them.)
  if (p.page_table) {
    it.page = in ? p.page_table[static_cast<int64_t>(b) * p.max_pages + it.blk] : -1;
    if (it.page >= 0 && it.page < p.num_pages) {
      if (tok > 0) {
        it.ks = p.k_scale[it.page * p.ks_sb + h * p.ks_sh];
        it.vs = p.v_scale[it.page * p.vs_sb + h * p.vs_sh];
      }
    } else {
      it.page = -1;                      // out of bounds for the tensor map: reads as zeros
    }
  } else if (tok > 0) {
    it.ks = p.k_scale[b * p.ks_sb + h * p.ks_sh + it.blk * p.ks_st];
    it.vs = p.v_scale[b * p.vs_sb + h * p.vs_sh + it.blk * p.vs_st];
  }
  return it;
}

// Block x of the list, for a warp whose first lane asks for block x0 <= x.
template <int THREADS>
__device__ __forceinline__ D8Item d8_item(const kvskip_decode8_params& p, const int2* pref, const int per, const int x0, const int x) {
  int lo = d8_find<THREADS>(pref, x0, 1, 0);
  if (pref[lo + 1].x <= x) {             // behind that share: the last t with pref[t].x <= x
    int hi = THREADS - 1;
    ++lo;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (pref[mid].x <= x) lo = mid; else hi = mid - 1;
    }
  }
  const uint32_t Hkv = p.Hkv;
  const int mul = p.block_idx ? 1 : p.Hkv;
  int rem = x - pref[lo].x, u = lo, cnt;
  if (per == 1) {
    cnt = pref[lo + 1].x - pref[lo].x;
    if (!p.block_idx) cnt = static_cast<int>(static_cast<uint32_t>(cnt) / Hkv);
  } else {
    u = lo * per, cnt = d8_count(p, u);
    while (rem >= cnt * mul) {
      rem -= cnt * mul;
      cnt = d8_count(p, ++u);
    }
  }
  if (p.block_idx) {
    const int b = static_cast<int>(static_cast<uint32_t>(u) / Hkv);
    return d8_block(p, b, u - b * p.Hkv, rem, cnt);
  }
  const int h = static_cast<int>(static_cast<uint32_t>(rem) / static_cast<uint32_t>(cnt));
  return d8_block(p, u, h, rem - h * cnt, cnt);
}

// Output rows: o[head][d0], [d0 + 1] of query head hq.
__device__ __forceinline__ void d8_store(const kvskip_decode8_params& p, const int64_t hq, const int d0, float a, float b) {
  uint32_t w;
  if (p.q_f16) w = pack_f16(a, b);
  else w = pack_bf16(a, b);
  *reinterpret_cast<uint32_t*>(p.out + hq * p.D + d0) = w;
  if (p.out_f32) *reinterpret_cast<float2*>(p.out_f32 + hq * p.D + d0) = make_float2(a, b);
}
// four channels of a row that is divided by its sum
__device__ __forceinline__ void d8_store4(const kvskip_decode8_params& p, const int64_t hq, const int d0, float4 x, const float l) {
  if (l == 0.f) x = make_float4(0.f, 0.f, 0.f, 0.f);
  else x.x /= l, x.y /= l, x.z /= l, x.w /= l;
  d8_store(p, hq, d0, x.x, x.y);
  d8_store(p, hq, d0 + 2, x.z, x.w);
}
__device__ __forceinline__ float d8_lse(float m, float l) {
  return l == 0.f ? -INFINITY : (m + log2f(l)) * LN2;   // (a NaN sum stays one)
}
__device__ __forceinline__ float d8_safe(float m) { return m == -INFINITY ? 0.f : m; }
// N pieces (maximum, sum, four channels) onto a sum relative to m_old, which becomes one relative to m.
template <int N>
__device__ __forceinline__ void d8_add(const float m_old, const float m, const float (&pm)[N], const float (&pl)[N],
                                       const float4 (&v)[N], float& l, float4& x) {
  const float mu = d8_safe(m), down = ex2(m_old - mu);
  l *= down;
  x.x *= down, x.y *= down, x.z *= down, x.w *= down;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float f = ex2(pm[i] - mu);
    l += pl[i] * f;
    x.x += v[i].x * f, x.y += v[i].y * f, x.z += v[i].z * f, x.w += v[i].w * f;
  }
}
// The sums of S threads (every `quads`-th from `at` on), in order; m: the first one's maximum, then that of all.
__device__ __forceinline__ void d8_join(const float4* sx, const float* sl, const float* sm, const int at, const int quads,
                                        const int S, float& m, float& l, float4& x) {
#pragma unroll 8
  for (int i = 1; i < S; ++i) m = fmaxf(m, sm[i * quads + at]);
  const float mu = d8_safe(m);
  l = 0.f, x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
  for (int i = 0; i < S; ++i) {
    const float f = ex2(sm[i * quads + at] - mu);
    const float4 v = sx[i * quads + at];
    l += sl[i * quads + at] * f;
    x.x += v.x * f, x.y += v.y * f, x.z += v.z * f, x.w += v.w * f;
  }
}
__device__ __forceinline__ float cluster_ld_f32(const uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ float4 cluster_ld_f32x4(const uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}

// SHORT: the form for few short heads, a launch as short as it gets.  A cluster of CTAs takes one head, its warps the
// head's blocks evenly; the pieces stay in shared memory and the CTAs of the cluster join a share of the output each,
// reading the others' through distributed shared memory.  No list, no second launch.
template <int KIND, int D, int MODE, bool SHORT>
__global__ void __launch_bounds__(D8Cfg<D, MODE>::kThreads, 1)
decode8_kernel(const __grid_constant__ kvskip_decode8_params p, const __grid_constant__ D8Maps maps) {
  using Cfg = D8Cfg<D, MODE>;
  constexpr int NW = Cfg::kWarps, NT = Cfg::kThreads, KS = D / 16;
  constexpr int CT = Cfg::kTiles, PT = Cfg::kParts, COLS = Cfg::kCols;

  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ uint64_t bars[NW * 2];
  __shared__ int2 pref[NT + 1];
  __shared__ int2 wsum[NW];

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int G = p.Hq / p.Hkv;
  const int g = lane >> 2, q4 = lane & 3;
  if (tid == 0) {
    tma_prefetch_desc(&maps.k);
    tma_prefetch_desc(&maps.v);
  }
  if (lane < 2) mbar_init(&bars[2 * warp + lane], 1);      // (a warp waits on its own barriers alone)
  mbar_fence_init();
  __syncwarp();
  pdl_wait_prior();
  pdl_launch_dependents();

  const int ranks = SHORT ? static_cast<int>(cluster_nctarank()) : 1, rank = SHORT ? static_cast<int>(cluster_ctarank()) : 0;
  const int bh = SHORT ? blockIdx.x / ranks : 0, bs = bh / p.Hkv, hs = bh - bs * p.Hkv;   // SHORT: the cluster's head
  const int cnt = SHORT ? d8_count(p, p.block_idx ? bh : bs) : 0;
  if (SHORT && cnt == 0) {               // (the whole cluster leaves)
    const int64_t hq0 = static_cast<int64_t>(bs) * p.Hq + hs * G;
    if (rank) return;
    for (int o = tid; o < G * (D / 4); o += NT) d8_store4(p, hq0 + o / (D / 4), 4 * (o % (D / 4)), make_float4(0.f, 0.f, 0.f, 0.f), 0.f);
    if (tid < G) p.lse[hq0 + tid] = -INFINITY;
    if (p.blk_max)
      for (int64_t o = tid; o < static_cast<int64_t>(G) * p.nb; o += NT) {
        p.blk_max[hq0 * p.nb + o] = -INFINITY;
        p.blk_sum[hq0 * p.nb + o] = 0.f;
      }
    return;
  }
  if (!SHORT && p.page_table) {
    // the page table into L2 while the lengths are on their way (128 bytes a thread: the first 4.8 MB of it with 8 warps)
    const int64_t at = (static_cast<int64_t>(blockIdx.x) * NT + tid) * 32;
    if (at < static_cast<int64_t>(p.B) * p.max_pages) asm volatile("prefetch.global.L2 [%0];" ::"l"(p.page_table + at));
  }
  // ---- the work list: blocks and heads before every thread's share of the units, and all of them
  const int units = SHORT ? 0 : p.block_idx ? p.B * p.Hkv : p.B;
  const int mul = p.block_idx ? 1 : p.Hkv;
  const int per = (units + NT - 1) / NT;
  int2 mine = make_int2(0, 0), total = make_int2(0, 0);
  if constexpr (!SHORT) {
    for (int u = tid * per; u < min(units, (tid + 1) * per); ++u) {
      const int n = d8_count(p, u);
      mine.x += n * mul, mine.y += n ? mul : 0;
    }
    int2 incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, incl.x, o), y = __shfl_up_sync(0xffffffffu, incl.y, o);
      if (lane >= o) incl.x += x, incl.y += y;
    }
    if (lane == 31) wsum[warp] = incl;
    __syncthreads();
    int2 before = make_int2(0, 0);
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const int2 t = wsum[w];
      if (w < warp) before.x += t.x, before.y += t.y;
      total.x += t.x, total.y += t.y;
    }
    pref[tid] = make_int2(before.x + incl.x - mine.x, before.y + incl.y - mine.y);
    if (tid == 0) pref[NT] = total;
    __syncthreads();
  }

  float* pieces = static_cast<float*>(p.work) + d8_piece_base(units);
  const D8Chunks cut(total.x, total.y, NW * gridDim.x);
  if (!SHORT && blockIdx.x == 0) {       // for the join: blocks and heads before every unit
    int2* out = static_cast<int2*>(p.work);
    int2 x = pref[tid];
    for (int u = tid * per; u < min(units, (tid + 1) * per); ++u) {
      out[u] = x;
      if (per > 1) {
        const int n = d8_count(p, u);
        x.x += n * mul, x.y += n ? mul : 0;
      }
    }
    if (tid == 0) out[units] = total;
  }
  // n blocks from `from` on in the lanes
  auto items = [&](const int from, const int n) {
    if constexpr (SHORT) return d8_block(p, bs, hs, from + min(lane, n - 1), cnt);
    else return d8_item<NT>(p, pref, per, from, from + min(lane, n - 1));
  };

  // neighbouring chunks on different SMs: a short list spreads over all of them
  const int chunk = SHORT ? warp * ranks + rank : warp * gridDim.x + blockIdx.x;
  int begin = 0, end = 0;                // what is left of it
  if constexpr (SHORT) {
    const int parts = NW * ranks, size = cnt / parts, longer = cnt - size * parts;
    begin = chunk * size + min(chunk, longer), end = begin + size + (chunk < longer);
  } else {
    if (static_cast<uint32_t>(chunk) < cut.count) {
      begin = d8_first<NT>(p, cut, pref, per, cut.edge(chunk));
      end = d8_first<NT>(p, cut, pref, per, cut.edge(chunk + 1));
    }
  }

  if (begin < end) {
    unsigned char* kstage = smem + warp * 2 * Cfg::kTile;
    unsigned char* vstage = kstage + Cfg::kTile;
    unsigned char* qstage = smem + NW * 2 * Cfg::kTile + warp * COLS * Cfg::kQRow;
    uint64_t* bar = bars + 2 * warp;     // K, V
    int phase = 0;
    // up to 32 items of the chunk are in the lanes of `now`, the ones behind them in `next`
    int n = min(32, end - begin), next_n = 0;
    D8Item now = items(begin, n), next = now;

    int64_t cur = -1;                    // first row of q of the head the warp is in
    int at_h = 0, at_t = 0, at_n = 0;    // head, row and page (or sequence) of the block that is loaded next
    auto load_k = [&](const D8Item& from, const int i) {
      at_h = __shfl_sync(0xffffffffu, from.info, i) >> 10;
      const int blk = __shfl_sync(0xffffffffu, from.blk, i);
      at_n = __shfl_sync(0xffffffffu, from.page, i);
      at_t = p.page_table ? 0 : blk * TILE;
      if (lane == 0) {
        mbar_expect_tx(&bar[0], Cfg::kTile);
        tma_load_4d(kstage, &maps.k, &bar[0], 0, at_t, at_h, at_n);
      }
      const int b = __shfl_sync(0xffffffffu, from.b, i);
      if (static_cast<int64_t>(b) * p.Hq + at_h * G != cur) {        // another head: its rows of q come along
        const uint16_t* src = p.q + b * p.q_sb + static_cast<int64_t>(at_h) * G * p.q_sh;
        for (int o = lane; o < G * (D / 4); o += 32)
          cp_async8(smem_u32(qstage + o / (D / 4) * Cfg::kQRow + o % (D / 4) * 8), src + o / (D / 4) * p.q_sh + o % (D / 4) * 4);
      }
    };
    auto load_v = [&]() {                // of the block whose K was loaded last
      if (lane == 0) {
        mbar_expect_tx(&bar[1], Cfg::kTile);
        tma_load_4d(vstage, &maps.v, &bar[1], 0, at_t, at_h, at_n);
      }
    };
    load_k(now, 0);
    load_v();

    uint32_t bq[CT][KS][2];
    float cm[CT][2];                       // softmax scale / row scale of q of this thread's two columns
    float m_run[CT][2], l_run[CT][2], acc[KS][CT][4];
    int began = 0;

    // the piece of head `cur`: written out if it is the whole head, else kept for the join
    auto flush = [&](const bool ends) {
      float l[CT][2];
#pragma unroll
      for (int t = 0; t < CT; ++t)
#pragma unroll
        for (int e = 0; e < 2; ++e) l[t][e] = quadcol_sum(l_run[t][e]);
      const int64_t hq0 = cur;
      if (MODE == 0) {
#pragma unroll
        for (int mt = 0; mt < KS; ++mt)
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[mt][0][i] += __shfl_xor_sync(0xffffffffu, acc[mt][0][i], 2);
        if (q4 >= 2) return;             // (the columns of the low parts: their sums are in the other half)
      }
      float* dst = SHORT ? reinterpret_cast<float*>(kstage) : pieces + (2 * static_cast<int64_t>(chunk) + began) * Cfg::kPiece;
#pragma unroll
      for (int t = 0; t < CT; ++t)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int head = 8 * t + 2 * q4 + e;
          if (head >= G) continue;
          if (!SHORT && began && ends) {
            const bool none = l[t][e] == 0.f;
            const float inv = none ? 0.f : __fdividef(1.f, l[t][e]);
#pragma unroll
            for (int mt = 0; mt < KS; ++mt)
              d8_store(p, hq0 + head, mt * 16 + 2 * g, none ? 0.f : acc[mt][t][e] * inv, none ? 0.f : acc[mt][t][e + 2] * inv);
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
    };

    int li = 0;
    for (;;) {
      if (li == 0 && begin + n < end) {
        next_n = min(32, end - begin - n);
        next = items(begin + n, next_n);
      }
      const bool last = li == n - 1;
      const int b = __shfl_sync(0xffffffffu, now.b, li);
      const int blk = __shfl_sync(0xffffffffu, now.blk, li);
      const int info = __shfl_sync(0xffffffffu, now.info, li);
      const int pos = __shfl_sync(0xffffffffu, now.pos, li);
      const float ks = __shfl_sync(0xffffffffu, now.ks, li);
      const float vs = __shfl_sync(0xffffffffu, now.vs, li);
      const int h = info >> 10, tok = info & 255;
      const int64_t hq0 = static_cast<int64_t>(b) * p.Hq + h * G;

      if (hq0 != cur) {
        cur = hq0;
        began = (info >> 8) & 1;
        // Q^T as the B operand: column n = lane / 4; row k = 2 c, 2 c + 1 (+8) of a 16-step is channel
        // 4 c + 0..3 of it, the order in which ldmatrix hands a lane the codes of a K row
        float inv[CT];
        cp_async_wait();
        __syncwarp();
#pragma unroll
        for (int t = 0; t < CT; ++t) {
          const int head = MODE == 0 ? (g & 3) : 8 * t + g;
          uint2 w[KS];
          const unsigned char* qp = qstage + min(head, G - 1) * Cfg::kQRow + 8 * q4;
#pragma unroll
          for (int s = 0; s < KS; ++s) w[s] = *reinterpret_cast<const uint2*>(qp + 32 * s);
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
          prev = (info & 256) ? -1 : p.block_idx[(static_cast<int64_t>(b) * p.Hkv + h) * p.max_blocks + pos - 1];
        if (info & 512) stop = p.nb;
        for (int x = max(0, prev + 1) + lane; x < min(stop, p.nb); x += 32)
          if (x != blk)
            for (int e = 0; e < G; ++e) {
              p.blk_max[(hq0 + e) * p.nb + x] = -INFINITY;
              p.blk_sum[(hq0 + e) * p.nb + x] = 0.f;
            }
      }

      const uint32_t kt = smem_u32(kstage), vt = kt + Cfg::kTile;
      // 16-byte chunk `ch` of row r: the tiles are swizzled over 128 bytes (D = 128) or 64 (D = 64)
      auto at = [&](const uint32_t tile, const int r, const int ch) -> uint32_t {
        if constexpr (D == 128) return tile + r * 128 + ((ch ^ (r & 7)) << 4);
        else return tile + r * 64 + ((ch ^ ((r >> 1) & 3)) << 4);
      };
      const int lrow = lane & 7, lmat = lane >> 3;

      if (!mbar_wait_warp(&bar[0], phase, 0x700u + warp)) {
        mbar_drain(&bar[1], phase);
        break;
      }
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
      if (!last) load_k(now, li + 1);
      else if (next_n > 0) load_k(next, 0);

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
          beta[t][e] = ex2(mb[e] - mu) * D8_PUNSCALE;
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
            if (head < G) {
              p.blk_max[(hq0 + head) * p.nb + blk] = mb[0] * LN2;
              p.blk_sum[(hq0 + head) * p.nb + blk] = e0 * D8_PUNSCALE;
            }
            if (head + 1 < G) {
              p.blk_max[(hq0 + head + 1) * p.nb + blk] = mb[1] * LN2;
              p.blk_sum[(hq0 + head + 1) * p.nb + blk] = e1 * D8_PUNSCALE;
            }
          }
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          l_run[t][e] = l_run[t][e] * alpha[t][e] + ls[e] * beta[t][e];
          beta[t][e] *= vs;
        }
      }

      if (!mbar_wait_warp(&bar[1], phase, 0x720u + warp)) {
        if (!last || next_n > 0) mbar_drain(&bar[0], phase ^ 1);
        break;
      }
      if (KIND == KVSKIP_KIND_E4M3 && tok < TILE) {
        // V rows behind the length: their weights are zero, but zero times a NaN code is not (int8 has none)
        for (int o = tok * D + lane * 16; o < TILE * D; o += 512) *reinterpret_cast<uint4*>(vstage + o) = make_uint4(0u, 0u, 0u, 0u);
        fence_proxy_async_smem();          // ordered before the next load into this stage
        __syncwarp();
      }
      // ---- O^T = alpha O^T + beta vs V^T P^T: row g of a tile is channel 2 g, row g + 8 channel 2 g + 1
      // (two adjacent codes of a token travel as one 16-bit unit through the transposing ldmatrix)
      if (__any_sync(0xffffffffu, rescale)) {
#pragma unroll
        for (int mt = 0; mt < KS; ++mt)
#pragma unroll
          for (int t = 0; t < CT; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[mt][t][e] *= alpha[t][e & 1];
      }
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
          for (int e = 0; e < 4; ++e) acc[mt][t][e] += beta[t][e & 1] * tmp[t][e];
      }
      __syncwarp();
      if (!last || next_n > 0) load_v();
      phase ^= 1;

      const bool ends = (info >> 9) & 1;
      if (ends || begin + li + 1 == end) flush(ends);
      if (ends) cur = -1;
      if (!last) {
        ++li;
        continue;
      }
      if (next_n == 0) break;
      now = next;
      begin += n, n = next_n;
      li = 0, next_n = 0;
    }
  }

  if constexpr (SHORT) {
    __shared__ float4 sx[NT];
    __shared__ float sl[NT], sm[NT];
    __syncwarp();
    cluster_arrive();
    cluster_wait();                      // every warp's piece is in its stage
    const int pieces_n = min(cnt, NW * ranks), all = G * (D / 4);
    const int quad0 = all * rank / ranks, quads = all * (rank + 1) / ranks - quad0;
    const int64_t hq0 = static_cast<int64_t>(bs) * p.Hq + hs * G;
    const uint32_t base = smem_u32(smem);
    const int S = quads == 0 || quads >= NT ? 1 : min(NT / quads, (pieces_n + 3) / 4);
    for (int q0 = 0; q0 < quads; q0 += NT) {
      const int s = S == 1 ? 0 : tid / quads, at = S == 1 ? q0 + tid : tid - s * quads;
      const bool on = s < S && at < quads;
      const int quad = quad0 + at, head = quad / (D / 4), d0 = 4 * (quad % (D / 4));
      float m = -INFINITY, l = 0.f;
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int c = s; on && c < pieces_n; c += 4 * S) {
        float pm[4], pl[4];
        float4 v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int y = min(c + i * S, pieces_n - 1);         // piece y: warp y / ranks of CTA y % ranks
          const uint32_t src = cluster_map(base + (y / ranks) * 2 * Cfg::kTile, y % ranks);
          pm[i] = cluster_ld_f32(src + (COLS * D + head) * 4);
          pl[i] = cluster_ld_f32(src + (COLS * D + COLS + head) * 4);
          v[i] = cluster_ld_f32x4(src + (head * D + d0) * 4);
        }
        const float m_old = m;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (c + i * S >= pieces_n) pm[i] = -INFINITY, pl[i] = 0.f, v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
          m = fmaxf(m, pm[i]);
        }
        d8_add<4>(m_old, m, pm, pl, v, l, x);
      }
      if (S > 1) {
        sx[tid] = x, sl[tid] = l, sm[tid] = m;
        __syncthreads();
        if (s == 0 && on) d8_join(sx, sl, sm, at, quads, S, m, l, x);
      }
      if (s == 0 && on) {
        d8_store4(p, hq0 + head, d0, x, l);
        if (d0 == 0) p.lse[hq0 + head] = d8_lse(m, l);
      }
    }
    __syncwarp();
    cluster_arrive();
    cluster_wait();                      // nobody leaves while its pieces are read
  }
}

// The join: block (bh, y) does its share of the output of KV head bh, if the head's items lie in more than one chunk, or
// writes the zeros of a head without items.  A thread has four channels of a query head (a quad) and every S-th piece,
// eight pieces in flight; the S sums are added in order.
constexpr int D8_MERGE_THREADS = 256;
template <int D, int MODE>
__global__ void __launch_bounds__(D8_MERGE_THREADS)
decode8_merge_kernel(const __grid_constant__ kvskip_decode8_params p, const int warps) {
  using Cfg = D8Cfg<D, MODE>;
  constexpr int COLS = Cfg::kCols, L = D / 4, NT = D8_MERGE_THREADS;
  __shared__ float4 sx[NT];
  __shared__ float sl[NT], sm[NT];
  __shared__ int2 wsum[NT / 32], span[2];
  const int bh = blockIdx.x, G = p.Hq / p.Hkv, tid = threadIdx.x, lane = tid & 31;
  const int units = p.block_idx ? p.B * p.Hkv : p.B;
  const int b = bh / p.Hkv, u = p.block_idx ? bh : b, mul = p.block_idx ? 1 : p.Hkv;
  int2 first, next, total;               // blocks and heads before the unit, behind it, in all
  if (units <= NT) {
    // Before the wait: the lengths are older than the kernel this one waits for (which let this one begin only after
    // its own wait), so the place of the head in the list can be had while that one is at work.
    const int n = tid < units ? d8_count(p, tid) : 0;
    int2 incl = make_int2(n * mul, n ? mul : 0);
    const int2 mine = incl;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, incl.x, o), y = __shfl_up_sync(0xffffffffu, incl.y, o);
      if (lane >= o) incl.x += x, incl.y += y;
    }
    if (lane == 31) wsum[tid >> 5] = incl;
    __syncthreads();
    total = make_int2(0, 0);
#pragma unroll
    for (int w = 0; w < NT / 32; ++w) {
      const int2 t = wsum[w];
      if (w < (tid >> 5)) incl.x += t.x, incl.y += t.y;
      total.x += t.x, total.y += t.y;
    }
    if (tid == u) span[0] = make_int2(incl.x - mine.x, incl.y - mine.y), span[1] = incl;
    __syncthreads();
    first = span[0], next = span[1];
  } else {
    pdl_wait_prior();
    const int2* pref = static_cast<const int2*>(p.work);
    first = pref[u], next = pref[u + 1], total = pref[units];
  }
  const uint32_t count = static_cast<uint32_t>(next.x - first.x) / static_cast<uint32_t>(mul);
  const D8Chunks cut(total.x, total.y, warps);
  int c0 = 0, c1 = 0;
  if (count) {
    const uint32_t h = p.block_idx ? 0 : bh - b * p.Hkv;
    const uint32_t at = static_cast<uint32_t>(first.x) * D8_COST + static_cast<uint32_t>(first.y) * cut.head + h * (count * D8_COST + cut.head);
    c0 = static_cast<int>(cut.of(at)), c1 = static_cast<int>(cut.of(at + cut.at(count - 1)));
  }
  pdl_wait_prior();
  pdl_launch_dependents();
  const int64_t hq0 = static_cast<int64_t>(b) * p.Hq + (bh - b * p.Hkv) * G;
  const int quad0 = G * L * blockIdx.y / gridDim.y, quads = G * L * (blockIdx.y + 1) / gridDim.y - quad0;
  if (count == 0) {
    for (int o = tid; o < quads; o += NT) d8_store4(p, hq0 + (quad0 + o) / L, 4 * ((quad0 + o) % L), make_float4(0.f, 0.f, 0.f, 0.f), 0.f);
    if (blockIdx.y) return;
    if (tid < G) p.lse[hq0 + tid] = -INFINITY;
    if (p.blk_max)
      for (int64_t o = tid; o < static_cast<int64_t>(G) * p.nb; o += NT) {
        p.blk_max[hq0 * p.nb + o] = -INFINITY;
        p.blk_sum[hq0 * p.nb + o] = 0.f;
      }
    return;
  }
  if (c0 == c1) return;                  // written by the warp that had it
  // the first piece begins the head, the others go on from a chunk's beginning
  const float* pieces = static_cast<const float*>(p.work) + d8_piece_base(units);
  const int S = quads >= NT ? 1 : min(NT / quads, (c1 - c0 + 8) / 8);
  for (int q0 = 0; q0 < quads; q0 += NT) {
    const int s = S == 1 ? 0 : tid / quads, at = S == 1 ? q0 + tid : tid - s * quads;
    const bool on = s < S && at < quads;
    const int quad = quad0 + at, head = quad / L, d0 = 4 * (quad % L);
    float m = -INFINITY, l = 0.f;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int c = c0 + s; on && c <= c1; c += 8 * S) {
      float pm[8], pl[8];
      float4 v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int y = min(c + i * S, c1);
        const float* src = pieces + (2 * static_cast<int64_t>(y) + (y == c0 ? 1 : 0)) * Cfg::kPiece;
        pm[i] = src[COLS * D + head];
        pl[i] = src[COLS * D + COLS + head];
        v[i] = *reinterpret_cast<const float4*>(src + head * D + d0);
      }
      const float m_old = m;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (c + i * S > c1) pm[i] = -INFINITY, pl[i] = 0.f, v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        m = fmaxf(m, pm[i]);
      }
      d8_add<8>(m_old, m, pm, pl, v, l, x);
    }
    if (S > 1) {
      sx[tid] = x, sl[tid] = l, sm[tid] = m;
      __syncthreads();
      if (s == 0 && on) d8_join(sx, sl, sm, at, quads, S, m, l, x);
    }
    if (s == 0 && on) {
      d8_store4(p, hq0 + head, d0, x, l);
      if (d0 == 0) p.lse[hq0 + head] = d8_lse(m, l);
    }
  }
}

}  // namespace kvb
