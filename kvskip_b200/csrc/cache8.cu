// C entry points of the 8-bit cache (see include/kvskip_b200.h): attention, write, page tables.
// A translation unit of its own, compiled beside kvskip_b200.cu.
#include "../../include/kvskip_b200.h"

#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <initializer_list>

#include "host.h"
#include "common.cuh"
#include "decode8.cuh"
#include "write8.cuh"
#include "pages.cuh"

namespace {

using kvb_host::fail;

#define KVB_CUDA(expr)                                                                       \
  do {                                                                                       \
    cudaError_t e_ = (expr);                                                                 \
    if (e_ != cudaSuccess) return fail(KVSKIP_E_CUDA, "%s: %s", #expr, cudaGetErrorString(e_)); \
  } while (0)

// Programmatic dependent launch: every kernel here waits for its predecessor before it touches global memory.
template <typename... KArgs, typename... Args>
cudaError_t launch_cluster(void (*kernel)(KArgs...), dim3 grid, int threads, unsigned cluster, size_t smem, cudaStream_t stream,
                           Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = kvb_host::use_pdl() ? 1 : 0;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<KArgs>(args)...);
}
template <typename... KArgs, typename... Args>
cudaError_t launch(void (*kernel)(KArgs...), dim3 grid, int threads, size_t smem, cudaStream_t stream, Args&&... args) {
  return launch_cluster(kernel, grid, threads, 0, smem, stream, static_cast<Args&&>(args)...);
}

bool misaligned(const void* p, unsigned n) { return reinterpret_cast<uintptr_t>(p) % n != 0; }

// Map over [n,Hkv,rows,D] codes; one box is 64 rows of one head, swizzled over the row's D bytes.
int make_map(CUtensorMap* map, const uint8_t* base, int64_t sb, int64_t sh, int64_t st, int n, int Hkv, int rows, int D) {
  const auto enc = kvb_host::encode_tiled();
  if (!enc) return fail(KVSKIP_E_CUDA, "cuTensorMapEncodeTiled is not available from this driver");
  // a dim of size 1 may carry any stride (0 too): give the map a valid one
  if (rows == 1 && st < D) st = D;
  if (Hkv == 1 && sh <= 0) sh = static_cast<int64_t>(rows) * st;
  if (n == 1 && sb <= 0) sb = static_cast<int64_t>(Hkv) * sh;
  if (st <= 0 || sh <= 0 || sb <= 0) return fail(KVSKIP_E_ARG, "decode8: k / v strides must be positive");
  const cuuint64_t gdim[4] = {static_cast<cuuint64_t>(D), static_cast<cuuint64_t>(rows), static_cast<cuuint64_t>(Hkv),
                              static_cast<cuuint64_t>(n)};
  const cuuint64_t gstr[3] = {static_cast<cuuint64_t>(st), static_cast<cuuint64_t>(sh), static_cast<cuuint64_t>(sb)};
  const cuuint32_t box[4] = {static_cast<cuuint32_t>(D), KVSKIP_TILE, 1, 1};
  const cuuint32_t est[4] = {1, 1, 1, 1};
  const CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, const_cast<uint8_t*>(base), gdim, gstr, box, est,
                         CU_TENSOR_MAP_INTERLEAVE_NONE, D == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return fail(KVSKIP_E_CUDA, "cuTensorMapEncodeTiled failed (%d) for strides %lld/%lld/%lld dims %d/%d/%d/%d",
                static_cast<int>(r), static_cast<long long>(sb), static_cast<long long>(sh), static_cast<long long>(st), n,
                Hkv, rows, D);
  return KVSKIP_OK;
}

// What of a launch follows from the bound on its items (the lengths are on the device).
struct Decode8Launch {
  int ctas, warps, cluster;            // cluster: CTAs per head of the short form, 0 where that is not taken
};
// Blocks per warp up to which the short form is taken when its CTAs are most of the SMs, and when they are fewer.  The
// lengths are on the device: with one bound on them for all, a longer form would leave SMs idle when they differ.
// B200, us in a graph, general and short form, 8 KV heads: D 128, batch 1 / 1k 9.0 and 7.7, 4k 9.2 and 8.9, 8k 10.2 and 11.3; batch 4 /
// 4k 12.9 and 12.1, batch 16 / 2k 19.1 and 17.0.  D 64, batch 1 / 1k 8.0 and 6.7, 4k 8.6 and 7.5, 8k 9.2 and 9.2, 12k 10.2 and
// 10.4; batch 4 / 4k 11.0 and 9.1, batch 16 / 2k 13.6 and 11.7.
// That the CTAs are at most as many as the SMs does not make them one wave: a cluster stays inside a GPC, and the GPCs do not
// divide evenly.  16 to 18 heads in clusters of 8 take two (4k: 16.7 to 17.0, the general form 9.9 to 10.2), 36 and 37 heads
// in clusters of 4 too (2k: 16.1 to 16.3, 10.2 to 10.3); 32 and 33 heads in clusters of 4 do not (8.8 and 8.9, 10.0).
constexpr int kShortMost = 4, kShortFew = 2;
template <int D, int MODE>
Decode8Launch decode8_launch(const kvskip_decode8_params& p) {
  const int64_t items = static_cast<int64_t>(p.B) * p.Hkv * (p.block_idx ? p.max_blocks : p.nb);
  Decode8Launch l;
  l.ctas = static_cast<int>(std::min<int64_t>(kvb_host::num_sms(), items));
  l.warps = l.ctas * kvb::D8Cfg<D, MODE>::kWarps;
  // the short form: as many CTAs per head as leave four blocks to each of them, no more than SMs in all
  constexpr int kWarps = kvb::D8Cfg<D, MODE>::kWarps;
  const int64_t heads = static_cast<int64_t>(p.B) * p.Hkv, longest = p.block_idx ? p.max_blocks : p.nb;
  int c = 1;
  while (c < 8 && 4 * c < longest && heads * 2 * c <= kvb_host::num_sms()) c *= 2;
  const bool most = 4 * heads * c >= 3 * kvb_host::num_sms();
  l.cluster = 0;
  // (not for more than 8 query heads: the pieces are four times as large, and joining them so took longer)
  if (MODE < 2 && heads * c <= kvb_host::num_sms() && longest <= static_cast<int64_t>(most ? kShortMost : kShortFew) * c * kWarps)
    l.cluster = c;
  return l;
}
template <int D, int MODE>
int64_t decode8_work(const kvskip_decode8_params& p) {
  const Decode8Launch l = decode8_launch<D, MODE>(p);
  if (l.cluster) return 16;
  const int64_t units = p.block_idx ? static_cast<int64_t>(p.B) * p.Hkv : p.B;
  return (kvb::d8_piece_base(units) + 2 * static_cast<int64_t>(l.warps) * kvb::D8Cfg<D, MODE>::kPiece) *
         static_cast<int64_t>(sizeof(float));
}

template <int KIND, int D, int MODE>
int launch_decode8(const kvskip_decode8_params& p, const kvb::D8Maps& maps, cudaStream_t stream) {
  using Cfg = kvb::D8Cfg<D, MODE>;
  const Decode8Launch l = decode8_launch<D, MODE>(p);
  if constexpr (MODE < 2) {
    if (l.cluster) {
      auto kernel = kvb::decode8_kernel<KIND, D, MODE, true>;
      if (int rc = kvb_host::ensure_smem(reinterpret_cast<const void*>(kernel), Cfg::kSmem)) return rc;
      KVB_CUDA(launch_cluster(kernel, dim3(static_cast<unsigned>(p.B) * p.Hkv * l.cluster), Cfg::kThreads,
                              static_cast<unsigned>(l.cluster), Cfg::kSmem, stream, p, maps));
      return KVSKIP_OK;
    }
  }
  auto kernel = kvb::decode8_kernel<KIND, D, MODE, false>;
  if (int rc = kvb_host::ensure_smem(reinterpret_cast<const void*>(kernel), Cfg::kSmem)) return rc;
  KVB_CUDA(launch(kernel, dim3(l.ctas), Cfg::kThreads, Cfg::kSmem, stream, p, maps));
  // few heads: the output of one goes to several blocks, of 8 quads at least
  const int quads = p.Hq / p.Hkv * D / 4, heads = p.B * p.Hkv;
  const int y = std::max(1, std::min(quads / 8, 2 * kvb_host::num_sms() / heads));
  KVB_CUDA(launch(kvb::decode8_merge_kernel<D, MODE>, dim3(heads, y), kvb::D8_MERGE_THREADS, 0, stream, p, l.warps));
  return KVSKIP_OK;
}

template <int KIND, int D>
int by_group(const kvskip_decode8_params& p, const kvb::D8Maps& maps, cudaStream_t s) {
  const int G = p.Hq / p.Hkv;
  if (G <= 4) return launch_decode8<KIND, D, 0>(p, maps, s);
  if (G <= 8) return launch_decode8<KIND, D, 1>(p, maps, s);
  return launch_decode8<KIND, D, 2>(p, maps, s);
}

// Map over the new tokens: (D, inner, Hkv, outer), boxes of 16 rows.  False where a stride has no place in one.
bool token_map(CUtensorMap* map, const kvskip_write8_params& p, const uint16_t* x, int64_t so, int64_t si, int64_t sh) {
  const auto enc = kvb_host::encode_tiled();
  const int64_t outer = p.n / p.inner;
  if (p.inner == 1) si = p.D;
  if (p.Hkv == 1) sh = p.D;
  if (outer == 1) so = p.D;
  if (!enc || si <= 0 || sh <= 0 || so <= 0) return false;
  const cuuint64_t gdim[4] = {static_cast<cuuint64_t>(p.D), static_cast<cuuint64_t>(p.inner), static_cast<cuuint64_t>(p.Hkv),
                              static_cast<cuuint64_t>(outer)};
  const cuuint64_t gstr[3] = {static_cast<cuuint64_t>(si) * 2, static_cast<cuuint64_t>(sh) * 2, static_cast<cuuint64_t>(so) * 2};
  const cuuint32_t box[4] = {static_cast<cuuint32_t>(p.D), 16, 1, 1}, est[4] = {1, 1, 1, 1};
  return enc(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<uint16_t*>(x), gdim, gstr, box, est,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int KIND, int D, bool F16, int CHUNK>
int launch_write8(const kvskip_write8_params& p, cudaStream_t s) {
  using Cfg = kvb::W8Cfg<D, CHUNK>;
  auto kernel = kvb::write8_kernel<KIND, D, CHUNK, F16>;
  if (int rc = kvb_host::ensure_smem(reinterpret_cast<const void*>(kernel), Cfg::kSmem)) return rc;
  kvb::W8Maps maps{};
  const bool tma = token_map(&maps.k, p, p.k_new, p.kn_so, p.kn_si, p.kn_sh) &&
                   token_map(&maps.v, p, p.v_new, p.vn_so, p.vn_si, p.vn_sh);
  const int64_t jobs = (p.n + CHUNK - 1) / CHUNK * 2 * p.Hkv;
  const int64_t ctas = std::min<int64_t>((jobs + Cfg::kWarps - 1) / Cfg::kWarps, kvb_host::num_sms() * (227 * 1024 / Cfg::kSmem));
  KVB_CUDA(launch(kernel, dim3(static_cast<unsigned>(ctas)), Cfg::kThreads, Cfg::kSmem, s, p, maps, static_cast<int>(jobs),
                  tma ? 1 : 0));
  return KVSKIP_OK;
}

template <int KIND, int D, bool F16>
int by_chunk(const kvskip_write8_params& p, cudaStream_t s) {
  // The slots of a warp: 64, or fewer where every warp of the GPU would not get a job, so that the tokens of a decode
  // step spread over it.  B200, us in a graph, 8 heads, with 4 and with 16: 64 tokens 3.1 and 9.1, 256 3.8 and 9.3, 512 6.0 and 9.3,
  // 1024 10.3 and 9.4, 1700 15.0 and 9.5 (with 4 the last tokens wait for a place: 6 CTAs fit on an SM, one less than the grid
  // counts on); prompts of 54k tokens with 64: 60.
  const int64_t warps = static_cast<int64_t>(kvb_host::num_sms()) * kvb::W8Cfg<D, 64>::kWarps, pairs = 2 * p.Hkv;
  if ((p.n + 63) / 64 * pairs >= warps) return launch_write8<KIND, D, F16, 64>(p, s);
  if ((p.n + 15) / 16 * pairs >= warps) return launch_write8<KIND, D, F16, 16>(p, s);
  return launch_write8<KIND, D, F16, 4>(p, s);
}

template <int KIND, int D>
int by_type(const kvskip_write8_params& p, cudaStream_t s) {
  return p.x_f16 ? by_chunk<KIND, D, true>(p, s) : by_chunk<KIND, D, false>(p, s);
}

// CTAs for `n` table or slot entries (200k slots, B200: 7.7 us with 4096 of them per CTA, 6.2 with 2048, 5.5 with 1024)
int pages_grid(int64_t n) {
  return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(kvb_host::num_sms(), n / 1024)));
}

int check_pages(const kvskip_pages_params* p, const char* who) {
  if (!p) return fail(KVSKIP_E_ARG, "null parameter block");
  if (!p->lens || !p->table || !p->free_pages || !p->n_free || !p->lens_out || !p->n_free_out)
    return fail(KVSKIP_E_ARG, "%s: lens, table, free_pages, n_free, lens_out and n_free_out are required", who);
  if (p->B < 1 || p->max_pages < 1 || p->num_free < 1) return fail(KVSKIP_E_ARG, "%s: B, max_pages, num_free >= 1", who);
  if (p->max_pages > kvb::PG_MOST_PAGES || p->num_free >= 1 << 30)
    return fail(KVSKIP_E_LIMIT, "%s: at most 2^26 tokens per request, less than 2^30 pages", who);
  return KVSKIP_OK;
}

// A stretch of memory that a call reads or writes; `same`: it may be that other one, exactly.
struct Span {
  const char* name;
  const void* at;
  int64_t bytes;
  const void* same = nullptr;
};
// The blocks of a launch run at the same time: what one writes must not be what another reads or writes.
int check_apart(const char* who, std::initializer_list<Span> written, std::initializer_list<Span> read) {
  const auto meet = [](const Span& a, const Span& b) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a.at), y = reinterpret_cast<uintptr_t>(b.at);
    return a.at && b.at && a.bytes > 0 && b.bytes > 0 && x < y + static_cast<uintptr_t>(b.bytes) && y < x + static_cast<uintptr_t>(a.bytes);
  };
  for (const Span* w = written.begin(); w != written.end(); ++w) {
    for (const Span* o = w + 1; o != written.end(); ++o)
      if (meet(*w, *o)) return fail(KVSKIP_E_ARG, "%s: %s and %s overlap", who, w->name, o->name);
    for (const Span& r : read)
      if (meet(*w, r) && !(w->same == r.at && w->at == r.at && w->bytes == r.bytes))
        return fail(KVSKIP_E_ARG, "%s: %s and %s overlap", who, w->name, r.name);
  }
  return KVSKIP_OK;
}

}  // namespace

namespace kvb_host {
int cache8_status(unsigned int* status) {
  KVB_CUDA(cudaMemcpyFromSymbol(status, kvb::g_status, sizeof(unsigned int)));
  if (*status) {
    const unsigned int zero = 0;
    KVB_CUDA(cudaDeviceSynchronize());
    KVB_CUDA(cudaMemcpyToSymbol(kvb::g_status, &zero, sizeof(zero)));
  }
  return KVSKIP_OK;
}
}  // namespace kvb_host

extern "C" {

int64_t kvskip_decode8_work_bytes(const kvskip_decode8_params* p) {
  if (!p || p->B < 1 || p->Hkv < 1 || p->Hq < p->Hkv || p->D < 1 || p->nb < 1 || (p->block_idx && p->max_blocks < 1)) return 0;
  const int G = p->Hq / p->Hkv, mode = G <= 4 ? 0 : G <= 8 ? 1 : 2;
  if (p->D == 128)
    return mode == 0 ? decode8_work<128, 0>(*p) : mode == 1 ? decode8_work<128, 1>(*p) : decode8_work<128, 2>(*p);
  return mode == 0 ? decode8_work<64, 0>(*p) : mode == 1 ? decode8_work<64, 1>(*p) : decode8_work<64, 2>(*p);
}

int kvskip_launch_decode8(const kvskip_decode8_params* p, void* stream) {
  if (!p) return fail(KVSKIP_E_ARG, "null parameter block");
  if (p->D != 64 && p->D != 128) return fail(KVSKIP_E_ARG, "decode8: head dim 64 or 128");
  if (p->kind != KVSKIP_KIND_E4M3 && p->kind != KVSKIP_KIND_INT8) return fail(KVSKIP_E_ARG, "decode8: kind 0 (e4m3) or 1 (int8)");
  if (p->B < 1 || p->Hkv < 1 || p->T < 1 || p->Hq < 1 || p->Hq % p->Hkv) return fail(KVSKIP_E_ARG, "decode8: bad B / Hq / Hkv / T");
  if (p->Hq / p->Hkv > 16) return fail(KVSKIP_E_ARG, "decode8: at most 16 query heads per KV head");
  if (p->Hkv > 1 << 20) return fail(KVSKIP_E_LIMIT, "decode8: more than 2^20 KV heads");
  if (!p->q || !p->k || !p->v || !p->k_scale || !p->v_scale || !p->out || !p->lse || !p->work)
    return fail(KVSKIP_E_ARG, "decode8: q, k, v, k_scale, v_scale, out, lse and work are required");
  if (p->nb != (p->T - 1) / KVSKIP_TILE + 1) return fail(KVSKIP_E_ARG, "decode8: nb must be ceil(T / 64)");
  if ((p->block_idx == nullptr) != (p->block_cnt == nullptr) || (p->block_idx && p->max_blocks < 1))
    return fail(KVSKIP_E_ARG, "decode8: block_idx, block_cnt and max_blocks go together");
  if ((p->blk_max == nullptr) != (p->blk_sum == nullptr)) return fail(KVSKIP_E_ARG, "decode8: blk_max and blk_sum go together");
  if (p->page_table && (p->num_pages < 1 || p->max_pages < p->nb))
    return fail(KVSKIP_E_ARG, "paged cache: the page table needs an entry for every block of the sequence");
  if (p->page_table && !p->lens) return fail(KVSKIP_E_ARG, "decode8: a paged cache needs lens");
  if (misaligned(p->q, 8) || p->q_sb % 4 || p->q_sh % 4) return fail(KVSKIP_E_ARG, "decode8: q rows must be 8-byte aligned");
  if (misaligned(p->out, 4) || misaligned(p->out_f32, 8) || misaligned(p->work, 16))
    return fail(KVSKIP_E_ARG, "decode8: misaligned out / out_f32 / work");
  if (misaligned(p->k, 16) || misaligned(p->v, 16) || (p->k_sb | p->k_sh | p->k_st | p->v_sb | p->v_sh | p->v_st) % 16)
    return fail(KVSKIP_E_ARG, "decode8: k / v must be 16-byte aligned, with strides that are multiples of 16");
  if (static_cast<int64_t>(p->B) * p->Hkv * (p->block_idx ? std::max(p->max_blocks, p->nb) : p->nb) > 1 << 29 ||
      static_cast<int64_t>(p->B) * p->Hq > 2147483647LL)
    return fail(KVSKIP_E_LIMIT, "decode8: more than 2^29 blocks of heads in a call");
  kvb::D8Maps maps;
  const int n = p->page_table ? p->num_pages : p->B, rows = p->page_table ? KVSKIP_TILE : p->T;
  if (int rc = make_map(&maps.k, p->k, p->k_sb, p->k_sh, p->k_st, n, p->Hkv, rows, p->D)) return rc;
  if (int rc = make_map(&maps.v, p->v, p->v_sb, p->v_sh, p->v_st, n, p->Hkv, rows, p->D)) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (p->kind == KVSKIP_KIND_E4M3)
    return p->D == 128 ? by_group<KVSKIP_KIND_E4M3, 128>(*p, maps, s) : by_group<KVSKIP_KIND_E4M3, 64>(*p, maps, s);
  return p->D == 128 ? by_group<KVSKIP_KIND_INT8, 128>(*p, maps, s) : by_group<KVSKIP_KIND_INT8, 64>(*p, maps, s);
}

int kvskip_launch_write8(const kvskip_write8_params* p, void* stream) {
  if (!p) return fail(KVSKIP_E_ARG, "null parameter block");
  if (p->D != 64 && p->D != 128) return fail(KVSKIP_E_ARG, "write8: head dim 64 or 128");
  if (p->kind != KVSKIP_KIND_E4M3 && p->kind != KVSKIP_KIND_INT8) return fail(KVSKIP_E_ARG, "write8: kind 0 (e4m3) or 1 (int8)");
  if (p->n < 0 || p->inner < 1 || p->n % p->inner || p->Hkv < 1 || p->blocks < 1 || p->tokens < 1 || p->num_blocks < 1)
    return fail(KVSKIP_E_ARG, "write8: bad n / inner / Hkv / blocks / tokens / num_blocks");
  if (p->n == 0) return KVSKIP_OK;
  if (!p->k_new || !p->v_new || !p->slots || !p->k || !p->v || !p->k_scale || !p->v_scale)
    return fail(KVSKIP_E_ARG, "write8: k_new, v_new, slots, k, v, k_scale and v_scale are required");
  if (misaligned(p->k_new, 16) || misaligned(p->v_new, 16) ||
      (p->kn_so | p->kn_si | p->kn_sh | p->vn_so | p->vn_si | p->vn_sh) % 8)
    return fail(KVSKIP_E_ARG, "write8: rows of k_new and v_new must be 16-byte aligned");
  if (misaligned(p->k, 8) || misaligned(p->v, 8) || (p->k_sb | p->k_sh | p->k_st | p->v_sb | p->v_sh | p->v_st) % 8)
    return fail(KVSKIP_E_ARG, "write8: rows of k and v must be 8-byte aligned");
  if (p->Hkv > 65535 || p->n > 2147483647LL - 64 || (p->n + 3) / 4 * 2 * p->Hkv > 1073741823LL)
    return fail(KVSKIP_E_LIMIT, "write8: grid limits exceeded (tokens, heads)");
  // K and V are written at the same time, and so are the heads and blocks of each
  if (p->k == p->v || p->k_scale == p->v_scale) return fail(KVSKIP_E_ARG, "write8: k and v, or their scales, are the same memory");
  const bool seqs = p->num_blocks > p->blocks, heads = p->Hkv > 1, blks = p->blocks > 1;
  if ((seqs && (!p->k_sb || !p->v_sb || !p->ks_sb || !p->vs_sb)) || (heads && (!p->k_sh || !p->v_sh || !p->ks_sh || !p->vs_sh)) ||
      (blks && (!p->ks_st || !p->vs_st)) || (p->tokens > 1 && (!p->k_st || !p->v_st)))
    return fail(KVSKIP_E_ARG, "write8: a stride of 0 in k, v or their scales: several tokens or blocks in one place");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (p->kind == KVSKIP_KIND_E4M3)
    return p->D == 128 ? by_type<KVSKIP_KIND_E4M3, 128>(*p, s) : by_type<KVSKIP_KIND_E4M3, 64>(*p, s);
  return p->D == 128 ? by_type<KVSKIP_KIND_INT8, 128>(*p, s) : by_type<KVSKIP_KIND_INT8, 64>(*p, s);
}

int kvskip_launch_extend_pages(const kvskip_pages_params* p, void* stream) {
  if (int rc = check_pages(p, "extend_pages")) return rc;
  if (!p->new_ || !p->granted || (p->n_tokens > 0 && (!p->slots || !p->positions)))
    return fail(KVSKIP_E_ARG, "extend_pages: new, granted, slots and positions are required");
  if (p->n_tokens < 0 || p->per_row < 0 || (p->per_row > 0 && p->n_tokens != static_cast<int64_t>(p->per_row) * p->B))
    return fail(KVSKIP_E_ARG, "extend_pages: n_tokens >= 0, and B * per_row of them in a padded list");
  const int64_t B = p->B;
  if (int rc = check_apart("extend_pages",
                           {{"lens_out", p->lens_out, 4 * B, p->lens}, {"n_free_out", p->n_free_out, 4, p->n_free},
                            {"table", p->table, 4 * B * p->max_pages}, {"slots", p->slots, 8 * p->n_tokens},
                            {"positions", p->positions, 4 * p->n_tokens}, {"granted", p->granted, B}},
                           {{"lens", p->lens, 4 * B}, {"n_free", p->n_free, 4}, {"new", p->new_, 4 * B},
                            {"free_pages", p->free_pages, 4LL * p->num_free}}))
    return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int grid = pages_grid(p->n_tokens);
  const bool in_place = p->lens_out == p->lens || p->n_free_out == p->n_free;
  const int one = grid == 1 || !in_place;       // several CTAs read lens and n_free: they change in a launch behind
  KVB_CUDA(launch(kvb::extend_pages_kernel, dim3(grid), kvb::PG_THREADS, 0, s, *p, 1, one));
  if (!one) KVB_CUDA(launch(kvb::extend_pages_kernel, dim3(1), kvb::PG_THREADS, 0, s, *p, 0, 1));
  return KVSKIP_OK;
}

int kvskip_launch_release_pages(const kvskip_pages_params* p, void* stream) {
  if (int rc = check_pages(p, "release_pages")) return rc;
  if (!p->done) return fail(KVSKIP_E_ARG, "release_pages: done is required");
  const int64_t B = p->B;
  if (int rc = check_apart("release_pages",
                           {{"lens_out", p->lens_out, 4 * B, p->lens}, {"n_free_out", p->n_free_out, 4, p->n_free},
                            {"free_pages", p->free_pages, 4LL * p->num_free}},
                           {{"lens", p->lens, 4 * B}, {"n_free", p->n_free, 4}, {"done", p->done, B},
                            {"table", p->table, 4 * B * p->max_pages}}))
    return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int grid = pages_grid(static_cast<int64_t>(p->B) * p->max_pages / 8);
  const bool in_place = p->lens_out == p->lens || p->n_free_out == p->n_free;
  const int one = grid == 1 || !in_place;
  KVB_CUDA(launch(kvb::release_pages_kernel, dim3(grid), kvb::PG_THREADS, 0, s, *p, 1, one));
  if (!one) KVB_CUDA(launch(kvb::release_pages_kernel, dim3(1), kvb::PG_THREADS, 0, s, *p, 0, 1));
  return KVSKIP_OK;
}

}  // extern "C"
