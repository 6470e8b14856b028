// Page and slot tables from request lengths (see kvskip_launch_extend_pages in the header).
//
// Whole numbers only, a few bytes per token: a chain of memory round trips, not a bandwidth.  Every CTA runs
// the same prefix sums over all requests (1024 at a time; they are a few kilobytes) and then maps its own
// share of the tokens and of the new table entries, finding the request of each by binary search in
// the sums.  The page of a token in a new block follows from the sums and the stack, so no CTA waits for a table
// entry that another one writes.
#pragma once
#include "common.cuh"

namespace kvb {

constexpr int PG_THREADS = 1024;
constexpr int PG_MOST_PAGES = 1 << 20;   // bound on max_pages: the new blocks of 1024 requests are at most 2^30,
constexpr int PG_MANY = (1 << 30) - 1;   // and those of all before them count as at most this: the sum fits 31 bits

// Exclusive prefix sums over the CTA of a 64-bit and a 32-bit number per thread, and their totals.
struct PgScan {
  int64_t a[32];
  int b[32];
};
__device__ __forceinline__ void pg_scan(PgScan& sh, int64_t& a, int& b, int64_t& ta, int& tb) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t a0 = a;
  const int b0 = b;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t x = __shfl_up_sync(0xffffffffu, a, o);
    const int y = __shfl_up_sync(0xffffffffu, b, o);
    if (lane >= o) a += x, b += y;
  }
  if (lane == 31) sh.a[warp] = a, sh.b[warp] = b;
  __syncthreads();
  // the sums before this warp: every warp adds up the 32 totals
  int64_t wa = sh.a[lane];
  int wb = sh.b[lane];
  const int64_t wa0 = wa;
  const int wb0 = wb;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t x = __shfl_up_sync(0xffffffffu, wa, o);
    const int y = __shfl_up_sync(0xffffffffu, wb, o);
    if (lane >= o) wa += x, wb += y;
  }
  ta = __shfl_sync(0xffffffffu, wa, 31), tb = __shfl_sync(0xffffffffu, wb, 31);
  a += __shfl_sync(0xffffffffu, wa - wa0, warp) - a0;
  b += __shfl_sync(0xffffffffu, wb - wb0, warp) - b0;
}
// last of 1024 ascending values that is <= x
template <typename T>
__device__ __forceinline__ int pg_find(const T* v, const T x) {
  int lo = 0;
#pragma unroll
  for (int step = PG_THREADS / 2; step > 0; step >>= 1)
    if (v[lo + step] <= x) lo += step;
  return lo;
}
__device__ __forceinline__ int pg_blocks(const int len) { return len / TILE + (len % TILE != 0); }

// map: this launch writes the slots and the table; finish: it writes lens_out and n_free_out.  Both in one
// launch unless these are lens and n_free themselves and several CTAs still have to read them.
__global__ void __launch_bounds__(PG_THREADS) extend_pages_kernel(const __grid_constant__ kvskip_pages_params p, const int map,
                                                                  const int finish) {
  __shared__ PgScan sh;
  __shared__ int64_t tok0[PG_THREADS];                      // tokens before the request
  __shared__ int need0[PG_THREADS];                         // new blocks before the request
  __shared__ int len_s[PG_THREADS], new_s[PG_THREADS];      // new_s: -1 - count for a refused request
  __shared__ int used_s;
  pdl_wait_prior();
  pdl_launch_dependents();
  const int tid = threadIdx.x;
  if (tid == 0) used_s = 0;
  const int nf = max(0, min(*p.n_free, p.num_free));
  const int64_t t0 = p.n_tokens * blockIdx.x / gridDim.x, t1 = p.n_tokens * (blockIdx.x + 1) / gridDim.x;
  int64_t toks = 0;
  int needs = 0;                         // (held at PG_MANY, as many as the largest stack has)
  for (int base = 0; base < p.B; base += PG_THREADS) {
    const int b = base + tid;
    int len = 0, add = 0;
    if (b < p.B) len = max(0, p.lens[b]), add = max(0, p.new_[b]);
    if (p.live_only && len == 0) add = 0;
    const int64_t want_t = static_cast<int64_t>(len) + add;
    const int64_t want = (want_t + TILE - 1) / TILE;
    // One scan: whether the tokens of a request still fit into the list is known only behind it, but of the requests
    // behind the first that does not none with a token fits, so its blocks may be counted all the same.
    bool fits = want <= p.max_pages && (!p.per_row || add <= p.per_row);
    const int need = fits ? max(0, min(static_cast<int>(want), p.max_pages) - pg_blocks(len)) : 0;
    int64_t at = add, ta;
    int nat = need, tn;
    pg_scan(sh, at, nat, ta, tn);
    at += toks;
    nat += needs;
    if (!p.per_row) fits = fits && (add == 0 || at + add <= p.n_tokens);    // (no token: no place needed)
    const bool granted = fits && (need == 0 || nat + need <= nf);
    tok0[tid] = p.per_row ? static_cast<int64_t>(b) * p.per_row : at;
    need0[tid] = nat;
    len_s[tid] = len;
    new_s[tid] = granted ? add : -1 - add;
    if (finish && blockIdx.x == 0) {
      // (the granted requests that need pages are the first ones: the last of them has them all before it)
      if (granted && need > 0) atomicMax(&used_s, nat + need);
      if (b < p.B) p.lens_out[b] = granted ? static_cast<int>(want_t) : p.lens[b];
    }
    if (map && blockIdx.x == 0 && b < p.B) p.granted[b] = granted;
    __syncthreads();
    if (map) {
      // tokens of these requests that are in this CTA's share of the list
      const int64_t c0 = p.per_row ? static_cast<int64_t>(base) * p.per_row : toks;
      const int64_t c1 = p.per_row ? min(p.n_tokens, static_cast<int64_t>(base + PG_THREADS) * p.per_row) : toks + ta;
      for (int64_t t = max(t0, c0) + tid; t < min(t1, c1); t += PG_THREADS) {
        const int r = !p.per_row ? pg_find(tok0, t) : p.per_row == 1 ? static_cast<int>(t) - base
                                                                     : static_cast<int>(t / p.per_row) - base;
        const int i = static_cast<int>(t - tok0[r]);
        int64_t slot = -1;
        int pos = -1;
        if (i < new_s[r]) {
          pos = len_s[r] + i;
          const int j = pos / TILE, hv = pg_blocks(len_s[r]);
          const int page = j < hv ? p.table[static_cast<int64_t>(base + r) * p.max_pages + j]
                                  : p.free_pages[nf - 1 - (need0[r] + j - hv)];
          slot = static_cast<int64_t>(page) * TILE + pos % TILE;
        }
        p.slots[t] = slot;
        p.positions[t] = pos;
      }
      for (int x = needs + blockIdx.x * PG_THREADS + tid; x < min(needs + tn, nf); x += gridDim.x * PG_THREADS) {
        const int r = pg_find(need0, x);
        if (new_s[r] < 0) continue;
        p.table[static_cast<int64_t>(base + r) * p.max_pages + pg_blocks(len_s[r]) + (x - need0[r])] = p.free_pages[nf - 1 - x];
      }
    }
    toks += ta;
    needs = min(needs + tn, PG_MANY);
    __syncthreads();
  }
  if (map && !p.per_row)
    for (int64_t t = max(t0, min(toks, p.n_tokens)) + tid; t < t1; t += PG_THREADS) p.slots[t] = -1, p.positions[t] = -1;
  if (finish && blockIdx.x == 0 && tid == 0) *p.n_free_out = nf - used_s;
}

__global__ void __launch_bounds__(PG_THREADS) release_pages_kernel(const __grid_constant__ kvskip_pages_params p, const int map,
                                                                   const int finish) {
  __shared__ PgScan sh;
  __shared__ int64_t have0[PG_THREADS];
  pdl_wait_prior();
  pdl_launch_dependents();
  const int tid = threadIdx.x;
  const int nf = max(0, min(*p.n_free, p.num_free));
  int64_t back = 0;
  for (int base = 0; base < p.B; base += PG_THREADS) {
    const int b = base + tid;
    int64_t at = 0, ta;
    int zero = 0, tz;
    bool done = false;
    if (b < p.B) {
      done = p.done[b] != 0;
      const int len = p.lens[b];
      if (done) at = min(p.max_pages, pg_blocks(max(0, len)));
      if (finish && blockIdx.x == 0) p.lens_out[b] = done ? 0 : len;
    }
    pg_scan(sh, at, zero, ta, tz);
    at += back;
    have0[tid] = at;
    __syncthreads();
    if (map)
      for (int64_t x = back + blockIdx.x * PG_THREADS + tid; x < back + ta; x += gridDim.x * PG_THREADS) {
        const int r = pg_find(have0, x);
        if (nf + x < p.num_free)
          p.free_pages[nf + x] = p.table[static_cast<int64_t>(base + r) * p.max_pages + (x - have0[r])];
      }
    back += ta;
    __syncthreads();
  }
  if (finish && blockIdx.x == 0 && tid == 0) *p.n_free_out = static_cast<int>(min(nf + back, static_cast<int64_t>(p.num_free)));
}

}  // namespace kvb
