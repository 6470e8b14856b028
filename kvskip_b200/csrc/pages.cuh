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

// Exclusive prefix sums of two numbers per thread over the CTA, and their totals.
struct PgScan {
  int64_t a[32], b[32];
};
__device__ __forceinline__ void pg_scan(PgScan& sh, int64_t& a, int64_t& b, int64_t& ta, int64_t& tb) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t a0 = a, b0 = b;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t x = __shfl_up_sync(0xffffffffu, a, o), y = __shfl_up_sync(0xffffffffu, b, o);
    if (lane >= o) a += x, b += y;
  }
  __syncthreads();                       // (the previous round's sums have been read)
  if (lane == 31) sh.a[warp] = a, sh.b[warp] = b;
  __syncthreads();
  int64_t pa = 0, pb = 0;
  ta = tb = 0;
#pragma unroll 8
  for (int w = 0; w < PG_THREADS / 32; ++w) {
    if (w < warp) pa += sh.a[w], pb += sh.b[w];
    ta += sh.a[w], tb += sh.b[w];
  }
  a += pa - a0;
  b += pb - b0;
}
// last of 1024 ascending values that is <= x
__device__ __forceinline__ int pg_find(const int64_t* v, const int64_t x) {
  int lo = 0;
#pragma unroll
  for (int step = PG_THREADS / 2; step > 0; step >>= 1)
    if (v[lo + step] <= x) lo += step;
  return lo;
}

// map: this launch writes the slots and the table; finish: it writes lens_out and n_free_out.  Both in one
// launch unless these are lens and n_free themselves and several CTAs still have to read them.
__global__ void __launch_bounds__(PG_THREADS) extend_pages_kernel(const __grid_constant__ kvskip_pages_params p, const int map,
                                                                  const int finish) {
  __shared__ PgScan sh;
  __shared__ int64_t tok0[PG_THREADS], need0[PG_THREADS];   // tokens / new blocks before the request
  __shared__ int len_s[PG_THREADS], new_s[PG_THREADS];      // new_s: -1 - count for a refused request
  pdl_wait_prior();
  pdl_launch_dependents();
  const int tid = threadIdx.x;
  const int64_t nf = max(0, min(*p.n_free, p.num_free));
  const int64_t t0 = p.n_tokens * blockIdx.x / gridDim.x, t1 = p.n_tokens * (blockIdx.x + 1) / gridDim.x;
  int64_t toks = 0, needs = 0, used = 0;
  for (int base = 0; base < p.B; base += PG_THREADS) {
    const int b = base + tid;
    int len = 0, add = 0, have = 0;
    int64_t need = 0;
    bool fits = true;
    int64_t want_t = 0;
    if (b < p.B) {
      len = max(0, p.lens[b]);
      add = max(0, p.new_[b]);
      have = len / TILE + (len % TILE != 0);
      want_t = static_cast<int64_t>(len) + add;
    }
    int64_t ta, tb, at = add, dummy = 0;
    pg_scan(sh, at, dummy, ta, tb);
    at += toks;                                             // tokens before the request
    fits = (want_t + TILE - 1) / TILE <= p.max_pages && (p.per_row ? add <= p.per_row : at + add <= p.n_tokens);
    need = fits ? max(static_cast<int64_t>(0), (want_t + TILE - 1) / TILE - have) : 0;
    int64_t nat = need, zero = 0, tn, tz;
    pg_scan(sh, nat, zero, tn, tz);
    nat += needs;
    const bool granted = fits && (need == 0 || nat + need <= nf);
    tok0[tid] = p.per_row ? static_cast<int64_t>(b) * p.per_row : at;
    need0[tid] = nat;
    len_s[tid] = len;
    new_s[tid] = granted ? add : -1 - add;
    __syncthreads();
    if (map) {
      // tokens of these requests that are in this CTA's share of the list
      const int64_t c0 = p.per_row ? static_cast<int64_t>(base) * p.per_row : toks;
      const int64_t c1 = p.per_row ? min(p.n_tokens, static_cast<int64_t>(base + PG_THREADS) * p.per_row) : toks + ta;
      for (int64_t t = max(t0, c0) + tid; t < min(t1, c1); t += PG_THREADS) {
        const int r = p.per_row ? static_cast<int>(t / p.per_row) - base : pg_find(tok0, t);
        const int i = static_cast<int>(t - tok0[r]);
        int64_t slot = -1;
        int pos = -1;
        if (i < new_s[r]) {
          pos = len_s[r] + i;
          const int j = pos / TILE, hv = len_s[r] / TILE + (len_s[r] % TILE != 0);
          const int page = j < hv ? p.table[static_cast<int64_t>(base + r) * p.max_pages + j]
                                  : p.free_pages[nf - 1 - (need0[r] + j - hv)];
          slot = static_cast<int64_t>(page) * TILE + pos % TILE;
        }
        p.slots[t] = slot;
        p.positions[t] = pos;
      }
      for (int64_t x = needs + static_cast<int64_t>(blockIdx.x) * PG_THREADS + tid; x < min(needs + tn, nf);
           x += static_cast<int64_t>(gridDim.x) * PG_THREADS) {
        const int r = pg_find(need0, x);
        if (new_s[r] < 0) continue;
        const int hv = len_s[r] / TILE + (len_s[r] % TILE != 0);
        p.table[static_cast<int64_t>(base + r) * p.max_pages + hv + (x - need0[r])] = p.free_pages[nf - 1 - x];
      }
      if (blockIdx.x == 0 && b < p.B) p.granted[b] = granted;
    }
    if (finish && blockIdx.x == 0 && b < p.B) p.lens_out[b] = granted ? static_cast<int>(want_t) : p.lens[b];
    int64_t g = granted ? need : 0, gz = 0, tg, tgz;
    if (finish && blockIdx.x == 0) {
      pg_scan(sh, g, gz, tg, tgz);
      used += tg;
    }
    toks += ta;
    needs += tn;
    __syncthreads();
  }
  if (map && !p.per_row)
    for (int64_t t = max(t0, min(toks, p.n_tokens)) + tid; t < t1; t += PG_THREADS) p.slots[t] = -1, p.positions[t] = -1;
  if (finish && blockIdx.x == 0 && tid == 0) *p.n_free_out = static_cast<int>(nf - used);
}

__global__ void __launch_bounds__(PG_THREADS) release_pages_kernel(const __grid_constant__ kvskip_pages_params p, const int map,
                                                                   const int finish) {
  __shared__ PgScan sh;
  __shared__ int64_t have0[PG_THREADS];
  pdl_wait_prior();
  pdl_launch_dependents();
  const int tid = threadIdx.x;
  const int64_t nf = max(0, min(*p.n_free, p.num_free));
  int64_t back = 0;
  for (int base = 0; base < p.B; base += PG_THREADS) {
    const int b = base + tid;
    int64_t at = 0, zero = 0, ta, tz;
    bool done = false;
    if (b < p.B) {
      done = p.done[b] != 0;
      const int len = max(0, p.lens[b]);
      if (done) at = min(static_cast<int64_t>(p.max_pages), static_cast<int64_t>(len / TILE + (len % TILE != 0)));
    }
    pg_scan(sh, at, zero, ta, tz);
    at += back;
    have0[tid] = at;
    __syncthreads();
    if (map)
      for (int64_t x = back + static_cast<int64_t>(blockIdx.x) * PG_THREADS + tid; x < back + ta;
           x += static_cast<int64_t>(gridDim.x) * PG_THREADS) {
        const int r = pg_find(have0, x);
        if (nf + x < p.num_free)
          p.free_pages[nf + x] = p.table[static_cast<int64_t>(base + r) * p.max_pages + (x - have0[r])];
      }
    if (finish && blockIdx.x == 0 && b < p.B) p.lens_out[b] = done ? 0 : p.lens[b];
    back += ta;
    __syncthreads();
  }
  if (finish && blockIdx.x == 0 && tid == 0) *p.n_free_out = static_cast<int>(min(nf + back, static_cast<int64_t>(p.num_free)));
}

}  // namespace kvb
