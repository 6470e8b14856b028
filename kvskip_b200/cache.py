"""KV caches either side of the decode kernels: a growing contiguous cache and a paged one.

`GrowingKV` has the behaviour of the reference's cache layer (format37/kvskip
src/kvskip_attn.py:67-113, `GrowingLayer`): one [B,Hkv,capacity,D] buffer per tensor that doubles
when it runs out, capacity a multiple of the 64-token block, `update()` returning views of the
current length, `crop()`.  It does not depend on transformers; an HF cache layer can delegate to it.
A single decode token is written by the library's append kernel (one launch for K and V), which
can also take the length from device memory, so the append is part of a captured step.

`PagedKV` stores the cache in 64-token pages, [pages,Hkv,64,D] per tensor, with a page table
int32 [B, max_pages]: block j of sequence b lives in page table[b, j].  The attention kernels read
a block straight from its page (the tensor map runs over the pool), so the planner's block list
and the page table together decide which pages a step touches; nothing is gathered.  The reference
reads [B,Hkv,T,D] views only; its notes name this layout as the natural one for block skipping
(docs/03-gate-digest.md:364).

`PagedKV8` is a paged cache for a batch of requests of different lengths, in 8-bit codes with one scale
per page and head, whose tables live on the device: handing out pages, writing tokens and
reading them back through `kvskip.decode8` needs no host synchronisation, so a decode step can be captured
once and replayed while the requests grow.
"""

import math

import torch

from . import kvskip as K

BLOCK = 64


class GrowingKV:
    """One layer's contiguous cache.  capacity: tokens to allocate at first (no doubling below it)."""

    def __init__(self, capacity: int = 0):
        self.capacity = capacity
        self._k = self._v = None
        self._n = 0

    def _ensure(self, need: int, ref: torch.Tensor) -> None:
        cap = 0 if self._k is None else self._k.shape[-2]
        if need <= cap:
            return
        new_cap = math.ceil(max(need + 512, 2 * cap, self.capacity) / BLOCK) * BLOCK
        B, H, _, D = ref.shape
        k = torch.empty(B, H, new_cap, D, dtype=ref.dtype, device=ref.device)
        v = torch.empty_like(k)
        if self._n:
            k[:, :, :self._n] = self._k[:, :, :self._n]
            v[:, :, :self._n] = self._v[:, :, :self._n]
        self._k, self._v = k, v

    def update(self, key_states: torch.Tensor, value_states: torch.Tensor):
        """Appends [B,Hkv,t,D] and returns (keys, values): views of the whole current length."""
        t = key_states.shape[-2]
        self._ensure(self._n + t, key_states)
        if t == 1 and key_states.is_cuda:
            K.ext().append(self._k, self._v, key_states[:, :, 0].contiguous(), value_states[:, :, 0].contiguous(),
                           self._n + 1)
        else:
            self._k[:, :, self._n:self._n + t] = key_states
            self._v[:, :, self._n:self._n + t] = value_states
        self._n += t
        return self.views()

    def views(self):
        return self._k[:, :, :self._n], self._v[:, :, :self._n]

    def full(self):
        """The whole buffers (for launches that read the length from device memory)."""
        return self._k, self._v

    def get_seq_length(self) -> int:
        return self._n

    def room(self) -> int:
        """Tokens that fit before the next re-allocation (a captured step is valid that long)."""
        return 0 if self._k is None else self._k.shape[-2] - self._n

    def crop(self, tokens_to_remove: int) -> None:
        """Negative: drop that many tokens from the end; positive: keep that many (legacy form)."""
        if tokens_to_remove > 0:
            tokens_to_remove = max(0, self._n - tokens_to_remove)
        self._n -= abs(tokens_to_remove)


class PagedKV:
    """A page pool shared by B sequences of equal length (the kernels take one length per launch).

    pages are handed out from a free list on the host; `order` ("ascending", "shuffled") only
    matters for tests, which use a shuffled pool to show that no layout is assumed."""

    def __init__(self, num_pages: int, B: int, Hkv: int, D: int, max_tokens: int, device, dtype=torch.bfloat16,
                 order: str = "ascending", seed: int = 0):
        self.k = torch.empty(num_pages, Hkv, BLOCK, D, dtype=dtype, device=device)
        self.v = torch.empty_like(self.k)
        self.max_pages = math.ceil(max_tokens / BLOCK)
        self.table_host = torch.full((B, self.max_pages), -1, dtype=torch.int32)
        self.table = self.table_host.to(device)
        free = list(range(num_pages))
        if order == "shuffled":
            perm = torch.randperm(num_pages, generator=torch.Generator().manual_seed(seed)).tolist()
            free = perm
        self._free = free[::-1]          # pop() hands out from the front of the order
        self.B, self.n = B, 0
        self._blocks = 0                 # blocks per sequence that have a page

    def _ensure(self, T: int) -> None:
        """Pages for every block below ceil(T/64), for all sequences; the table goes to the device
        only when a block boundary is crossed."""
        have = self._blocks
        need = math.ceil(T / BLOCK)
        if need <= have:
            return
        if need > self.max_pages:
            raise RuntimeError(f"PagedKV: {T} tokens exceed max_tokens")
        for j in range(have, need):
            for b in range(self.B):
                if not self._free:
                    raise RuntimeError("PagedKV: the pool is exhausted")
                self.table_host[b, j] = self._free.pop()
        self._blocks = need
        self.table.copy_(self.table_host, non_blocking=True)

    def write(self, k: torch.Tensor, v: torch.Tensor) -> None:
        """Prefill: [B,Hkv,T,D] into pages (sequence length becomes T)."""
        B, H, T, D = k.shape
        self._ensure(T)
        self.n = T
        nb = math.ceil(T / BLOCK)
        pad = nb * BLOCK - T
        if pad:
            k = torch.nn.functional.pad(k, (0, 0, 0, pad))
            v = torch.nn.functional.pad(v, (0, 0, 0, pad))
        pages = self.table[:, :nb].long().reshape(-1)                                     # [B*nb]
        self.k[pages] = k.reshape(B, H, nb, BLOCK, D).permute(0, 2, 1, 3, 4).reshape(B * nb, H, BLOCK, D)
        self.v[pages] = v.reshape(B, H, nb, BLOCK, D).permute(0, 2, 1, 3, 4).reshape(B * nb, H, BLOCK, D)

    def append(self, k_new: torch.Tensor, v_new: torch.Tensor, t_dev: torch.Tensor | None = None) -> None:
        """One token per sequence, [B,Hkv,D] each.  With t_dev the row index comes from the device
        (t_dev already holds the length after the append)."""
        self._ensure(self.n + 1)
        self.n += 1
        K.ext().append(self.k, self.v, k_new.contiguous(), v_new.contiguous(),
                       self.n if t_dev is None else self.max_pages * BLOCK, t_dev, self.table)

    def reserve(self, T: int) -> None:
        """Hand out pages up to length T now (a captured step must not run out of pages)."""
        self._ensure(T)

    # hooks of kvskip_b200.graph.StepGraph: an append inside a captured step is replayed without
    # this object seeing it
    def graph_scalars(self) -> tuple:
        return ()

    def note_replayed(self) -> None:
        if math.ceil((self.n + 1) / BLOCK) > self._blocks:
            raise RuntimeError("PagedKV: a replayed append ran past the reserved pages (call reserve() first)")
        self.n += 1

    def gather(self):
        """Contiguous copies [B,Hkv,n,D] of the cache (tests, debugging)."""
        nb = math.ceil(self.n / BLOCK)
        pages = self.table[:, :nb].long()
        k = self.k[pages].permute(0, 2, 1, 3, 4).reshape(self.B, self.k.shape[1], nb * BLOCK, -1)[:, :, :self.n]
        v = self.v[pages].permute(0, 2, 1, 3, 4).reshape(self.B, self.v.shape[1], nb * BLOCK, -1)[:, :, :self.n]
        return k.contiguous(), v.contiguous()

    def get_seq_length(self) -> int:
        return self.n


class PagedKV8:
    """A pool of 64-token pages in 8-bit codes (float8_e4m3fn or int8) shared by up to B requests; row b of the
    batch is request b, `lens[b]` tokens long (0: no request).

        slots = cache.extend(new, per_row=S)     # pages for new[b] more tokens of every request
        cache.write(k_new, v_new, slots)         # [B,Hkv,S,D] (or packed: [N,Hkv,D] with n_tokens=N)
        out = cache.decode(q, scale)["out"]
        cache.release(done)                      # pages of finished requests go back

    Nothing here synchronises; a request that finds no page is refused (`granted`) and keeps its length.
    `lens`, `table`, `free_pages`, `n_free` and `granted` are device tensors that change in place, so that they say after a
    replayed step what that step did.  `positions` (of the last extension's list) is another tensor for every call of `extend`;
    after a step that `StepGraph` replays it is the one of the captured call."""

    def __init__(self, num_pages: int, B: int, Hkv: int, D: int, max_tokens: int, device,
                 dtype=torch.float8_e4m3fn):
        if dtype not in (torch.float8_e4m3fn, torch.int8):
            raise ValueError("PagedKV8: float8_e4m3fn or int8")
        if D not in (64, 128):
            raise ValueError("PagedKV8: head dim 64 or 128")
        if min(num_pages, B, Hkv, max_tokens) < 1:
            raise ValueError("PagedKV8: num_pages, B, Hkv and max_tokens are at least 1")
        self.k = torch.zeros(num_pages, Hkv, BLOCK, D, dtype=torch.uint8, device=device).view(dtype)
        self.v = torch.zeros(num_pages, Hkv, BLOCK, D, dtype=torch.uint8, device=device).view(dtype)
        self.k_scale = torch.ones(num_pages, Hkv, dtype=torch.float32, device=device)
        self.v_scale = torch.ones_like(self.k_scale)
        self.B, self.max_pages = B, math.ceil(max_tokens / BLOCK)
        self.lens = torch.zeros(B, dtype=torch.int32, device=device)
        self.table = torch.full((B, self.max_pages), -1, dtype=torch.int32, device=device)
        self.free_pages = torch.arange(num_pages - 1, -1, -1, dtype=torch.int32, device=device)   # page 0 on top
        self.n_free = torch.full((1,), num_pages, dtype=torch.int32, device=device)
        self.granted = torch.zeros(B, dtype=torch.bool, device=device)
        self.positions = None
        self._ones = torch.ones(B, dtype=torch.int32, device=device)

    def extend(self, new: torch.Tensor | None = None, *, n_tokens: int | None = None, per_row: int | None = None,
               live_only: bool = False):
        """Room for new[b] (int32 [B], default one in every row, rows of length 0 too unless live_only) more tokens of
        every request; returns their slots (see `kvskip.extend_pages`), `granted` and `positions` are kept on the object."""
        if new is None:
            new = self._ones
        if n_tokens is None and per_row is None:
            per_row = 1
        r = K.extend_pages(self.lens, new, self.table, self.free_pages, self.n_free, n_tokens=n_tokens, per_row=per_row,
                           lens_out=self.lens, n_free_out=self.n_free, granted_out=self.granted,
                           live_only=live_only)
        self.positions = r["positions"]
        return r["slots"]

    def write(self, k_new: torch.Tensor, v_new: torch.Tensor, slots: torch.Tensor) -> None:
        K.write8(k_new, v_new, slots, self.k, self.v, self.k_scale, self.v_scale)

    def append(self, k_new: torch.Tensor, v_new: torch.Tensor, new: torch.Tensor | None = None) -> None:
        """One token per request, [B,Hkv,D] each.  new (int32 [B] of 0 and 1): the rows that get one, a row without a
        request among them (which begins it); by default every row that holds a request, `lens[b] > 0`."""
        slots = self.extend(new, per_row=1, live_only=new is None)
        self.write(k_new.unsqueeze(2), v_new.unsqueeze(2), slots)

    def release(self, done: torch.Tensor) -> None:
        K.release_pages(done, self.lens, self.table, self.free_pages, self.n_free, lens_out=self.lens,
                        n_free_out=self.n_free)

    def decode(self, q, scale: float, plan=None, stats: bool = False, out_f32: bool = False,
               max_len: int | None = None) -> dict:
        """Attention of one token per request.  The launch is sized by the table's width unless `max_len` gives a smaller bound on
        the lengths (longer requests are cut off there): 1000 tokens of one request take 7.7 us under a bound of 1024 and
        8.9 under one of 65536."""
        return K.decode8(q, self.k, self.v, self.k_scale, self.v_scale, scale, lens=self.lens, page_table=self.table,
                         max_len=max_len, plan=plan, stats=stats, out_f32=out_f32)

    # hooks of kvskip_b200.graph.StepGraph: the lengths are on the device, a replayed step needs nothing here
    def graph_scalars(self) -> tuple:
        return ()

    def note_replayed(self) -> None:
        pass

    def graph_outputs(self):
        return self.positions

    def take_outputs(self, positions) -> None:
        self.positions = positions

    def gather(self, b: int):
        """fp32 copies [Hkv,n,D] of request b's keys and values (tests, debugging; reads the length back)."""
        n = int(self.lens[b])
        pages = self.table[b, :math.ceil(n / BLOCK)].long()
        out = []
        for codes, scale in ((self.k, self.k_scale), (self.v, self.v_scale)):
            x = codes[pages].float() * scale[pages][:, :, None, None]
            out.append(x.transpose(0, 1).reshape(x.shape[1], -1, x.shape[3])[:, :n])
        return tuple(out)
