"""The paged key / value cache of text generation.

The reference keeps `[past | new]` keys and values of every layer in tensors that grow by concatenation (use_cache /
layer_past, megatron/model/transformer.py:361-365, 602-610).  Here a layer's keys and values live in pages of `page_size`
token slots; sequences take pages as they grow and give them back when they end, so nothing is copied and sequences of any
lengths share one batch.  `PagedKV` is one layer's pages, `PagedStep` what one step of a batch brings; `ops.paged_kv_append`
and `ops.paged_attn_fwd` work on a pair of them.  `PagedKVCache` holds the pages of all layers and hands them out; a
`PagedPast` of one of its layers is what `ParallelTransformerLayer.forward` takes as `layer_past`.
"""
import ctypes

import torch

from ._lib import MmPagedKV, MmPagedStep, dtype_code


class PagedKV:
    """One layer's pages: k and v [num_pages, heads, page_size, hn] in fp16 / bf16, head size 64 or 128.  Any strides, the same for
    both, that are multiples of 8 elements with the head dim contiguous: both may be views of one tensor."""

    def __init__(self, k, v):
        if k.dim() != 4 or k.shape != v.shape or k.dtype != v.dtype or k.device != v.device or not k.is_cuda:
            raise RuntimeError("PagedKV: k and v must be GPU tensors [num_pages, heads, page_size, hn] of one shape, dtype and device")
        if k.size(3) not in (64, 128):
            raise RuntimeError(f"PagedKV: head size {k.size(3)} not supported (64 or 128)")
        if min(k.shape) < 1:
            raise RuntimeError(f"PagedKV: empty cache {tuple(k.shape)}")
        if k.stride() != v.stride() or k.stride(3) != 1 or any(s % 8 or s <= 0 for s in k.stride()[:3]) or k.data_ptr() % 16 or v.data_ptr() % 16:
            raise RuntimeError("PagedKV: pages must be 16-byte aligned with a contiguous head dim and positive strides that are multiples "
                               f"of 8, the same for k and v; got {k.stride()} and {v.stride()}")
        self.k, self.v = k, v
        self.num_pages, self.heads, self.page_size, self.hn = k.shape
        self.dtype, self.device = k.dtype, k.device
        self._c = MmPagedKV(k.data_ptr(), v.data_ptr(), *k.stride()[:3], self.num_pages, self.page_size, self.heads,
                            self.hn, dtype_code(k.dtype))
        self._ref = ctypes.addressof(self._c)


class PagedStep:
    """What one step of a batch brings, shared by all layers.  block_table int32 [seqs, max_pages]: the pages of each sequence in
    order; cu_new int32 [seqs + 1], ascending: sequence i brings the packed rows cu_new[i] .. cu_new[i + 1] - 1; kv_lens int32
    [seqs]: its length including them.  max_new, max_kv: upper bounds of a sequence's new rows and length (defaults: read from
    the arrays, which waits for the GPU).  The kernels read the arrays when they run, so their contents may be rewritten between
    the replays of a captured step; a step that breaks the bounds, or names pages the cache does not have, gives NaN rows and
    leaves the cache alone, and a row at a negative position attends to nothing: 0 (include/mm_hip.h, mm_paged_step)."""

    def __init__(self, block_table, cu_new, kv_lens, max_new=None, max_kv=None):
        if block_table.dim() != 2 or cu_new.dim() != 1 or kv_lens.dim() != 1:
            raise RuntimeError("PagedStep: block_table [seqs, max_pages], cu_new [seqs + 1] and kv_lens [seqs] expected")
        for t in (block_table, cu_new, kv_lens):
            if t.dtype != torch.int32 or not t.is_cuda or t.device != cu_new.device:
                raise RuntimeError("PagedStep: block_table, cu_new and kv_lens must be int32 tensors on one GPU")
        self.seqs = kv_lens.numel()
        if cu_new.numel() != self.seqs + 1 or block_table.size(0) != self.seqs or block_table.size(1) < 1:
            raise RuntimeError(f"PagedStep: block_table {tuple(block_table.shape)} and cu_new {tuple(cu_new.shape)} do not fit "
                               f"{self.seqs} sequences")
        if not (cu_new.is_contiguous() and kv_lens.is_contiguous()) or block_table.stride(1) != 1 or block_table.stride(0) < block_table.size(1):
            raise RuntimeError("PagedStep: cu_new, kv_lens and the rows of block_table must be contiguous and the rows must not overlap")
        if max_new is None:
            max_new = int((cu_new[1:] - cu_new[:-1]).max()) if self.seqs else 0
        if max_kv is None:
            max_kv = int(kv_lens.max()) if self.seqs else 0
        if not (0 <= max_new < 1 << 31 and 0 <= max_kv < 1 << 31):
            raise RuntimeError(f"PagedStep: max_new={max_new}, max_kv={max_kv} must be in [0, 2^31)")
        self.block_table, self.cu_new, self.kv_lens = block_table, cu_new, kv_lens
        self.max_new, self.max_kv, self.device = int(max_new), int(max_kv), cu_new.device
        self._c = MmPagedStep(block_table.data_ptr(), cu_new.data_ptr(), kv_lens.data_ptr(), block_table.stride(0), self.seqs,
                              block_table.size(1), self.max_new, self.max_kv)
        self._ref = ctypes.addressof(self._c)


class PagedPast:
    """`layer_past` of a layer in generation: its pages, the step, and how many positions a sequence can have (the length of the
    rotary tables)."""

    def __init__(self, kv, step, max_positions):
        self.kv, self.step, self.max_positions = kv, step, int(max_positions)


class PagedKVCache:
    """Pages for all layers of a model, and the host side of handing them out.  num_heads: this tensor-parallel rank's."""

    def __init__(self, num_layers, num_heads, head_size, num_pages, page_size=16, dtype=torch.bfloat16, device="cuda"):
        if min(num_layers, num_heads, num_pages, page_size) < 1:
            raise RuntimeError("PagedKVCache: layers, heads, pages and page_size must be positive")
        pages = torch.empty(num_layers, 2, num_pages, num_heads, page_size, head_size, dtype=dtype, device=device)
        self.layers = [PagedKV(pages[i, 0], pages[i, 1]) for i in range(num_layers)]
        self.page_size, self.device = page_size, pages.device
        self._free = list(range(num_pages - 1, -1, -1))
        self._pages = {}   # sequence -> its pages, in order
        self._next = 0

    def _of(self, seq):
        if seq not in self._pages:
            raise RuntimeError(f"PagedKVCache: no sequence {seq}")
        return self._pages[seq]

    @property
    def free_pages(self):
        return len(self._free)

    def add(self, tokens):
        """A new sequence with room for `tokens` tokens; returns its handle."""
        seq, self._next = self._next, self._next + 1
        self._pages[seq] = []
        try:
            self.reserve(seq, tokens)
        except RuntimeError:
            del self._pages[seq]
            raise
        return seq

    def reserve(self, seq, tokens):
        """Room for `tokens` tokens in all; raises, and takes nothing, when the free pages do not suffice."""
        pages = self._of(seq)
        need = -(-int(tokens) // self.page_size) - len(pages)
        if need > len(self._free):
            raise RuntimeError(f"PagedKVCache: {need} pages needed, {len(self._free)} free")
        for _ in range(need):
            pages.append(self._free.pop())

    def release(self, seq):
        """Give a sequence's pages back.  Work on the GPU that still reads them must have been enqueued on the stream of the work
        that will write them next."""
        self._free.extend(reversed(self._of(seq)))
        del self._pages[seq]

    def block_table(self, seqs):
        """int32 [len(seqs), pages of the longest] on the device; entries behind a sequence's last page are -1."""
        width = max([len(self._of(s)) for s in seqs] + [1])
        rows = [self._pages[s] + [-1] * (width - len(self._pages[s])) for s in seqs]
        return torch.tensor(rows, dtype=torch.int32).view(len(seqs), width).to(self.device)

    def step(self, seqs, new, lens):
        """The step that brings new[i] rows to sequence seqs[i], whose length is lens[i] afterwards (host numbers).  A sequence comes
        once: two rows of a step must not share a slot."""
        if not len(seqs) == len(new) == len(lens):
            raise RuntimeError(f"PagedKVCache: {len(seqs)} sequences, but {len(new)} and {len(lens)} numbers for them")
        if len(set(seqs)) != len(seqs):
            raise RuntimeError(f"PagedKVCache: a sequence comes twice in {list(seqs)}")
        for s, n, l in zip(seqs, new, lens):
            if not 0 <= n <= l or l > len(self._of(s)) * self.page_size:
                raise RuntimeError(f"PagedKVCache: sequence {s} has room for {len(self._pages[s]) * self.page_size} tokens, not for "
                                   f"{n} new ones up to {l}")
        cu = [0]
        for n in new:
            cu.append(cu[-1] + int(n))
        meta = torch.tensor(cu + [int(l) for l in lens], dtype=torch.int32).to(self.device)
        return PagedStep(self.block_table(seqs), meta[:len(cu)], meta[len(cu):], max_new=max(list(new) + [0]), max_kv=max(list(lens) + [0]))
