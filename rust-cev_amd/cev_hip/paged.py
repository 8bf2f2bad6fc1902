"""Serving over a paged K/V cache: the step's bookkeeping from the requests'
lengths, rotary positions with the cache stores, and attention of each
request's new tokens over its pages.

The caches of a layer are (n_pages, page_size, hkv, d) tensors of any strides
with unit last stride; request r's key j lies in page block_table[r][j //
page_size].  A step:

    paged_tables(lengths, new_len, block_table, page_size, cu, pos, slots, free, ring)    # once
    attention.plan(cu, lengths)                                                           # once a step (and window)
    rope(q, k, pos, angles, v_in=v, k_out=k_cache, v_out=v_cache, slots=slots)            # every layer
    attention(q, k_cache, v_cache, block_table, out=out)

(qknorm_rope_kv stores into the same caches, as their (slots, hkv, d) view.)
Lengths, tables and positions stay on the device, so a captured step can be
replayed while the requests grow.  What the kernels need of them is checked
there: a step whose numbers are out of bounds leaves a status (paged_tables)
or NaN rows (PagedAttention).
"""
from __future__ import annotations

import contextlib
import ctypes as C
from typing import Optional

from ._abi import CEV_BF16, CEV_F32, CEV_ROPE_LINEAR, CEV_ROPE_PLAIN, CEV_ROPE_WAVELENGTH, CEV_ROPE_YARN, CevError, PagedDesc, RopeScaling, calls, check, lib


_HERE = contextlib.nullcontext()


def _on(stream):
    """Allocations for work on `stream` (None: the current one)."""
    import torch
    return _HERE if stream is None else torch.cuda.stream(stream)


def _like(x):
    """A contiguous tensor of x's shape and type, without values."""
    import torch
    return torch.empty_like(x, memory_format=torch.contiguous_format)


def _i32(name: str, value) -> int:
    """value as an int that 32 bits hold (ctypes would wrap it)."""
    value = int(value)
    if not -(1 << 31) <= value < 1 << 31:
        raise CevError(-1, f"{name} {value} does not fit 32 bits")
    return value


def paged_tables(lengths, new_len, block_table, page_size: int, cu, pos, slots, free=None, ring=None, n_pages: Optional[int] = None,
                 lengths_out=None, ring_out=None, stream=None):
    """A step's bookkeeping on the device (cev_paged_tables): takes the pages
    that the new tokens need from the free ring, enters them in block_table,
    gives back the pages of ended requests (new_len -1), and writes the row
    offsets cu (requests + 1), each packed row's position and cache slot (0 and
    -1 behind the last row), the new lengths and the ring's new state.

    A page has one holder: the ring takes back every page that an ended
    request's row names.  Entries outside [0, n_pages) are passed over, so enter
    -1 where a page is another request's (a shared prefix) or was given back
    before (behind a window) and then end the request.  New tokens go to the
    last page that is not full: share whole pages.

    All tensors are int32 on the GPU: lengths, new_len (requests), block_table
    (requests, pages), pos and slots (the most rows of a step), free (n_pages)
    and ring (4): [head, count, status, 0], the free pages being
    free[(head + i) % n_pages] for i < count.  lengths_out and ring_out default
    to lengths and ring (in place); their values before the call do not matter.  ring[2] is 0, or says why the step was not
    made (cev_hip.h); its cu is then all 0.  free None: the block table holds
    the new tokens' pages already (n_pages is then required)."""
    if ring is None:
        raise CevError(-1, "paged_tables: ring is required (4 int32 values; it receives the status)")
    if n_pages is None:
        if free is None:
            raise CevError(-1, "paged_tables: n_pages is required without a free ring")
        n_pages = free.shape[0]
    calls().paged_tables(lengths, new_len, block_table, int(page_size), cu, pos, slots, int(n_pages), free, ring,
                         lengths if lengths_out is None else lengths_out, ring if ring_out is None else ring_out, stream)


def free_ring(n_pages: int, device, first: int = 0):
    """(free, ring) of a cache whose pages from `first` on are free."""
    import torch
    free = torch.arange(first, first + n_pages, dtype=torch.int32, device=device) % n_pages
    return free, torch.tensor([0, n_pages - first, 0, 0], dtype=torch.int32, device=device)


_SCALINGS = {"none": CEV_ROPE_PLAIN, "linear": CEV_ROPE_LINEAR, "yarn": CEV_ROPE_YARN, "wavelength": CEV_ROPE_WAVELENGTH}


class RotaryAngles:
    """The angles of rope(): pair i turns by theta^(-2i / rotary_dim) radians a
    position, scaled for long contexts (cev_rope_angles): "none", "linear"
    (factor), "yarn" (factor, original; pairs between low and high turns of the
    original context are blended, 1 and 32 by default) or "wavelength" (the
    same by wavelength; low and high 1 and 4)."""

    def __init__(self, theta: float, rotary_dim: int, device, scaling: str = "none", factor: float = 1.0, original: float = 0.0,
                 low: Optional[float] = None, high: Optional[float] = None, attention_factor: float = 0.0):
        import torch
        if scaling not in _SCALINGS:
            raise CevError(-2, f"rotary scaling {scaling!r} not supported ({', '.join(_SCALINGS)})")
        s = RopeScaling(_SCALINGS[scaling], _i32("rotary_dim", rotary_dim), float(theta), float(factor), float(original), 1.0 if low is None else float(low),
                        (4.0 if scaling == "wavelength" else 32.0) if high is None else float(high), float(attention_factor))
        steps = (C.c_uint64 * max(1, int(rotary_dim) // 2))()
        f = C.c_float()
        check(lib().cev_rope_angles(C.byref(s), steps, C.byref(f)))
        self.rotary_dim, self.factor = int(rotary_dim), f.value
        self.turns = list(steps)  # of 2^-64 turns a position
        signed = [x - (1 << 64) if x >> 63 else x for x in self.turns]
        self.steps = torch.tensor(signed, dtype=torch.int64, device=device)


def rope(q_in, k_in, pos, rot: RotaryAngles, interleaved: bool = False, transposed: bool = False, v_in=None, q_out=None, k_out=None,
         v_out=None, slots=None, stream=None):
    """Rotary positions of q (t, hq, d) and k (t, hkv, d) at pos (t) int32
    (cev_rope): pairs (i, i + rotary_dim / 2), or (2i, 2i + 1) with
    interleaved.  With slots (t) int32, k and v go to those slots of k_out and
    v_out, (pages, page_size, hkv, d) caches; a slot outside them stores
    nothing, and no two tokens may have the same one.  transposed: the gradient
    of q_in and k_in from that of q_out and k_out (the call itself records
    nothing for autograd).  Outputs may be their inputs.  Returns (q_out,
    k_out), with v_in also v_out."""
    if slots is not None and (k_out is None or (v_in is not None and v_out is None)):
        raise CevError(-1, "rope: slots need caches to store into")
    if stream is not None:  # (outputs that the call makes come from the current stream's pool)
        with _on(stream):
            q_out = _like(q_in) if q_out is None else q_out
            k_out = _like(k_in) if k_out is None else k_out
            v_out = _like(v_in) if v_in is not None and v_out is None else v_out
    return calls().rope(q_in, k_in, v_in, pos, rot.steps, rot.rotary_dim, rot.factor, interleaved, transposed, slots, q_out, k_out, v_out, stream)


class PagedAttention:
    """Attention of each request's new tokens, its last positions, over its
    pages (cev_paged_attention) for calls of one shape: q and out (t, hq, d),
    caches (n_pages, page_size, hkv, d), block_table (requests, pages).
    max_new: no request has more new tokens in a step (default t; a decoding
    step that says so is one launch less).  window: a
    row sees that many last keys, itself among them, and the first `sinks`
    ones; 0: all.  plan() makes the step's work list from cu and lengths on the
    device; every call until the next plan() uses it.  out may be q.  The object
    is made on the current stream, which other streams wait for as for a
    tensor; its workspace (17 MB for decoding steps, 85 to 152 MB for bf16
    steps with chunks) serves one step at a time."""

    def __init__(self, q, k_cache, block_table, max_new: Optional[int] = None, window: int = 0, sinks: int = 0, scale: Optional[float] = None):
        import torch
        if q.dim() != 3 or k_cache.dim() != 4 or block_table.dim() != 2:
            raise CevError(-1, "PagedAttention: q must be (t, hq, d), the cache (pages, page_size, hkv, d), the block table (requests, pages)")
        if k_cache.dtype != q.dtype or k_cache.shape[3] != q.shape[2]:
            raise CevError(-1, "PagedAttention: q and the cache must share the dtype and head_dim")
        if q.dtype not in (torch.float32, torch.bfloat16):
            raise CevError(-2, f"dtype {q.dtype} not supported (float32, bfloat16)")
        for x in (*q.shape, *k_cache.shape, *block_table.shape):
            _i32("size", x)
        d = PagedDesc()
        check(lib().cev_paged_desc_init(C.byref(d), CEV_F32 if q.dtype == torch.float32 else CEV_BF16, q.shape[1], k_cache.shape[2], q.shape[2],
                                        block_table.shape[0], q.shape[0], k_cache.shape[1], k_cache.shape[0], block_table.shape[1]))
        if max_new is not None:
            d.max_new = _i32("max_new", max_new)
        d.window, d.sinks = _i32("window", window), _i32("sinks", sinks)
        if scale is not None:
            d.scale = float(scale)
        n = C.c_size_t()
        check(lib().cev_paged_work_size(C.byref(d), C.byref(n)))
        self.desc = d
        self.work = torch.zeros(n.value, dtype=torch.uint8, device=q.device)

    def plan(self, cu, lengths, stream=None):
        """The step's work list: cu (requests + 1) and lengths (requests, new
        tokens included) as paged_tables writes them."""
        calls().paged_plan(self.desc, cu, lengths, self.work, stream)
        return self

    def __call__(self, q, k_cache, v_cache, block_table, out=None, stream=None):
        if out is None:
            with _on(stream):
                out = _like(q)
        calls().paged_attention(self.desc, q, k_cache, v_cache, block_table, out, self.work, stream)
        return out
