"""Page bookkeeping of the paged KV caches that ``flash_attn_varlen_func`` reads: forking, freeing and compacting.

A pool of ``num_pages`` pages backs any number of cache tensors ``[num_pages, page_size, heads, width]`` (K and V of
every layer, codes and block scales of 4-bit caches, ...); a row of ``block_table`` names the pages of one sequence,
``ref_counts[p]`` says how often page ``p`` is held (0: free).  Decisions and copies run on the device on the current
stream: no length or count is read on the host, so a step can be captured into a CUDA graph.  Metadata comes back in
new tensors; the caches are changed in place, only in pages that were free.

The reference leaves this to the serving engine.  There is no CPU fallback: without the native library the calls raise
``RuntimeError``.
"""

from __future__ import annotations

import ctypes
import threading

import torch

from . import runtime

ABI_VERSION = 1
_i64, _i32, _u32, _ptr = ctypes.c_int64, ctypes.c_int32, ctypes.c_uint32, ctypes.c_void_p


class Cache(ctypes.Structure):
    """Mirror of ``atrex_kvpages_sm100_cache`` (include/atrex_kvpages_sm100.h)."""

    _fields_ = [("page_stride", _i64), ("row_stride", _i64), ("head_stride", _i64), ("heads", _i32),
                ("row_bytes", _i32)]


class Params(ctypes.Structure):
    """Mirror of ``atrex_kvpages_sm100_params``; order and types must match the header."""

    _fields_ = (
        [("struct_bytes", _u32), ("abi_version", _u32)]
        + [(n, _ptr) for n in ("block_table", "seq_lens", "ref_counts", "parents", "new_table", "new_lens", "new_refs",
                               "page_map", "count")]
        + [("caches", ctypes.POINTER(Cache)), ("bases", _ptr), ("table_row_stride", _i64)]
        + [(n, _i32) for n in ("batch", "width", "num_pages", "page_size", "num_caches", "sm_count")]
    )


_bound = False


def library():
    global _bound
    lib = runtime.load_library()
    if not _bound:
        lib.atrex_kvpages_sm100_params_bytes.restype = ctypes.c_size_t
        lib.atrex_kvpages_sm100_cache_bytes.restype = ctypes.c_size_t
        lib.atrex_kvpages_sm100_workspace_bytes.restype = ctypes.c_uint64
        lib.atrex_kvpages_sm100_workspace_bytes.argtypes = [_i32, _i32]
        for name in ("reassign", "compact"):
            getattr(lib, f"atrex_kvpages_sm100_{name}").argtypes = [ctypes.POINTER(Params), _ptr, ctypes.c_uint64, _ptr]
        if (lib.atrex_kvpages_sm100_abi_version() != ABI_VERSION
                or lib.atrex_kvpages_sm100_params_bytes() != ctypes.sizeof(Params)
                or lib.atrex_kvpages_sm100_cache_bytes() != ctypes.sizeof(Cache)):
            raise RuntimeError("libatrex_fa_sm100.so does not match this Python binding (page blocks)")
        _bound = True
    return lib


def _validate(block_table, seq_lens, ref_counts, caches, parents=None):
    if not isinstance(caches, list) or not caches:
        raise ValueError("at least one cache is needed")
    named = [("block_table", block_table, 2), ("seq_lens", seq_lens, 1), ("ref_counts", ref_counts, 1)]
    if parents is not None:
        named.append(("parents", parents, 1))
    for name, t, rank in named:
        if not isinstance(t, torch.Tensor) or t.dtype != torch.int32 or t.ndim != rank or \
                (t.numel() and t.stride(-1) != 1):
            raise ValueError(f"{name} must be int32 of rank {rank} with contiguous rows")
    batch = block_table.shape[0]
    if seq_lens.shape != (batch,) or (parents is not None and parents.shape != (batch,)):
        raise ValueError("seq_lens and parents must have one entry per block_table row")
    for t in caches:
        if not isinstance(t, torch.Tensor) or t.ndim != 4:
            raise ValueError("caches must be [num_pages, page_size, heads, width] tensors")
        if t.shape[0] != ref_counts.shape[0] or t.shape[1] != caches[0].shape[1]:
            raise ValueError("caches must have one page per entry of ref_counts and one page size")
        if t.requires_grad:
            raise NotImplementedError("paged caches are inference-only")
        if min(t.shape[1:]) < 1:
            raise ValueError("caches must have at least one row, head and element per page")
        if t.shape[3] > 1 and t.stride(3) != 1:
            raise NotImplementedError("cache rows must be contiguous")
        if any(n > 1 and s == 0 for n, s in zip(t.shape, t.stride())):
            raise NotImplementedError("caches must not be expanded tensors")
    if any(t.device != block_table.device for t in (seq_lens, ref_counts, *caches)) or \
            (parents is not None and parents.device != block_table.device):
        raise ValueError("all tensors must be on one device")
    if block_table.device.type != "cuda":
        raise NotImplementedError("Atrex sm100 page bookkeeping runs on CUDA devices only")
    return caches


_LAYOUT_LIMIT = 64
_local = threading.local()


def _prepared(block_table, seq_lens, ref_counts, caches, parents):
    """``(caches, parameter block, bytes of scratch)`` of a call that passed the checks.

    A serving loop repeats one layout with fresh addresses: a call whose shapes, strides, types and devices already
    passed skips the checks, and the block with the caches' layouts is kept per host thread.  No tensor contents or
    identities enter the key."""
    try:
        caches = [caches] if isinstance(caches, torch.Tensor) else list(caches)
        key = tuple([(t.shape, t.stride(), t.dtype, t.device, t.requires_grad) for t in caches])
        key = (key, block_table.shape, block_table.stride(), block_table.dtype, block_table.device, seq_lens.shape,
               seq_lens.stride(), seq_lens.dtype, seq_lens.device, ref_counts.shape, ref_counts.stride(), ref_counts.dtype,
               ref_counts.device,
               None if parents is None else (parents.shape, parents.stride(), parents.dtype, parents.device))
    except (AttributeError, TypeError, RuntimeError):
        key = None                                  # not tensors of the usual kind: the checks say what is wrong
    layouts = getattr(_local, "layouts", None)
    if layouts is None:
        layouts = _local.layouts = {}
    entry = layouts.get(key) if key is not None else None
    if entry is None:
        caches = _validate(block_table, seq_lens, ref_counts, caches, parents)
        entries = (Cache * len(caches))()
        for e, t in zip(entries, caches):
            size = t.element_size()
            e.page_stride, e.row_stride, e.head_stride = (s * size for s in t.stride()[:3])
            e.heads, e.row_bytes = t.shape[2], t.shape[3] * size
        p = Params()
        p.struct_bytes, p.abi_version = ctypes.sizeof(Params), ABI_VERSION
        p.caches, p.table_row_stride = entries, block_table.stride(0)
        p.batch, p.width = block_table.shape
        p.num_pages, p.page_size, p.num_caches = ref_counts.shape[0], caches[0].shape[1], len(caches)
        entry = (p, entries, ctypes.c_void_p * len(caches),
                 library().atrex_kvpages_sm100_workspace_bytes(p.batch, p.num_pages))
        if len(layouts) >= _LAYOUT_LIMIT:
            layouts.clear()
        if key is not None:
            layouts[key] = entry
    return caches, entry


def _launch(name, block_table, seq_lens, ref_counts, caches, parents=None, with_map=False):
    caches, (p, _, pointers, scratch_bytes) = _prepared(block_table, seq_lens, ref_counts, caches, parents)
    device = block_table.device
    # The kernels write rows without gaps.  empty_like would order the result's dimensions by the given table's strides,
    # which need not be those of dense rows: rows of a table may overlap, as those of base.unfold(0, 4, 1) do.
    # torch.empty with a dtype and a device takes the host twice as long.
    new_table, new_refs = block_table.new_empty(block_table.shape), torch.empty_like(ref_counts)
    new_lens = torch.empty_like(seq_lens) if parents is not None else None
    page_map = torch.empty_like(ref_counts) if with_map else None
    count, scratch = block_table.new_empty(1), block_table.new_empty(scratch_bytes // 4)
    bases = pointers(*[t.data_ptr() for t in caches])
    p.bases = ctypes.addressof(bases)
    p.block_table, p.seq_lens, p.ref_counts = block_table.data_ptr(), seq_lens.data_ptr(), ref_counts.data_ptr()
    p.parents, p.new_lens = runtime._ptr_of(parents), runtime._ptr_of(new_lens)
    p.new_table, p.new_refs, p.page_map = new_table.data_ptr(), new_refs.data_ptr(), runtime._ptr_of(page_map)
    p.count = count.data_ptr()
    call = getattr(library(), name)
    if device.index == torch.cuda.current_device():
        code = call(ctypes.byref(p), scratch.data_ptr(), scratch_bytes, runtime._raw_stream(device))
    else:
        with torch.cuda.device(device):
            code = call(ctypes.byref(p), scratch.data_ptr(), scratch_bytes, runtime._raw_stream(device))
    if code:
        runtime.raise_for_status(code)
    return new_table, new_lens, new_refs, page_map, count


def reassign_sequences(block_table, seq_lens, ref_counts, parents, caches):
    """Fork and free the sequences of a batch in one step: ``(block_table, seq_lens, ref_counts, shortage)``, new.

    Row ``b`` continues the sequence that row ``parents[b]`` held before the call: ``b`` itself, another row (a fork, as
    in beam search or parallel sampling), or none when ``parents[b]`` lies outside ``[0, batch)`` (the row is freed).
    Finished pages are shared.  The unfinished last page of a sequence stays with the parent row if that continues
    itself, else with the lowest row that continues it; every other such row gets a page of its own, the lowest free
    ones in row order, into which the page's tokens are copied in every cache of ``caches`` (the rest of that page is
    left as it was).  Pages that the call frees are free after it, not during it.

    ``shortage`` (int32 ``[1]``) is 0, or the number of free pages that were missing; then nothing is changed and the
    returned tensors equal the given ones.  Entries past a sequence's last page come back as -1.
    """
    if parents is None:
        raise ValueError("parents must be int32 of rank 1 with contiguous rows")
    new_table, new_lens, new_refs, _, shortage = _launch("atrex_kvpages_sm100_reassign", block_table, seq_lens, ref_counts,
                                                         caches, parents)
    return new_table, new_lens, new_refs, shortage


def compact_pages(block_table, seq_lens, ref_counts, caches):
    """Move the live pages of a pool to its front: ``(block_table, ref_counts, page_map, num_live)``, new.

    With ``n`` live pages (``ref_counts > 0``), the ``i``-th live page at or behind page ``n`` moves to the ``i``-th
    free page before it, whole, in every cache of ``caches``; afterwards pages ``0 .. n - 1`` are live and the pool
    behind them can be given up.  ``page_map[p]`` (int32 ``[num_pages]``) is where page ``p`` is now, -1 for a free page:
    holders outside ``block_table`` update their page numbers with it.  ``num_live`` is int32 ``[1]``.  Entries past a
    sequence's last page come back as -1.
    """
    new_table, _, new_refs, page_map, num_live = _launch("atrex_kvpages_sm100_compact", block_table, seq_lens, ref_counts,
                                                         caches, with_map=True)
    return new_table, new_refs, page_map, num_live
