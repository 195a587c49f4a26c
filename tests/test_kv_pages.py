"""Page bookkeeping of paged caches: the oracle's properties and the refusals on CPU, exact results on a B200."""

import ctypes
import os
import re

import numpy as np
import pytest
import torch

import atrex
from atrex.src.nvidia.flash_attn.sm100 import kv_cache, kv_pages, runtime
from oracle import kv_pages_oracle

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _state(batch, page, width, pool, seed, empty=0.2, shared=True, full=0.2):
    """Random sequences over a shuffled pool; some rows share their finished pages with the row before."""
    r = np.random.RandomState(seed)
    order = r.permutation(pool)
    table, lens, refs, at = np.full((batch, width), -7, np.int32), np.zeros(batch, np.int32), np.zeros(pool, np.int32), 0
    for b in range(batch):
        if r.rand() < empty:
            continue
        n = int(r.randint(1, width * page + 1))
        if r.rand() < full:
            n = -(-n // page) * page
        pages, prefix = -(-n // page), 0
        if shared and b and r.rand() < 0.4:
            prefix = min(n, int(lens[b - 1])) // page
        if at + pages - prefix > pool:
            continue
        table[b, :prefix] = table[b - 1, :prefix]
        table[b, prefix:pages] = order[at:at + pages - prefix]
        at += pages - prefix
        lens[b] = n
        np.add.at(refs, table[b, :pages], 1)
    return table, lens, refs


def _parents(batch, seed):
    r = np.random.RandomState(seed)
    p = r.randint(0, batch, batch)
    kind = r.rand(batch)
    p[kind < 0.2] = -1                          # freed
    p[kind > 0.95] = batch + 3
    keep = (kind > 0.2) & (kind < 0.5)
    p[keep] = np.arange(batch)[keep]            # goes on as it is
    return p.astype(np.int32)


# ------------------------------------------------------------------ CPU
def test_oracle_keeps_the_counts():
    """Counts of the result are those of the result's table; every sequence reads the same tokens as before."""
    for seed in range(20):
        table, lens, refs = _state(9, 4, 6, 60, seed)
        parents = _parents(9, seed)
        cache = np.arange(60 * 4).reshape(60, 4)
        before = cache.copy()
        new_table, new_lens, new_refs, short = kv_pages_oracle.reassign(table, lens, refs, parents, [cache], 4)
        assert not short
        counted = np.zeros_like(refs)
        for b in range(9):
            used = new_table[b, : -(-new_lens[b] // 4)]
            np.add.at(counted, used, 1)
            if 0 <= parents[b] < 9:
                was = before[table[parents[b], : len(used)]].reshape(-1)[: new_lens[b]]
                assert np.array_equal(cache[used].reshape(-1)[: new_lens[b]], was)
            last = new_lens[b] % 4
            if last:                       # an unfinished page has one holder, unless it was shared before
                assert new_refs[used[-1]] == 1
        assert np.array_equal(counted, new_refs)
        t2, r2, page_map, n = kv_pages_oracle.compact(new_table, new_lens, new_refs, [cache], 4)
        assert (r2[:n] > 0).all() and not r2[n:].any() and r2.sum() == new_refs.sum()


def _cpu_call():
    return dict(block_table=torch.zeros(2, 3, dtype=torch.int32), seq_lens=torch.zeros(2, dtype=torch.int32),
                ref_counts=torch.zeros(8, dtype=torch.int32), caches=[torch.zeros(8, 16, 2, 64)])


@pytest.mark.parametrize("change,error,match", [
    (dict(caches=[]), ValueError, "at least one"),
    (dict(block_table=torch.zeros(2, 3)), ValueError, "block_table"),
    (dict(block_table=torch.zeros(3, 2, dtype=torch.int32).T), ValueError, "block_table"),
    (dict(seq_lens=torch.zeros(3, dtype=torch.int32)), ValueError, "one entry"),
    (dict(ref_counts=torch.zeros(7, dtype=torch.int32)), ValueError, "one page per entry"),
    (dict(ref_counts=torch.zeros(8, dtype=torch.int64)), ValueError, "ref_counts"),
    (dict(caches=[torch.zeros(8, 16, 128)]), ValueError, "num_pages, page_size"),
    (dict(caches=[torch.zeros(8, 16, 2, 64), torch.zeros(8, 32, 2, 64)]), ValueError, "one page size"),
    (dict(caches=[torch.zeros(8, 16, 64, 2).transpose(2, 3)]), NotImplementedError, "contiguous"),
    (dict(caches=[torch.zeros(1, 16, 2, 64).expand(8, 16, 2, 64)]), NotImplementedError, "expanded"),
    (dict(caches=[torch.zeros(8, 16, 2, 64, requires_grad=True)]), NotImplementedError, "inference-only"),
    (dict(), NotImplementedError, "CUDA devices only"),
])
def test_refusals(change, error, match):
    call = dict(_cpu_call(), **change)
    with pytest.raises(error, match=match):
        kv_pages.compact_pages(**call)
    with pytest.raises(error, match=match):
        kv_pages.reassign_sequences(**call, parents=torch.zeros(2, dtype=torch.int32))


@pytest.mark.parametrize("parents", [None, torch.zeros(2), torch.zeros(3, dtype=torch.int32)])
def test_parents_are_checked(parents):
    with pytest.raises(ValueError, match="parents"):
        kv_pages.reassign_sequences(**_cpu_call(), parents=parents)


def test_native_interface():
    with open(os.path.join(ROOT, "include", "atrex_kvpages_sm100.h")) as f:
        names = set(re.findall(r"ATREX_FA_API\s+\w+\s+(atrex_kvpages_\w+)\(", f.read()))
    lib = kv_pages.library()
    assert len(names) == 6
    for name in names:
        assert hasattr(lib, name), name
    assert lib.atrex_kvpages_sm100_reassign(None, None, 0, None) == 1
    p = kv_pages.Params()
    assert lib.atrex_kvpages_sm100_compact(ctypes.byref(p), None, 0, None) == 6
    p.struct_bytes, p.abi_version, p.page_size = ctypes.sizeof(p), 1, 16
    assert lib.atrex_kvpages_sm100_compact(ctypes.byref(p), None, 0, None) == 1     # no count
    p.count = 4096
    assert lib.atrex_kvpages_sm100_compact(ctypes.byref(p), None, 0, None) == 3     # no workspace
    p.batch = -1
    assert lib.atrex_kvpages_sm100_compact(ctypes.byref(p), 4096, 1 << 20, None) == 1
    assert lib.atrex_kvpages_sm100_workspace_bytes(0, 0) > 0


# ------------------------------------------------------------------ GPU
def _caches(pool, page, seed, kinds):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def fill(t):
        raw = t.view(torch.uint8) if t.is_contiguous() else t
        raw.copy_(torch.randint(0, 256, raw.shape, generator=g, device="cuda", dtype=torch.uint8))
        return t

    made = []
    for kind in kinds:
        if kind == "bf16":                      # token-major
            made.append(fill(torch.empty(pool, page, 2, 256, dtype=torch.uint8, device="cuda")).view(torch.bfloat16))
        elif kind == "pool":                    # K and V interleaved in one pool
            both = fill(torch.empty(pool, 2, page, 1, 64, dtype=torch.uint8, device="cuda"))
            made += [both[:, 0], both[:, 1]]
        elif kind == "fp4":                     # head-major codes and block scales
            k, ks, v, vs = kv_cache.allocate_fp4_kv_cache(pool, page, 3, 128)
            made += [fill(k), fill(ks.view(torch.uint8)), fill(v), fill(vs.view(torch.uint8))]
        elif kind == "gaps":                    # gaps between rows, heads and pages
            made.append(fill(torch.empty(pool + 1, page, 4, 48, dtype=torch.uint8, device="cuda"))[:-1, :, ::2, :40])
        else:                                   # odd widths: one byte at a time
            made.append(fill(torch.empty(pool, page, 3, 7, dtype=torch.uint8, device="cuda")))
    return made


def _host(caches):
    return [c.contiguous().view(torch.uint8).cpu().numpy().copy() for c in caches]


def _dev(*arrays):
    return [torch.from_numpy(a).cuda() for a in arrays]


def _check(got, want, caches, host):
    for g, w in zip(got, want):
        assert np.array_equal(g.cpu().numpy().reshape(np.shape(w)), w)
    for c, h in zip(caches, host):
        assert np.array_equal(c.contiguous().view(torch.uint8).cpu().numpy(), h)


ALL = ("bf16", "pool", "fp4", "gaps", "odd")


@pytest.mark.gpu
@pytest.mark.parametrize("batch,page,width,pool,kinds", [
    (1, 16, 1, 3, ("bf16",)), (2, 1, 5, 30, ("fp4", "odd")), (7, 16, 5, 60, ALL), (40, 32, 3, 200, ALL),
    (33, 5, 9, 500, ("gaps", "odd")), (1500, 16, 2, 9000, ("odd",)), (64, 64, 4, 400, ("bf16", "fp4")),
    (1024, 4, 2, 2048, ("odd",)), (1024, 4, 3, 4000, ("odd",)), (20, 8, 30, 2049, ("fp4",)), (64, 4, 128, 2048, ("odd",)), (300, 2, 30, 16384, ("odd",)), (50, 2, 6, 16385, ALL), (600, 2, 40, 40000, ("fp4",)),
])
def test_reassign(batch, page, width, pool, kinds):
    for seed in (0, 1):
        table, lens, refs = _state(batch, page, width, pool, seed + batch)
        parents = _parents(batch, seed)
        if seed:
            parents[::3] = parents[0]           # many forks of one row
        caches = _caches(pool, page, seed, kinds)
        host = _host(caches)
        args = _dev(table, lens, refs, parents)
        got = kv_pages.reassign_sequences(*args, caches)
        want = kv_pages_oracle.reassign(table, lens, refs, parents, host, page)
        _check(got, (*want[:3], np.array([want[3]])), caches, host)
        assert all(torch.equal(a, b) for a, b in zip(args, _dev(table, lens, refs, parents)))


@pytest.mark.gpu
@pytest.mark.parametrize("batch,page,width,pool,kinds", [
    (1, 16, 1, 3, ("bf16",)), (2, 1, 5, 30, ("fp4", "odd")), (7, 16, 5, 60, ALL), (40, 32, 3, 200, ALL),
    (33, 5, 9, 500, ("gaps", "odd")), (1500, 16, 2, 20000, ("odd",)), (30, 16, 4, 4096, ("fp4",)), (90, 2, 60, 8192, ("odd",)),
    (300, 2, 50, 16384, ("odd",)), (50, 2, 6, 16385, ALL), (5, 4, 3, 1025, ("pool",)), (2000, 2, 3, 9001, ("fp4",)),
])
def test_compact(batch, page, width, pool, kinds):
    table, lens, refs = _state(batch, page, width, pool, batch)
    caches = _caches(pool, page, 3, kinds)
    host = _host(caches)
    got = kv_pages.compact_pages(*_dev(table, lens, refs), caches)
    want = kv_pages_oracle.compact(table, lens, refs, host, page)
    _check(got, (*want[:3], np.array([want[3]])), caches, host)


@pytest.mark.gpu
def test_all_free_all_live_and_empty():
    table, lens, refs = _state(4, 16, 3, 12, 1, empty=0.0, shared=False, full=1.0)
    caches = _caches(12, 16, 0, ("bf16",))
    host = _host(caches)
    for r in (np.zeros_like(refs), np.ones_like(refs)):
        t, n = (table, lens) if r.any() else (np.full_like(table, -1), np.zeros_like(lens))
        got = kv_pages.compact_pages(*_dev(t, n, r), caches)
        want = kv_pages_oracle.compact(t, n, r, host, 16)
        _check(got, (*want[:3], np.array([want[3]])), caches, host)
    none = torch.empty(0, 3, dtype=torch.int32, device="cuda"), torch.empty(0, dtype=torch.int32, device="cuda")
    got = kv_pages.reassign_sequences(*none, torch.from_numpy(refs).cuda(), none[1], caches)
    assert got[0].shape == (0, 3) and got[3].item() == 0 and np.array_equal(got[2].cpu().numpy(), refs)
    got = kv_pages.compact_pages(*none, torch.from_numpy(refs).cuda(), caches)
    assert got[3].item() == (refs > 0).sum()


@pytest.mark.gpu
def test_shortage_changes_nothing():
    table, lens, refs = _state(6, 16, 3, 40, 2, empty=0.0, full=0.0)
    assert lens[1] % 16                          # row 1 ends inside a page
    free = np.flatnonzero(refs == 0)
    refs[free[2:]] = 1                           # held from outside the table: two pages are left for five forks
    parents = np.ones(6, np.int32)
    caches = _caches(40, 16, 0, ("fp4", "gaps"))
    host = _host(caches)
    before = [h.copy() for h in host]
    got = kv_pages.reassign_sequences(*_dev(table, lens, refs, parents), caches)
    want = kv_pages_oracle.reassign(table, lens, refs, parents, host, 16)
    assert want[3] == 3
    _check(got, (*want[:3], np.array([want[3]])), caches, before)


@pytest.mark.gpu
@pytest.mark.parametrize("caches", [17, 64, 65, 270])
def test_many_caches(caches):
    table, lens, refs = _state(8, 4, 3, 40, 5)
    store = torch.randint(0, 256, (caches, 40, 4, 1, 12), device="cuda", dtype=torch.uint8)
    host = _host(store.unbind())
    caches = list(store.unbind())
    parents = _parents(8, 1)
    got = kv_pages.reassign_sequences(*_dev(table, lens, refs, parents), caches)
    want = kv_pages_oracle.reassign(table, lens, refs, parents, host, 4)
    _check(got, (*want[:3], np.array([want[3]])), caches, host)
    got = kv_pages.compact_pages(got[0], got[1], got[2], tuple(caches))
    want = kv_pages_oracle.compact(*want[:3], host, 4)
    _check(got, (*want[:3], np.array([want[3]])), caches, host)


@pytest.mark.gpu
def test_single_tensor_and_sliced_table():
    table, lens, refs = _state(5, 16, 4, 40, 6)
    wide = torch.full((5, 11), 99999, dtype=torch.int32, device="cuda")
    wide[:, 2:6] = torch.from_numpy(table).cuda()
    cache = _caches(40, 16, 0, ("bf16",))[0]
    host = _host([cache])
    parents = _parents(5, 0)
    got = kv_pages.reassign_sequences(wide[:, 2:6], *_dev(lens, refs, parents), cache)
    want = kv_pages_oracle.reassign(table, lens, refs, parents, host, 16)
    _check(got, (*want[:3], np.array([want[3]])), [cache], host)


@pytest.mark.gpu
def test_captured_steps():
    """A captured step reads its tables again at every replay; another stream runs its own step meanwhile."""
    pool, page = 200, 16
    states = [_state(12, page, 5, pool, s) for s in (31, 32)]
    parents = [_parents(12, s) for s in (31, 32)]
    caches = _caches(pool, page, 0, ("fp4", "bf16"))
    host = _host(caches)
    args = _dev(*states[0], parents[0])
    kv_pages.reassign_sequences(*args, [c.clone() for c in caches])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = kv_pages.reassign_sequences(*args, caches)
        packed = kv_pages.compact_pages(got[0], got[1], got[2], caches)
    side, other = torch.cuda.Stream(), _caches(pool, page, 5, ("odd",))
    other_host = _host(other)
    for (table, lens, refs), par in zip(states, parents):
        for t, a in zip(args, (table, lens, refs, par)):
            t.copy_(torch.from_numpy(a))
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            side_got = kv_pages.reassign_sequences(*args, other)
        graph.replay()
        torch.cuda.synchronize()
        want = kv_pages_oracle.reassign(table, lens, refs, par, host, page)
        want_packed = kv_pages_oracle.compact(*want[:3], host, page)
        _check(got, (*want[:3], np.array([want[3]])), caches, host)
        _check(packed, (*want_packed[:3], np.array([want_packed[3]])), caches, host)
        side_want = kv_pages_oracle.reassign(table, lens, refs, par, other_host, page)
        _check(side_got, side_want[:3], other, other_host)


@pytest.mark.gpu
def test_beam_search_over_a_4_bit_cache():
    """Write, fork, write on, compact: every beam's attention equals that of its tokens written in one piece."""
    page, pool, hq, hkv, d, beams, width = 16, 64, 8, 2, 128, 4, 6
    g = torch.Generator().manual_seed(8)
    cache = kv_cache.allocate_fp4_kv_cache(pool, page, hkv, d)
    table = torch.full((beams, width), -1, dtype=torch.int32, device="cuda")
    lens = torch.zeros(beams, dtype=torch.int32, device="cuda")
    refs = torch.zeros(pool, dtype=torch.int32, device="cuda")
    history = [[] for _ in range(beams)]

    def write(caches, slots, rows):
        k, ks, v, vs = caches
        key, value = (torch.stack([r[i] for r in rows]).cuda() for i in (0, 1))
        kv_cache.write_kv_cache(key, value, k, v, slots.cuda(), key_block_scale=ks, value_block_scale=vs)

    def attend(caches, tab, n, q):
        k, ks, v, vs = caches
        return atrex.flash_attn_varlen_func(
            q, k, v, 1, torch.arange(beams + 1, dtype=torch.int32, device="cuda"), width * page, seqused_k=n,
            block_table=tab, causal=True, k_block_scale=ks, v_block_scale=vs, num_splits=1)

    for step in range(30):
        # every beam appends a token, in a new page where the last one is full (the engine's own bookkeeping)
        host_table, host_lens, host_refs = (t.cpu() for t in (table, lens, refs))
        slots = []
        for b in range(beams):
            n = int(host_lens[b])
            if n % page == 0:
                fresh = int(torch.nonzero(host_refs == 0)[-1 if b % 2 else 0])
                host_table[b, n // page], host_refs[fresh] = fresh, 1
            slots.append(int(host_table[b, n // page]) * page + n % page)
            history[b] = history[b] + [tuple(torch.randn(hkv, d, generator=g).bfloat16() for _ in range(2))]
            host_lens[b] += 1
        table, lens, refs = host_table.cuda(), host_lens.cuda(), host_refs.cuda()
        write(cache, torch.tensor(slots), [h[-1] for h in history])
        parents = torch.randint(0, beams, (beams,), generator=g).to(torch.int32)
        table, lens, refs, short = kv_pages.reassign_sequences(table, lens, refs, parents.cuda(), cache)
        assert short.item() == 0
        history = [history[p] for p in parents.tolist()]
        if step % 7 == 6:
            table, refs, _, live = kv_pages.compact_pages(table, lens, refs, cache)
            assert int(table.max()) < live.item()
        q = torch.randn(beams, hq, d, generator=g).bfloat16().cuda()
        whole = kv_cache.allocate_fp4_kv_cache(beams * width, page, hkv, d)
        plain = torch.arange(beams * width, dtype=torch.int32).view(beams, width)
        for b in range(beams):
            write(whole, torch.arange(len(history[b])) + b * width * page, history[b])
        assert torch.equal(attend(cache, table, lens, q), attend(whole, plain.cuda(), lens, q))


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [3, 5])
def test_tables_whose_rows_overlap(rows):
    """Rows one element apart, fewer of them than columns and more: the result is dense whatever the table's strides."""
    page, pool, width = 4, 40, 4
    base = torch.randperm(pool, generator=torch.Generator().manual_seed(3)).to(torch.int32)[: rows + width - 1]
    table = base.unfold(0, width, 1)
    lens = np.array([14, 9, 16, 0, 3], np.int32)[:rows]
    parents = np.array([0, 0, 1, 2, -1], np.int32)[:rows]
    refs = np.zeros(pool, np.int32)
    for b in range(rows):
        np.add.at(refs, table[b, : -(-lens[b] // page)].numpy(), 1)
    caches = _caches(pool, page, 0, ("odd",))
    host = _host(caches)
    on_device = base.cuda().unfold(0, width, 1)
    assert on_device.stride() == (1, 1)
    got = kv_pages.reassign_sequences(on_device, *_dev(lens, refs, parents), caches)
    want = kv_pages_oracle.reassign(table.numpy().copy(), lens, refs, parents, host, page)
    assert got[0].is_contiguous()
    _check(got, (*want[:3], np.array([want[3]])), caches, host)
    got = kv_pages.compact_pages(on_device, *_dev(lens, refs), caches)
    want = kv_pages_oracle.compact(table.numpy().copy(), lens, refs, host, page)
    assert got[0].is_contiguous()
    _check(got, (*want[:3], np.array([want[3]])), caches, host)


@pytest.mark.gpu
@pytest.mark.parametrize("sm_count", [1, 4, 8])
@pytest.mark.parametrize("batch,page,width,pool", [(7, 4, 5, 60), (300, 2, 50, 1024), (300, 2, 50, 16384), (50, 2, 6, 16385)])
def test_few_sms_through_the_c_abi(batch, page, width, pool, sm_count):
    """The block's sm_count sizes the grids; whatever it says, every page and every entry of the tables is written."""
    table, lens, refs = _state(batch, page, width, pool, 7)
    parents = _parents(batch, 7)
    caches = _caches(pool, page, 0, ("odd",))
    host = _host(caches)
    call = dict(zip(("block_table", "seq_lens", "ref_counts", "parents"), _dev(table, lens, refs, parents)))
    for name in ("reassign", "compact"):
        (block, _, pointers, scratch_bytes) = kv_pages._prepared(*list(call.values())[:3], caches, call["parents"])[1]
        p = kv_pages.Params.from_buffer_copy(block)
        bases = pointers(*[c.data_ptr() for c in caches])
        p.bases, p.sm_count = ctypes.addressof(bases), sm_count
        new = {f"new_{n}": torch.full_like(call[key], -9) for n, key in
               (("table", "block_table"), ("lens", "seq_lens"), ("refs", "ref_counts"))}
        new["page_map"], new["count"] = torch.full_like(call["ref_counts"], -9), torch.full_like(call["ref_counts"][:1], -9)
        for field, tensor in (*call.items(), *new.items()):
            setattr(p, field, tensor.data_ptr())
        scratch = torch.empty(scratch_bytes, dtype=torch.uint8, device="cuda")
        launch = getattr(kv_pages.library(), f"atrex_kvpages_sm100_{name}")
        runtime.raise_for_status(launch(ctypes.byref(p), scratch.data_ptr(), scratch_bytes,
                                        torch.cuda.current_stream().cuda_stream))
        if name == "reassign":
            want = kv_pages_oracle.reassign(table, lens, refs, parents, host, page)
            _check((new["new_table"], new["new_lens"], new["new_refs"], new["count"]), (*want[:3], np.array([want[3]])),
                   caches, host)
        else:
            want = kv_pages_oracle.compact(table, lens, refs, host, page)
            _check((new["new_table"], new["new_refs"], new["page_map"], new["count"]), (*want[:3], np.array([want[3]])),
                   caches, host)
