"""The 4-bit KV cache: its format and refusals on CPU, the quantising write and the attention over it on a B200.

The write is compared byte for byte with the 64-bit oracle.  The attention's tolerance is derived, not chosen:

* the output is rounded to BF16 once: 2^-8 |out| (half a step, relative);
* P is rounded to FP16 (2^-11 relative) and its FP32 arithmetic (scaling, ex2, rescaling, the sums) stays below 2^-16:
  together e_p = 2^-11 + 2^-16, relative to sum p |v| / sum p;
* a score is a sum of D exact products accumulated in FP32: its error is at most D 2^-23 sum |q_i k_i| scale, which
  moves p by that much relative (and the row's sum by as much again);
* FP16 ends at steps of 2^-24, so a stored 2^7 2^(s - m) below 2^-14 is off by up to 2^-25 absolute.  The reference m
  is at most the row's maximum, so the row's sum is at least 2^m, and p = 2^(s - m) / sum is off by at most 2^-32 per
  key: 2^-32 sum |v| over the keys of the row.
"""

import ctypes
import os
import re

import numpy as np
import pytest
import torch

import atrex
from atrex.src.nvidia.flash_attn.sm100 import kv4, kv_cache, runtime
from atrex.utils.device_target import DeviceTarget
from oracle import kv4_oracle

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


# ------------------------------------------------------------------ CPU: the format
def test_oracle_tables():
    every = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(every, kv4_oracle.E4M3)
    mid = (kv4_oracle.E2M1[1:] + kv4_oracle.E2M1[:-1]) / 2
    got = kv4_oracle.E2M1[kv4_oracle.nearest_code(mid, kv4_oracle.E2M1)]
    assert got.tolist() == [0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0]        # ties to the even code


def test_oracle_round_trip():
    """What the format can hold comes back unchanged; a stored value is never further off than half a gap."""
    r = np.random.RandomState(3)
    codes, scales = r.randint(0, 256, (40, 64), dtype=np.uint8), r.randint(8, 100, (40, 8), dtype=np.uint8)
    codes[:, ::8] = (codes[:, ::8] & 0xf0) | 7                         # a 6 in every block: its scale is the block's
    x = kv4_oracle.dequantise(codes, scales)
    again, scale_again, values = kv4_oracle.quantise(x)
    assert np.array_equal(values, x) and np.array_equal(scales, scale_again)
    x = torch.from_numpy(r.randn(50, 128)).bfloat16().float().numpy()
    _, scales, values = kv4_oracle.quantise(x)
    step = np.repeat(kv4_oracle.E4M3[scales], 16, -1)
    # largest gap of E2M1 is 2 steps; rounding the scale down (half a step in 16) lets the top saturate by 6/16
    assert np.all(np.abs(values - x) <= (1.0 + 6 / 16) * step + 1e-12)


def test_allocate_is_a_zero_cache():
    k, ks, v, vs = kv_cache.allocate_fp4_kv_cache(3, 16, 2, 128, device="cpu")
    assert k.shape == v.shape == (3, 16, 2, 64) and ks.shape == vs.shape == (3, 16, 2, 8)
    assert k.dtype == torch.uint8 and ks.dtype == torch.float8_e4m3fn
    assert not k.any() and not ks.view(torch.uint8).any()
    with pytest.raises(ValueError, match="multiple of 16"):
        kv_cache.allocate_fp4_kv_cache(3, 16, 2, 120, device="cpu")


# ------------------------------------------------------------------ CPU: refusals
@pytest.fixture
def as_b200(monkeypatch):
    from atrex.api import flash_attn

    monkeypatch.setattr(flash_attn, "detect_device_target", lambda device: DeviceTarget("nvidia", "sm100", "12.9", 0))
    yield flash_attn
    flash_attn._validated.clear()


def _call(hq=8, hkv=2, d=128, page=64):
    k, ks, v, vs = kv_cache.allocate_fp4_kv_cache(10, page, hkv, d, device="cpu")
    return dict(q=torch.zeros(6, hq, d, dtype=torch.bfloat16), k=k, v=v, max_seqlen_q=4,
                cu_seqlens_q=torch.tensor([0, 2, 6], dtype=torch.int32), max_seqlen_k=256, causal=True,
                seqused_k=torch.tensor([100, 200], dtype=torch.int32),
                block_table=torch.zeros(2, 4, dtype=torch.int32), k_block_scale=ks, v_block_scale=vs)


def test_calls_that_are_served(as_b200):
    assert atrex.can_use_flash_attn_varlen_func(**_call())
    assert atrex.can_use_flash_attn_varlen_func(**_call(hq=24, hkv=2, d=256, page=128))
    ones = torch.ones(2, 2)
    assert atrex.can_use_flash_attn_varlen_func(**_call(), k_descale=ones, v_descale=ones[:, :1].expand(2, 2),
                                                window_size=(100, 0), return_softmax_lse=True, num_splits=3)


@pytest.mark.parametrize("given,taken", [
    ((5, None), (5, -1)), ((2**31 - 1, 0), (2**30, 0)), ((2**32 + 5, 2**63), (2**30, 2**30)), ((-2**33 + 3, -2), (-1, -1))])
def test_windows_wider_than_32_bits(as_b200, given, taken):
    """They neither wrap to a small window nor to one that shows nothing."""
    seen = {}

    def validate(call, real=as_b200._validate_flash_attn_call):
        seen["result"] = real(call)
        raise NotImplementedError("stop here")

    as_b200._validate_flash_attn_call, real = validate, as_b200._validate_flash_attn_call
    try:
        assert not atrex.can_use_flash_attn_varlen_func(**dict(_call(), causal=False), window_size=given)
    finally:
        as_b200._validate_flash_attn_call = real
    assert seen["result"][1] == taken


BAD = [
    (dict(k_block_scale=None), ValueError, "block scales"),
    (dict(v_block_scale=None), ValueError, "block scales"),
    (dict(k_block_scale=torch.zeros(10, 64, 2, 8)), NotImplementedError, "float8_e4m3fn"),
    (dict(k=torch.zeros(10, 64, 2, 128, dtype=torch.bfloat16)), NotImplementedError, "uint8"),
    (dict(v_block_scale=torch.zeros(10, 64, 2, 16).to(torch.float8_e4m3fn)), ValueError, "head_dim / 16"),
    (dict(q=torch.zeros(6, 8, 128)), NotImplementedError, "bfloat16 Q"),
    (dict(q=torch.zeros(6, 8, 256, dtype=torch.bfloat16)), NotImplementedError, "head dimensions"),
    (dict(q=torch.zeros(6, 8, 128, dtype=torch.bfloat16, requires_grad=True)), NotImplementedError, "forward-only"),
    (dict(q_descale=torch.ones(2, 2)), NotImplementedError, "q_descale"),
    (dict(k_descale=torch.ones(2, 8)), ValueError, "descales"),
    (dict(softcap=20.0), NotImplementedError, "softcap"),
    (dict(softmax_scale=-1.0), NotImplementedError, "softmax_scale"),
    (dict(softmax_scale=float("nan")), NotImplementedError, "softmax_scale"),
    (dict(cp_world_size=2, cp_rank=0, cp_tot_seqused_k=torch.ones(2, dtype=torch.int32)), NotImplementedError,
     "context parallelism"),
    (dict(num_splits=257), NotImplementedError, "num_splits"),
    (dict(out=torch.zeros(6, 8, 128)), ValueError, "out must have"),
]


@pytest.mark.parametrize("change,error,match", BAD)
def test_calls_that_are_refused(as_b200, change, error, match):
    call = dict(_call(), **change)
    assert not atrex.can_use_flash_attn_varlen_func(**call)
    with pytest.raises(error, match=match):
        atrex.flash_attn_varlen_func(**call)


def test_packed_and_odd_pages_are_refused(as_b200):
    call = _call()
    k, ks = call["k"].reshape(-1, 2, 64), call["k_block_scale"].reshape(-1, 2, 8)
    packed = dict(call, k=k, v=k, k_block_scale=ks, v_block_scale=ks, block_table=None, seqused_k=None,
                  cu_seqlens_k=torch.tensor([0, 100, 300], dtype=torch.int32))
    assert not atrex.can_use_flash_attn_varlen_func(**packed)
    with pytest.raises(NotImplementedError, match="page_size"):
        atrex.flash_attn_varlen_func(**_call(page=48))
    odd = _call()
    store = torch.zeros(10, 2, 64, 9, dtype=torch.uint8).view(torch.float8_e4m3fn)
    odd["k_block_scale"] = store[..., :8].transpose(1, 2)
    with pytest.raises(NotImplementedError, match="boundaries"):
        atrex.flash_attn_varlen_func(**odd)


def test_other_caches_still_refuse_descales(as_b200):
    call = _call()
    bf16 = torch.zeros(10, 64, 2, 128, dtype=torch.bfloat16)
    call.update(k=bf16, v=bf16, k_block_scale=None, v_block_scale=None)
    assert atrex.can_use_flash_attn_varlen_func(**call)
    assert not atrex.can_use_flash_attn_varlen_func(**call, k_descale=torch.ones(2, 2))


def test_write_refusals():
    k, ks, v, vs = kv_cache.allocate_fp4_kv_cache(4, 16, 2, 128, device="cpu")
    key = torch.zeros(5, 2, 128, dtype=torch.bfloat16)
    slots = torch.zeros(5, dtype=torch.int64)

    def call(key=key, value=key, kc=k, vc=v, slots=slots, **more):
        args = dict(key_block_scale=ks, value_block_scale=vs)
        args.update(more)
        return kv_cache.write_kv_cache(key, value, kc, vc, slots, **args)

    for change, error, match in [
        (dict(key_block_scale=None), ValueError, "block scales"),
        (dict(kc=torch.zeros(4, 16, 2, 128, dtype=torch.bfloat16)), NotImplementedError, "uint8"),
        (dict(key=key[:4]), ValueError, "one shape"),
        (dict(key=key.float(), value=key.float()), NotImplementedError, "bfloat16"),
        (dict(slots=slots.int()), ValueError, "slot_mapping"),
        (dict(key_out=key[:3]), ValueError, "key's shape"),
        (dict(key_out=key.float()), NotImplementedError, "bfloat16"),
        (dict(), NotImplementedError, "CUDA devices only"),
    ]:
        with pytest.raises(error, match=match):
            call(**change)
    bf16 = torch.zeros(4, 16, 2, 128, dtype=torch.bfloat16)
    with pytest.raises(NotImplementedError, match="4-bit caches only"):
        kv_cache.write_kv_cache(key, key, bf16, bf16, slots, key_out=key)


# ------------------------------------------------------------------ CPU: the C ABI
def _header():
    with open(os.path.join(ROOT, "include", "atrex_kv4_sm100.h")) as f:
        return f.read()


def test_header_symbols_are_exported():
    lib = runtime.load_library()
    names = set(re.findall(r"ATREX_FA_API\s+\w+\s+(atrex_kv4_\w+)\(", _header()))
    assert len(names) == 6
    for name in names:
        assert hasattr(lib, name), name


def _plan_block(**change):
    p = kv4.Params()
    p.struct_bytes, p.abi_version = ctypes.sizeof(p), kv4.ABI_VERSION
    fa = p.fa
    fa.struct_bytes, fa.abi_version = ctypes.sizeof(runtime.Params), runtime.ABI_VERSION
    for name in ("q", "k", "v", "out", "cu_seqlens_q", "seqused_k", "block_table"):
        setattr(fa, name, 4096)
    p.k_block_scale = p.v_block_scale = 4096
    fa.q_row_stride, fa.q_head_stride, fa.out_row_stride, fa.out_head_stride = 1024, 128, 1024, 128
    for side in "kv":
        for axis, stride in (("page", 64 * 128), ("row", 64), ("head", 64 * 64)):
            setattr(fa, f"{side}_{axis}_stride", stride)
            setattr(p, f"{side}_scale_{axis}_stride", stride // 8)
    fa.batch, fa.total_q, fa.num_pages, fa.page_size, fa.max_pages_per_seq = 2, 2, 40, 64, 16
    fa.max_seqlen_q, fa.max_seqlen_k, fa.num_q_heads, fa.num_kv_heads, fa.head_dim = 1, 1024, 8, 2, 128
    fa.causal, fa.window_left, fa.window_right, fa.sm_count, fa.softmax_scale = 1, -1, -1, 148, 0.1
    for name, value in change.items():
        setattr(p if hasattr(kv4.Params, name) and name != "fa" else fa, name, value)
    return p


def _plan_status(**change):
    p, info = _plan_block(**change), runtime.PlanInfo()
    return kv4.library().atrex_kv4_sm100_plan(ctypes.byref(p), ctypes.byref(info)), info


@pytest.mark.parametrize("change,status", [
    (dict(), 0), (dict(batch=-1), 1), (dict(num_q_heads=7), 1), (dict(out=None), 1), (dict(block_table=None), 1),
    (dict(page_size=0), 1), (dict(k_block_scale=None), 1), (dict(dtype=1), 2), (dict(head_dim=64), 2),
    (dict(page_size=24), 2), (dict(softcap=1.0), 2), (dict(softmax_scale=0.0), 2), (dict(k_row_stride=8), 2),
    (dict(k_scale_row_stride=4), 2), (dict(k_page_stride=-64), 2), (dict(num_splits=300), 2), (dict(route=9), 1),
    (dict(q=4104), 2), (dict(return_lse=1), 1),
])
def test_native_refusals(change, status):
    assert _plan_status(**change)[0] == status


def test_native_plan():
    _, info = _plan_status(num_splits=4)             # up to eight splits of a small call join inside the kernel
    assert info.num_splits == 4 and info.kernel_launches == 1 and info.workspace_bytes == 0
    _, info = _plan_status(num_splits=9)
    assert info.num_splits == 9 and info.kernel_launches == 2
    assert info.workspace_bytes >= 9 * 2 * 8 * 129 * 4
    _, info = _plan_status(max_seqlen_k=0)
    assert info.num_splits == 1 and info.workspace_bytes == 0
    status, _ = _plan_status(batch=2 ** 30)
    assert status == 2
    assert kv4.library().atrex_kv4_sm100_plan(None, None) == 1
    assert kv4.library().atrex_kv4_sm100_write(None, None) == 1


def _write_status(tokens, heads, dim, **rows):
    """Status of the C entry for rows given as (address, token stride, head stride); 0 or a CUDA error without a device."""
    p = kv4.WriteParams()
    p.struct_bytes, p.abi_version = ctypes.sizeof(p), kv4.ABI_VERSION
    p.num_tokens, p.num_kv_heads, p.head_dim, p.page_size, p.num_pages = tokens, heads, dim, 16, 0
    p.slot_mapping = 4096
    for name, (base, token, head) in rows.items():
        setattr(p, name, base)
        setattr(p, f"{name}_token_stride", token)
        setattr(p, f"{name}_head_stride", head)
    return kv4.library().atrex_kv4_sm100_write(ctypes.byref(p), None)


def test_out_rows_that_overlap_are_refused(monkeypatch):
    """Against the bytes of every row, one by one.  No pool is behind the calls and no device here: a call that passes
    the checks ends at the device's."""
    if torch.cuda.is_available():
        pytest.skip("addresses are made up")
    r = np.random.RandomState(0)
    dim, refused, accepted = 16, 0, 0

    def taken(rows, tokens, heads):
        base, token, head = rows
        return [{base + 2 * (t * token + h * head) + b for b in range(2 * dim)} for t in range(tokens) for h in range(heads)]

    for _ in range(1500):
        tokens, heads = int(r.randint(1, 5)), int(r.randint(1, 4))
        strides = [(int(a), int(b)) for a, b in ((heads * dim, dim), (3 * heads * dim, dim), (dim, tokens * dim), (0, dim),
                                                 (heads * dim, 0), (48, 16), (32, 48))]
        strides = strides[r.randint(0, 4 if r.rand() < 0.7 else len(strides))]
        key, value = [(1 << 20) + 32 * int(r.randint(0, 30)) for _ in range(2)]
        rows = {"key": (key, *strides), "value": (value if r.rand() < 0.8 else key, *strides)}
        for name, own in (("key_out", key), ("value_out", value)):
            if r.rand() < 0.7:
                rows[name] = (own if r.rand() < 0.5 else (1 << 20) + 32 * int(r.randint(0, 60)), *strides)
        bad, sets = False, {name: taken(at, tokens, heads) for name, at in rows.items()}
        for out, own in (("key_out", "key"), ("value_out", "value")):
            if out not in rows:
                continue
            bad |= len(set().union(*sets[out])) < 2 * dim * tokens * heads
            for name in rows:
                if name != out and not (name == own and rows[name] == rows[out]):
                    bad |= bool(set().union(*sets[out]) & set().union(*sets[name]))
        assert (_write_status(tokens, heads, dim, **rows) == 1) == bad, (tokens, heads, rows)
        refused, accepted = refused + bad, accepted + (not bad)
    assert min(refused, accepted) > 300
    # rows of a fused QKV tensor lie between each other; other strides in the same range are refused, outside it are not
    fused = {"key": (4096, 384, 16), "value": (4096 + 2 * 128, 384, 16)}
    assert _write_status(9, 8, 16, key_out=fused["key"], value_out=fused["value"], **fused) != 1
    assert _write_status(9, 8, 16, key_out=(4096 + 2 * 256, 400, 16), **fused) == 1
    assert _write_status(9, 8, 16, key_out=(1 << 20, 128, 16), **fused) != 1
    assert _write_status(1, 8, 16, key_out=(4096, 128, 16), **fused) != 1        # one token: its stride says nothing


@pytest.mark.parametrize("d,resident", [(128, 3), (256, 2)])
def test_splits_join_in_the_kernel_within_one_wave(d, resident):
    """... of the CTAs that fit the SMs (by registers: three and two an SM); beyond it through scratch."""
    rows = {f"{side}_{kind}row_stride": d // w for side in "kv" for kind, w in (("", 2), ("scale_", 16))}
    wave = resident * 148
    for batch, splits in ((wave // 4, 4), (wave // 4 + 1, 4), (wave // 8, 8), (wave // 8 + 1, 8), (wave // 2 + 1, 2), (148, 4)):
        status, info = _plan_status(batch=batch, total_q=batch, num_q_heads=4, num_kv_heads=1, head_dim=d, num_splits=splits, **rows)
        assert status == 0 and info.num_splits == splits
        assert info.kernel_launches == (1 if batch * splits <= wave else 2)


def _prompt_plan(batch, max_q, total_q, hq, hkv, d, max_k, window=-1, route=2):
    rows = {f"{side}_{kind}row_stride": d // w for side in "kv" for kind, w in (("", 2), ("scale_", 16))}
    status, info = _plan_status(batch=batch, max_seqlen_q=max_q, total_q=total_q, num_q_heads=hq, num_kv_heads=hkv,
                                head_dim=d, max_seqlen_k=max_k, window_left=window, route=route,
                                max_pages_per_seq=-(-max_k // 64), **rows)
    assert status == 0
    return info


def test_long_prompts_are_not_split():
    """Splits that save a fraction of a round of work do not pay for the partial results they leave in scratch."""
    for batch, max_q, total_q, hq, hkv, max_k in ((4, 9984, 39936, 64, 8, 131072), (3, 1060, 2940, 32, 8, 12974),
                                                  (26, 1148, 11648, 24, 2, 45081), (309, 61, 6798, 64, 4, 93574)):
        info = _prompt_plan(batch, max_q, total_q, hq, hkv, 256, max_k)
        assert info.num_splits == 1 and info.workspace_bytes < 4096
    # few row tiles over a long context are split until the SMs have work
    for batch, max_q, total_q, hq, hkv, d, max_k, window in ((1, 16, 16, 16, 2, 256, 8192, -1), (1, 5, 5, 64, 4, 256, 14372, 4129),
                                                             (2, 100, 200, 8, 2, 256, 10000, -1), (1, 5, 5, 64, 4, 128, 16384, -1)):
        assert 8 <= _prompt_plan(batch, max_q, total_q, hq, hkv, d, max_k, window).num_splits <= 40
    assert _prompt_plan(8, 5, 40, 64, 4, 128, 8192).num_splits == 4          # 32 items: four splits fill 128 of 148 SMs


def test_scratch_of_automatic_splits_is_bounded():
    """At most three rounds of 128-row items are split, and only where their partial results cost less than they gain."""
    r = np.random.RandomState(4)
    heads = ((32, 8), (64, 8), (64, 4), (24, 2), (16, 2), (8, 1), (12, 1), (64, 1))
    for _ in range(4000):
        hq, hkv = heads[r.randint(len(heads))]
        batch, max_q, max_k = (int(2 ** r.uniform(0, top)) for top in (9, 13, 18))
        d, total_q = int(r.choice([128, 256])), batch * int(r.randint(1, max_q + 1))
        info = _prompt_plan(batch, max_q, total_q, hq, hkv, d, max_k, int(r.choice([-1, 1000])))
        assert info.workspace_bytes <= 2 ** 28 + 16 * batch + 1024       # partial results, and the plan of the row tiles
        if info.num_splits > 1:
            assert total_q * hq <= 3 * 148 * 128


# ------------------------------------------------------------------ GPU: the write
def _pool(layout, pages, page, heads, dim, fill=0xA5):
    """(codes, scales) in one of the layouts the attention call accepts, every byte ``fill``."""
    def tensor(width):
        if layout == "token":
            return torch.full((pages, page, heads, width), fill, dtype=torch.uint8, device="cuda")
        if layout == "head":
            return torch.full((pages, heads, page, width), fill, dtype=torch.uint8, device="cuda").transpose(1, 2)
        # gaps between rows and between pages
        store = torch.full((pages, 2, page * 2, heads, width), fill, dtype=torch.uint8, device="cuda")
        return store[:, 1, ::2]

    return tensor(dim // 2), tensor(dim // 16).view(torch.float8_e4m3fn)


def same_bytes(got, want):
    wrong = np.argwhere(got != want)
    first = [(tuple(i.tolist()), int(got[tuple(i)]), int(want[tuple(i)])) for i in wrong[:4]]
    assert not len(wrong), f"{len(wrong)} of {got.size} differ: {first}"


def _rows(tokens, heads, dim, seed, special):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(tokens, heads, dim, generator=g)
    x *= torch.exp(2 * torch.randn(tokens, heads, 1, generator=g))
    if special:
        inf, nan = float("inf"), float("nan")
        x[0, 0, :16] = 0.0
        x[0, 0, 16:32] = torch.tensor([6, 5, 3.5, 2.5, 1.75, 1.25, 0.75, 0.25, -5, -3.5, -2.5, -1.75, -0.25, -0.0, 0, 6])
        x[0, -1, :16] = torch.tensor([nan] + [1.0] * 15)
        x[0, -1, 16:32] = torch.tensor([inf, -inf] + [2.0] * 14)
        x[0, -1, 32:48] = torch.tensor([nan] * 16)
        x[-1, 0, :16] = 3e38
        x[-1, 0, 16:32] = 1e-30
        x[-1, 0, 32:48] = 2.0 ** -9 * 3          # a subnormal scale
        x[-1, 0, 48:64] = torch.tensor([nan, inf] + [0.5] * 14)
    return x.bfloat16()


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,heads,dim,page,layout,factor", [
    (1, 1, 128, 16, "head", None), (7, 2, 128, 16, "token", None), (130, 8, 128, 64, "head", "head"),
    (65, 3, 256, 32, "gaps", "one"), (33, 1, 16, 16, "token", None), (50, 5, 48, 64, "head", "head"),
    (700, 4, 128, 192, "gaps", None),
])
def test_write_is_exact(tokens, heads, dim, page, layout, factor):
    pages = tokens // page + 3
    key, value = (_rows(tokens, heads, dim, s, dim >= 128) for s in (tokens, tokens + 1))
    g = torch.Generator().manual_seed(5)
    slots = torch.randperm(pages * page, generator=g)[:tokens]
    slots[2::5] = -1                              # padding
    if tokens > 6:
        slots[5], slots[6] = pages * page, 2 ** 40    # past the pool: skipped
    kc, ks = _pool(layout, pages, page, heads, dim)
    vc, vs = _pool(layout, pages, page, heads, dim)
    factors = (None, None)
    if factor == "one":
        factors = torch.tensor([0.37], device="cuda"), torch.tensor([2.0 ** -5], device="cuda")
    elif factor == "head":
        factors = torch.rand(2, heads, generator=g).add_(0.01).cuda().unbind()
    outs = torch.full_like(key, 7.0).cuda(), torch.full_like(value, 7.0).cuda()
    kv_cache.write_kv_cache(key.cuda(), value.cuda(), kc, vc, slots.cuda(), *factors, key_block_scale=ks,
                            value_block_scale=vs, key_out=outs[0], value_out=outs[1])
    keep = (slots >= 0) & (slots < pages * page)
    at, row = (slots[keep] // page).numpy(), (slots[keep] % page).numpy()
    for x, c, s, f, out in ((key, kc, ks, factors[0], outs[0]), (value, vc, vs, factors[1], outs[1])):
        f = 1.0 if f is None else f.cpu().numpy()[..., None]
        codes, scales, values = kv4_oracle.quantise(x.float().numpy(), f)
        want_c = np.full(c.shape, 0xA5, np.uint8)
        want_s = np.full(s.shape, 0xA5, np.uint8)
        want_c[at, row], want_s[at, row] = codes[keep.numpy()], scales[keep.numpy()]
        same_bytes(s.view(torch.uint8).cpu().numpy(), want_s)
        same_bytes(c.cpu().numpy(), want_c)
        # stored values are exact in FP32 before their one rounding to BF16: 64 bits and FP32 round alike
        want = torch.from_numpy(values).float().bfloat16()
        want[~keep] = 7.0
        same_bytes(out.cpu().view(torch.int16).numpy(), want.view(torch.int16).numpy())


@pytest.mark.gpu
def test_write_in_place_and_strided_rows():
    """Rows taken out of a fused QKV tensor, and key_out = key."""
    page, heads, dim, tokens = 16, 2, 128, 21
    fused = _rows(tokens, 3 * heads, dim, 11, False).cuda()
    key, value = fused[:, heads:2 * heads], fused[:, 2 * heads:]
    want_k, want_v = (kv4_oracle.quantise(t.float().cpu().numpy()) for t in (key, value))
    kc, ks = _pool("head", 3, page, heads, dim)
    vc, vs = _pool("head", 3, page, heads, dim)
    slots = torch.arange(tokens, device="cuda")
    before = fused[:, :heads].clone()
    kv_cache.write_kv_cache(key, value, kc, vc, slots, key_block_scale=ks, value_block_scale=vs, key_out=key)
    assert torch.equal(key.cpu(), torch.from_numpy(want_k[2]).float().bfloat16())
    assert torch.equal(fused[:, :heads], before)
    got = vc.permute(0, 1, 2, 3).reshape(-1, heads, dim // 2)[:tokens].cpu().numpy()
    assert np.array_equal(got, want_v[0])
    empty = key[:0]
    kv_cache.write_kv_cache(empty, empty, kc, vc, slots[:0], key_block_scale=ks, value_block_scale=vs)
    with pytest.raises(NotImplementedError, match="32-byte"):
        odd = torch.zeros(tokens * heads * dim + 8, dtype=torch.bfloat16, device="cuda")[8:].view(tokens, heads, dim)
        kv_cache.write_kv_cache(odd, value, kc, vc, slots, key_block_scale=ks, value_block_scale=vs)


# ------------------------------------------------------------------ GPU: attention
def make_case(q_lens, kv_lens, hq, hkv, d, page, layout="head", seed=0, extra_pages=3, factors=False, sinks=False,
              q_gain=None, wide=2):
    r = np.random.RandomState(seed)
    g = torch.Generator().manual_seed(seed)
    counts = [-(-n // page) for n in kv_lens]
    pages = sum(counts) + extra_pages
    order = r.permutation(pages)
    table, at = np.full((len(kv_lens), max(counts + [1]) + wide), -1, np.int32), 0
    for b, n in enumerate(counts):
        table[b, :n] = order[at:at + n]
        at += n
    caches = []
    for _ in range(2):
        x = torch.randn(pages, page, hkv, d, generator=g) * torch.exp(0.5 * torch.randn(hkv, d, generator=g))
        codes, scales, _ = kv4_oracle.quantise(x.bfloat16().float().numpy())
        # what lies behind a request's last row and in pages nobody holds is garbage with NaN scales
        dead = np.ones((pages, page), bool)
        for b, n in enumerate(kv_lens):
            for i in range(n):
                dead[table[b, i // page], i % page] = False
        codes[dead], scales[dead] = 0xFF, 0x7F
        c, s = _pool(layout, pages, page, hkv, d)
        c.copy_(torch.from_numpy(codes))
        s.view(torch.uint8).copy_(torch.from_numpy(scales))
        caches += [c, s, codes, scales]
    total = sum(q_lens)
    q = torch.randn(total, hq, d, generator=g)
    if q_gain is not None:
        q = q * torch.tensor(q_gain)[torch.arange(total) % len(q_gain)][:, None, None]
    cu = np.concatenate([[0], np.cumsum(q_lens)]).astype(np.int32)
    case = dict(q=q.bfloat16(), cu=cu, kv_lens=np.asarray(kv_lens, np.int32), table=table, page=page,
                k=caches[0], ks=caches[1], v=caches[4], vs=caches[5], host=(caches[2], caches[3], caches[6], caches[7]),
                kf=None, vf=None, sinks=None)
    if factors:
        case["kf"], case["vf"] = torch.rand(2, len(kv_lens), hkv, generator=g).add_(0.3).unbind()
    if sinks:
        case["sinks"] = torch.randn(hq, generator=g).bfloat16()
    return case


def gpu_args(c, **more):
    dev = "cuda"
    q_lens = np.diff(c["cu"])
    args = dict(q=c["q"].to(dev), k=c["k"], v=c["v"], max_seqlen_q=int(max([1, *q_lens])),
                cu_seqlens_q=torch.from_numpy(c["cu"]).to(dev), max_seqlen_k=int(max([1, *c["kv_lens"]])),
                seqused_k=torch.from_numpy(c["kv_lens"]).to(dev), block_table=torch.from_numpy(c["table"]).to(dev),
                k_block_scale=c["ks"], v_block_scale=c["vs"], causal=True, return_softmax_lse=True)
    for name, key in (("k_descale", "kf"), ("v_descale", "vf"), ("s_aux", "sinks")):
        if c[key] is not None:
            args[name] = c[key].to(dev)
    args.update(more)
    return args


def check(c, out, lse, causal=True, window=(-1, -1), scale=None):
    kc, ks, vc, vs = c["host"]
    f = lambda t: None if t is None else t.numpy()  # noqa: E731
    k = kv4_oracle.dequantise(kc, np.where(ks == 0x7F, 0, ks))
    v = kv4_oracle.dequantise(vc, np.where(vs == 0x7F, 0, vs))
    want, want_lse, slack, weight, reach = kv4_oracle.attention(
        c["q"].double().numpy(), k, v, c["cu"], c["kv_lens"], c["table"], causal, window,
        None if c["sinks"] is None else c["sinks"].double().numpy(), f(c["kf"]), f(c["vf"]), scale)
    d = c["q"].shape[2]
    e_s = d * 2.0 ** -23 * slack                                       # [row, head]
    e_p = 2.0 ** -11 + 2.0 ** -16 + 2 * e_s
    got = out.double().cpu().numpy()
    tol = 2.0 ** -8 * np.abs(want) + e_p[..., None] * weight * (1 + 2.0 ** -8) + 2.0 ** -32 * reach + 1e-30
    assert np.isfinite(got).all()
    assert (np.abs(got - want) <= tol).all(), float((np.abs(got - want) / tol).max())
    if lse is not None:
        got = lse.double().cpu().numpy()
        empty = np.isneginf(want_lse)
        assert np.array_equal(np.isneginf(got), empty)
        tol = 2.0 ** -16 + e_s.T + 2.0 ** -21 * np.abs(np.where(empty, 0, want_lse))
        assert (np.abs(np.where(empty, 0, got - np.where(empty, 0, want_lse))) <= tol).all()


CASES = [
    # q_lens, kv_lens, hq, hkv, d, page, layout
    ([1], [1], 8, 2, 128, 16, "head"), ([1, 1, 1], [0, 17, 333], 8, 2, 128, 16, "token"),
    ([1] * 5, [31, 32, 33, 64, 129], 32, 8, 128, 64, "head"), ([1, 1], [700, 1500], 8, 1, 128, 192, "gaps"),
    ([1, 1], [255, 513], 24, 2, 128, 32, "token"), ([1, 2], [90, 1000], 16, 1, 128, 128, "head"),
    ([4, 4, 0, 4], [100, 4, 50, 777], 16, 4, 128, 64, "head"), ([3, 1, 7], [2, 40, 300], 6, 2, 128, 16, "head"),
    ([1, 1, 5], [1, 130, 600], 8, 1, 256, 128, "head"), ([2, 33], [64, 200], 12, 1, 256, 16, "token"),
    ([1, 40], [500, 41], 24, 2, 256, 64, "gaps"), ([70, 1, 130], [70, 260, 400], 8, 2, 128, 64, "head"),
    ([150], [149], 4, 4, 128, 32, "token"), ([300, 5], [310, 900], 16, 2, 256, 64, "head"),
    ([140, 20], [300, 20], 4, 2, 128, 16, "gaps"), ([100, 0, 3], [500, 70, 0], 6, 2, 128, 192, "token"),
    ([90, 1], [1000, 30], 16, 2, 128, 128, "head"), ([600], [600], 2, 1, 128, 32, "gaps"),
]


@pytest.fixture(params=["auto", "mma", "umma"])
def route(request, monkeypatch):
    """Both kernel families take every call; the launcher's own choice is the first."""
    monkeypatch.setattr(kv4, "DEFAULT_ROUTE", dict(auto=0, mma=1, umma=2)[request.param])


@pytest.mark.gpu
@pytest.mark.parametrize("q_lens,kv_lens,hq,hkv,d,page,layout", CASES)
@pytest.mark.parametrize("num_splits", [0, 1, 3, 11])
def test_attention(q_lens, kv_lens, hq, hkv, d, page, layout, num_splits, route):
    c = make_case(q_lens, kv_lens, hq, hkv, d, page, layout, seed=len(kv_lens) + d)
    out, lse = atrex.flash_attn_varlen_func(**gpu_args(c, num_splits=num_splits))
    check(c, out, lse)
    assert runtime.check_device_status("cuda:0") == 0           # no bounded wait expired


MANY = [
    # q rows per request, hq, hkv, d, page, longest: more row tiles than CTAs that fit the device at once
    ([1], 16, 8, 128, 64, 200), ([1], 8, 8, 128, 16, 40), ([1, 2, 0, 1], 16, 8, 128, 32, 700), ([3, 1], 24, 4, 128, 64, 300),
    ([1], 8, 4, 256, 64, 400), ([2, 1], 24, 4, 256, 16, 150), ([5, 0, 2], 8, 8, 128, 16, 90),
]


@pytest.mark.gpu
@pytest.mark.parametrize("rows,hq,hkv,d,page,longest", MANY)
@pytest.mark.parametrize("causal,window", [(True, (-1, -1)), (False, (20, 3))])
def test_many_requests(rows, hq, hkv, d, page, longest, causal, window, monkeypatch):
    """Requests from empty to long, in calls of several waves; a call gives the same bits again."""
    monkeypatch.setattr(kv4, "DEFAULT_ROUTE", 1)
    r = np.random.RandomState(longest)
    batch = 80 if hkv == 8 else 150
    q_lens = [rows[i % len(rows)] for i in range(batch)]
    kv_lens = [int(n) for n in r.randint(0, longest + 1, batch)]
    kv_lens[:4], kv_lens[-3:] = [0, 1, longest, 32], [33, 0, 0]
    c = make_case(q_lens, kv_lens, hq, hkv, d, page, seed=longest, factors=hq == 16, sinks=hq != 8)
    args = gpu_args(c, causal=causal, window_size=window)
    out, lse = atrex.flash_attn_varlen_func(**args)
    check(c, out, lse, causal, window)
    for _ in range(3):
        again, again_lse = atrex.flash_attn_varlen_func(**args)
        assert torch.equal(again, out) and torch.equal(again_lse, lse)


@pytest.mark.gpu
@pytest.mark.parametrize("d,splits", [(128, 1), (256, 1), (256, 2)])
def test_runs_of_requests_without_keys(d, splits, monkeypatch):
    """A CTA of the tcgen05 kernel meets several items without keys one after the other, then one with keys."""
    monkeypatch.setattr(kv4, "DEFAULT_ROUTE", 2)
    kv_lens = [0] * 700
    for b in (0, 1, 300, 699):
        kv_lens[b] = 70 + b % 50
    c = make_case([1] * 700, kv_lens, 2, 2, d, 64, seed=d, sinks=d == 256)
    out, lse = atrex.flash_attn_varlen_func(**gpu_args(c, num_splits=splits))
    check(c, out, lse)
    assert runtime.check_device_status("cuda:0") == 0


@pytest.mark.gpu
@pytest.mark.parametrize("d,hkv", [(128, 8), (256, 4)])
def test_one_long_request_among_many(d, hkv, monkeypatch):
    """One long request, ones of a single key, and ones without keys, replayed with other lengths."""
    monkeypatch.setattr(kv4, "DEFAULT_ROUTE", 1)
    batch = 640 // hkv
    kv_lens = [1] * batch
    kv_lens[batch // 2], kv_lens[3] = 20000, 0
    c = make_case([1] * batch, kv_lens, hkv, hkv, d, 64, seed=d, sinks=True)
    args = gpu_args(c)
    atrex.flash_attn_varlen_func(**args)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = atrex.flash_attn_varlen_func(**args)
    for change in ({}, {batch // 2: 777}, {i: 0 for i in range(batch)}):
        for b, n in change.items():
            c["kv_lens"][b] = n
        args["seqused_k"].copy_(torch.from_numpy(c["kv_lens"]))
        graph.replay()
        torch.cuda.synchronize()
        check(c, out, lse)


@pytest.mark.gpu
@pytest.mark.parametrize("causal,window", [(True, (0, 0)), (True, (33, 0)), (True, (500, 0)), (False, (-1, -1)),
                                           (False, (20, 10)), (False, (-1, 5)), (False, (40, -1))])
@pytest.mark.parametrize("q_lens,kv_lens,hq,hkv,d,page", [
    ([1, 3, 6], [700, 2, 260], 8, 2, 128, 16), ([2, 90], [1000, 200], 12, 1, 256, 64), ([160, 1], [400, 90], 16, 2, 128, 64)])
def test_masks(causal, window, q_lens, kv_lens, hq, hkv, d, page, route):
    c = make_case(q_lens, kv_lens, hq, hkv, d, page, seed=3, factors=True, sinks=hq == 8)
    for splits in (1, 2):
        out, lse = atrex.flash_attn_varlen_func(**gpu_args(c, causal=causal, window_size=window, num_splits=splits))
        check(c, out, lse, causal, window)


@pytest.mark.gpu
@pytest.mark.parametrize("q_lens", [[1, 1, 1], [9, 1, 64], [140, 3, 2]])
def test_factors_sinks_scale_and_q_range(q_lens, route):
    """Query rows of very unlike size: each is brought into FP16's range by its own power of two."""
    c = make_case(q_lens, [260, 0, 900], 16, 2, 128, 64, seed=9, factors=True, sinks=True,
                  q_gain=[1e30, 1e-30, 1.0, 300.0])
    # scores far beyond the softmax's range: only one key counts, so compare with a scale that keeps them moderate
    c["q"][torch.arange(c["q"].shape[0]) % 4 == 0] = 0
    out, lse = atrex.flash_attn_varlen_func(**gpu_args(c, softmax_scale=0.02, num_splits=0))
    check(c, out, lse, scale=0.02)
    c["q"] = make_case(q_lens, [260, 0, 900], 16, 2, 128, 64, seed=9, q_gain=[1e25])["q"]
    out, lse = atrex.flash_attn_varlen_func(**gpu_args(c, softmax_scale=1e-26))
    check(c, out, lse, scale=1e-26)


@pytest.mark.gpu
def test_rows_behind_the_last_sequence_stay(route):
    c = make_case([2, 3], [100, 40], 8, 2, 128, 16, seed=1)
    args = gpu_args(c)
    q = torch.cat([args["q"], torch.full((4, 8, 128), float("nan"), device="cuda", dtype=torch.bfloat16)])
    for splits in (1, 2):
        out = torch.full_like(q, 5.0)
        got, lse = atrex.flash_attn_varlen_func(**dict(args, q=q, out=out, num_splits=splits))
        assert got is out and (out[5:] == 5.0).all()
        check(c, out[:5], lse[:, :5])


@pytest.mark.gpu
@pytest.mark.parametrize("splits", [0, 1, 4, 11])
@pytest.mark.parametrize("q_lens", [[1, 1, 1], [4, 0, 6], [150, 1, 20]])
def test_a_nan_query_row_shows(q_lens, splits, route):
    """One query row of NaN in one head: its output is NaN and its LSE no number, all others what they were to be."""
    c = make_case(q_lens, [700, 30, 90], 8, 2, 128, 64, seed=5)
    out, lse = atrex.flash_attn_varlen_func(**gpu_args(c, num_splits=splits))
    check(c, out, lse)
    args = gpu_args(c, num_splits=splits)
    row, head = sum(q_lens) - 1, 5
    args["q"] = args["q"].clone()
    args["q"][row, head] = float("nan")
    got, got_lse = atrex.flash_attn_varlen_func(**args)
    assert got[row, head].isnan().all() and not got_lse[head, row].isfinite()
    got[row, head], got_lse[head, row] = out[row, head], lse[head, row]
    check(c, got, got_lse)


@pytest.mark.gpu
@pytest.mark.parametrize("q_lens", [[1, 1], [200, 30]])
def test_graph_replay_with_other_metadata_and_streams(q_lens, route):
    """A captured call reads lengths, pages and caches again at every replay; two streams do not share scratch."""
    a = make_case(q_lens, [1500, 700], 8, 2, 128, 64, seed=21)
    args = gpu_args(a)
    atrex.flash_attn_varlen_func(**args)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = atrex.flash_attn_varlen_func(**args)
    graph.replay()
    torch.cuda.synchronize()
    check(a, out, lse)
    a["kv_lens"] = np.array([333, 64] if q_lens[0] == 1 else [333, 30], np.int32)
    a["table"][:, :20] = a["table"][::-1, :20].copy()
    a["table"] = np.where(a["table"] < 0, 0, a["table"])
    a["host"] = tuple(t.cpu().numpy() if t.dtype == torch.uint8 else t.view(torch.uint8).cpu().numpy()
                      for t in (a["k"], a["ks"], a["v"], a["vs"]))
    for name in ("ks", "vs"):                       # the pages that are read now hold real rows only
        raw = a[name].view(torch.uint8)
        raw.copy_(torch.where(raw == 0x7F, torch.full_like(raw, 0x30), raw))
    a["host"] = tuple(t.cpu().numpy() if t.dtype == torch.uint8 else t.view(torch.uint8).cpu().numpy()
                      for t in (a["k"], a["ks"], a["v"], a["vs"]))
    args["seqused_k"].copy_(torch.from_numpy(a["kv_lens"]))
    args["block_table"].copy_(torch.from_numpy(a["table"]))
    graph.replay()
    torch.cuda.synchronize()
    check(a, out, lse)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    results = []
    for _ in range(5):
        with torch.cuda.stream(side):
            results.append(atrex.flash_attn_varlen_func(**args))
        results.append(atrex.flash_attn_varlen_func(**args))
    torch.cuda.synchronize()
    for got, got_lse in results:
        assert torch.equal(got, out) and torch.equal(got_lse, lse)


@pytest.mark.gpu
def test_stale_length_is_clamped(route):
    """A length beyond the table's width reads the table's pages only."""
    c = make_case([1], [128], 4, 1, 128, 64, seed=4, wide=0)
    args = gpu_args(c)
    args["seqused_k"].fill_(10 ** 6)
    out, lse = atrex.flash_attn_varlen_func(**args)
    check(c, out, lse)


@pytest.mark.gpu
@pytest.mark.parametrize("d,hq,hkv", [(128, 8, 2), (256, 6, 1)])
def test_prompt_and_decode_steps_together(d, hq, hkv):
    """Rows are written step by step through the 4-bit cache and attended after every step."""
    page, pages = 16, 12
    k, ks, v, vs = kv_cache.allocate_fp4_kv_cache(pages, page, hkv, d)
    g = torch.Generator().manual_seed(2)
    table = torch.randperm(pages, generator=g).to(torch.int32)[None]
    done = 0
    factor = torch.tensor([0.25] * hkv, device="cuda")
    for step in (70, 1, 1, 4):
        key, value = (torch.randn(step, hkv, d, generator=g).bfloat16().cuda() for _ in range(2))
        at = torch.arange(done, done + step)
        slots = (table[0, at // page].long() * page + at % page).cuda()
        kv_cache.write_kv_cache(key, value, k, v, slots, factor, factor, key_block_scale=ks, value_block_scale=vs)
        done += step
        q = torch.randn(step, hq, d, generator=g).bfloat16()
        c = dict(q=q, cu=np.array([0, step], np.int32), kv_lens=np.array([done], np.int32), table=table.numpy(), page=page,
                 k=k, ks=ks, v=v, vs=vs, kf=torch.full((1, hkv), 0.25), vf=torch.full((1, hkv), 0.25), sinks=None,
                 host=tuple(t.view(torch.uint8).cpu().numpy() for t in (k, ks, v, vs)))
        out, lse = atrex.flash_attn_varlen_func(**gpu_args(c))
        check(c, out, lse)


@pytest.mark.gpu
def test_pools_beyond_4_gb(monkeypatch):
    """Pages, slots and copies whose byte offsets do not fit 32 bits give the bits that a small pool gives."""
    from atrex.src.nvidia.flash_attn.sm100 import kv_pages

    heads, d, page, small = 8, 128, 64, 12
    pages = 2 ** 32 // (page * heads * d // 2) + 40
    g = torch.Generator().manual_seed(1)
    tokens = small * page
    key, value = (torch.randn(tokens, heads, d, generator=g).bfloat16().cuda() for _ in range(2))
    near = kv_cache.allocate_fp4_kv_cache(small, page, heads, d)
    far = [torch.empty(pages, heads, page, t.shape[3], dtype=t.dtype, device="cuda").transpose(1, 2) for t in near]
    slots = torch.arange(tokens, device="cuda")
    for pool, first in ((near, 0), (far, pages - small)):
        kv_cache.write_kv_cache(key, value, pool[0], pool[2], slots + first * page, key_block_scale=pool[1],
                                value_block_scale=pool[3])
    for a, b in zip(near, far):
        assert torch.equal(a.view(torch.uint8), b[pages - small:].view(torch.uint8))
    lens = torch.tensor([300, 1, 190], dtype=torch.int32, device="cuda")
    table = torch.tensor([[0, 1, 2, 3, 4], [5, -1, -1, -1, -1], [6, 9, 7, -1, -1]], dtype=torch.int32, device="cuda")
    far_table = torch.where(table >= 0, table + (pages - small), table)
    for rows in (1, 4, 40):
        q = torch.randn(3 * rows, 16, d, generator=g).bfloat16().cuda()
        cu = torch.arange(0, 3 * rows + 1, rows, dtype=torch.int32, device="cuda")
        for route in (1, 2):
            monkeypatch.setattr(kv4, "DEFAULT_ROUTE", route)
            got = [atrex.flash_attn_varlen_func(q, pool[0], pool[2], rows, cu, 300, seqused_k=lens, block_table=t, causal=False,
                                                num_splits=1, k_block_scale=pool[1], v_block_scale=pool[3])
                   for pool, t in ((near, table), (far, far_table))]
            assert torch.equal(*got)
    # a fork whose page is copied to the lowest free one, and everything moved to the front
    refs = torch.zeros(pages, dtype=torch.int32, device="cuda")
    refs[far_table[far_table >= 0].long()] = 1
    rows, lens, refs, shortage = kv_pages.reassign_sequences(far_table, lens, refs, torch.tensor([0, 0, 2], dtype=torch.int32,
                                                                                                device="cuda"), far)
    assert shortage.item() == 0 and rows[1].tolist() == [*(far_table[0, :4].tolist()), 0]
    for a, b in zip(near, far):
        assert torch.equal(b[0, :300 % page].view(torch.uint8), a[4, :300 % page].view(torch.uint8))
    rows, refs, _, live = kv_pages.compact_pages(rows, lens, refs, far)
    assert live.item() == 9 and int(rows.max()) == 8
    for b, i, src in ((0, 0, 0), (0, 3, 3), (0, 4, 4), (2, 0, 6), (2, 1, 9)):
        for a, c in zip(near, far):
            assert torch.equal(c[int(rows[b, i])].view(torch.uint8), a[src].view(torch.uint8))


@pytest.mark.gpu
@pytest.mark.parametrize("splits", [1, 2, 5, 9, 16])
@pytest.mark.parametrize("q_lens", [[1, 1, 1], [6, 0, 4], [130, 1, 20]])
@pytest.mark.parametrize("sinks", [False, True])
def test_the_lse_of_a_nan_query_row_is_nan(q_lens, splits, sinks, route):
    """However the splits join (in the kernel, over a cluster, through scratch): -inf would mean that no key was seen,
    and give the row weight 0 in a merge.  A row of NaN that sees no key is still empty."""
    c = make_case(q_lens, [700, 30, 500], 8, 2, 128, 64, seed=6, sinks=sinks)
    args = gpu_args(c, num_splits=splits)
    head = 5
    args["q"] = args["q"].clone()
    args["q"][:, head] = float("nan")
    out, lse = atrex.flash_attn_varlen_func(**args)
    assert out[:, head].isnan().all() and lse[head].isnan().all()
    others = [h for h in range(8) if h != head]
    assert out[:, others].isfinite().all() and lse[others].isfinite().all()
    args["seqused_k"].zero_()
    out, lse = atrex.flash_attn_varlen_func(**args)
    assert not out.any()
    want = args["s_aux"].float()[:, None].expand_as(lse) if sinks else torch.full_like(lse, -float("inf"))
    # |sink| log2 e + 7 stays below 16, where a rounding is off by 2^-21; the exponential and the products by 2^-22 relative
    assert torch.allclose(lse, want, rtol=2.0 ** -20, atol=2.0 ** -20)


@pytest.mark.gpu
@pytest.mark.parametrize("splits", [0, 1, 3])
@pytest.mark.parametrize("q_lens,d", [([1, 1, 1], 128), ([2, 9, 1], 256), ([1, 40, 150], 128)])
def test_factors_of_either_sign_and_zero(q_lens, d, splits, route):
    c = make_case(q_lens, [700, 30, 90], 8, 2, d, 64, seed=15, factors=True, sinks=True)
    c["kf"], c["vf"] = c["kf"] * torch.tensor([[1.0, -1], [-1, 0], [-1, 1]]), c["vf"] * torch.tensor([[-1.0, 1], [0, 1], [-1, -1]])
    out, lse = atrex.flash_attn_varlen_func(**gpu_args(c, num_splits=splits))
    check(c, out, lse)


@pytest.mark.gpu
@pytest.mark.parametrize("splits", [0, 1, 3, 9])
@pytest.mark.parametrize("q_lens,d", [([1, 1, 1], 128), ([2, 50, 1], 256), ([1, 40, 150], 128)])
def test_a_nan_factor_shows(q_lens, d, splits, route):
    """A NaN k_descale of one KV head: its rows are NaN if they see a key and empty if they see none; the others keep
    their bits."""
    c = make_case(q_lens, [700, 30, 90], 8, 2, d, 64, seed=16, factors=True)
    args = gpu_args(c, num_splits=splits)
    out, lse = atrex.flash_attn_varlen_func(**args)
    check(c, out, lse)
    args["k_descale"] = args["k_descale"].clone()
    args["k_descale"][1:, 1] = float("nan")
    got, got_lse = atrex.flash_attn_varlen_func(**args)
    rows, other = slice(q_lens[0], None), slice(0, q_lens[0])
    assert torch.equal(got[:, :4], out[:, :4]) and torch.equal(got_lse[:4], lse[:4])
    assert torch.equal(got[other], out[other]) and torch.equal(got_lse[:, other], lse[:, other])
    sees = ~lse[4:, rows].isneginf()
    assert got_lse[4:, rows][sees].isnan().all() and got[rows, 4:].transpose(0, 1)[sees].isnan().all()
    assert got_lse[4:, rows][~sees].isneginf().all() and not got[rows, 4:].transpose(0, 1)[~sees].any()
    assert bool((~sees).any()) == (q_lens[1] > 30)


@pytest.mark.gpu
def test_write_refuses_outs_that_overlap_its_inputs():
    heads, dim, tokens, page = 4, 128, 40, 16
    k, ks, v, vs = kv_cache.allocate_fp4_kv_cache(4, page, heads, dim)
    store = _rows(tokens + 1, heads, dim, 3, False).cuda()
    rows, shifted, other = store[:-1], store[1:], torch.zeros_like(store[:-1])
    slots, before = torch.arange(tokens, device="cuda"), store.clone()
    for outs in (dict(key_out=rows), dict(value_out=rows), dict(key_out=other, value_out=other), dict(key_out=shifted),
                 dict(value_out=other[:1].expand_as(rows))):
        with pytest.raises(ValueError, match="overlap"):
            kv_cache.write_kv_cache(rows, rows, k, v, slots, key_block_scale=ks, value_block_scale=vs, **outs)
    torch.cuda.synchronize()
    assert torch.equal(store, before) and not k.any() and not v.any()
    kv_cache.write_kv_cache(rows, rows, k, v, slots, key_block_scale=ks, value_block_scale=vs, key_out=other)
    want = torch.from_numpy(kv4_oracle.quantise(rows.float().cpu().numpy())[2]).float().bfloat16()
    assert torch.equal(other.cpu(), want) and torch.equal(store, before) and torch.equal(k, v)


@pytest.mark.gpu
@pytest.mark.parametrize("q_lens,kv_lens", [([1, 3, 6], [700, 2, 260]), ([160, 90], [400, 30])])
@pytest.mark.parametrize("window,same", [((2**31 - 1, 2**31 - 1), (-1, -1)), ((2**40, 5), (-1, 5)), ((33, 2**31 - 1), (33, -1))])
def test_very_wide_windows(q_lens, kv_lens, window, same, route):
    """As wide as an int32 or wider: what an unbounded side shows.  Through the C block, too, which is given as it is."""
    c = make_case(q_lens, kv_lens, 8, 2, 128, 64, seed=3)
    args = gpu_args(c, causal=False)
    out, lse = atrex.flash_attn_varlen_func(**args, window_size=window)
    check(c, out, lse, False, same)
    direct = {k: args[k] for k in ("q", "k", "v", "k_block_scale", "v_block_scale", "cu_seqlens_q", "seqused_k", "max_seqlen_q",
                                   "max_seqlen_k")}
    left, right = (min(w, 2**31 - 1) for w in window)
    out, lse = kv4.forward(**direct, page_table=args["block_table"], softmax_scale=128 ** -0.5, causal=False, window_left=left,
                           window_right=right, sink=None, out=None, return_lse=True, k_descale=None, v_descale=None,
                           num_splits=0)
    check(c, out, lse, False, same)


@pytest.mark.gpu
@pytest.mark.parametrize("q_lens,kv_lens,hq,hkv,d,page", [
    ([1] * 40, list(range(30, 1230, 30)), 16, 4, 128, 64), ([8, 3, 9, 1], [700, 500, 90, 1200], 64, 4, 128, 128),
    ([20, 40, 1], [1000, 60, 300], 24, 2, 256, 64), ([300, 150, 2], [600, 150, 700], 16, 2, 128, 16)])
@pytest.mark.parametrize("splits", [0, 3])
def test_a_call_gives_the_same_bits_again(q_lens, kv_lens, hq, hkv, d, page, splits, route):
    c = make_case(q_lens, kv_lens, hq, hkv, d, page, seed=77, factors=True, sinks=True)
    args = gpu_args(c, num_splits=splits)
    out, lse = atrex.flash_attn_varlen_func(**args)
    for _ in range(5):
        again, again_lse = atrex.flash_attn_varlen_func(**args)
        assert torch.equal(again, out) and torch.equal(again_lse, lse)
