"""What the entry points of attention by formula and rules, the 8-bit cache and the page tables refuse, without a GPU; and their
restatements against independent ones."""
import ctypes

import pytest
import torch

from oracle import scored as os_


@pytest.fixture(scope="module")
def lib():
    import importlib.util
    import os
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    spec = importlib.util.spec_from_file_location("stof_build", os.path.join(root, "sc25-stof-ad_b200", "build.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    mod.build_library()
    from stof_b200 import _lib
    return _lib.lib()


ONE = ctypes.c_void_p(16)


def _rules(**kw):
    from stof_b200 import _lib
    r = _lib.ScoreRules(softmax_scale=0.125)
    for name, value in kw.items():
        setattr(r, name, value)
    return r


def _scored(lib, rules=None, null_rules=False, dtype=0, batch=1, heads=2, kv_heads=1, q_len=8, k_len=8, dim=64, stride=64, q=ONE, k=ONE):
    from stof_b200 import _lib
    s = _lib.strides3((stride, stride, stride))
    r = ctypes.byref(rules or _rules()) if not null_rules else None
    return lib.stof_scored_attn(q, k, ONE, ONE, dtype, batch, heads, kv_heads, q_len, k_len, dim, s, s, s, s, r, None, None)


@pytest.mark.parametrize("kw,code,text", [
    (dict(dim=96), -1, b"head_dim"), (dict(heads=3, kv_heads=2), -1, b"multiple"), (dict(dtype=1), -1, b"fp16 or bf16"), (dict(dtype=3), -1, b"fp16 or bf16"),
    (dict(k_len=0), -1, b"no keys"), (dict(q=None), -1, b"null pointer"), (dict(k=ctypes.c_void_p(24)), -1, b"16-byte"), (dict(stride=60), -1, b"strides"),
    (dict(stride=0), -1, b"strides"), (dict(stride=-64), -1, b"strides"), (dict(q_len=-1), -1, b"bad shape"), (dict(k_len=1 << 30), -1, b"2^29"),
    (dict(null_rules=True), -1, b"null rules"), (dict(rules=dict(softmax_scale=0.0)), -1, b"softmax_scale"), (dict(rules=dict(softmax_scale=float("nan"))), -1, b"softmax_scale"),
    (dict(rules=dict(softcap=-1.0)), -1, b"softcap"), (dict(rules=dict(softcap=float("inf"))), -1, b"softcap"), (dict(rules=dict(window=-1)), -1, b"window"),
    (dict(rules=dict(distance_bias=16, bias_radius=2049)), -1, b"radius"), (dict(rules=dict(distance_bias=16, bias_radius=-1)), -1, b"radius"),
    (dict(rules=dict(prefix_lens=16)), -1, b"causal"), (dict(rules=dict(documents=16), q_len=9), -1, b"documents"),
    (dict(rules=dict(documents=16, documents_stride=200000), k_len=131073), -4, b"131072"), (dict(rules=dict(documents=16, documents_stride=4), batch=2), -1, b"row stride")])
def test_scored_attn_refusals(lib, kw, code, text):
    kw = dict(kw)
    if "rules" in kw:
        kw["rules"] = _rules(**kw["rules"])
    assert _scored(lib, **kw) == code and text in lib.stof_last_error()


def test_scored_attn_of_nothing(lib):
    assert _scored(lib, batch=0) == 0 and _scored(lib, q_len=0) == 0


def _cache(lib, rules=None, dtype=0, cache_dtype=3, pages=4, page=16, kv_heads=1, dim=64, width=2, stride=2, requests=1, tokens=1, heads=2, table=ONE, workspace=ONE,
           nbytes=1 << 30, st=64, q=ONE):
    from stof_b200 import _lib
    s = _lib.strides3((st, st, st))
    return lib.stof_cache_attn(q, ONE, dtype, s, s, ONE, ONE, ONE, ONE, cache_dtype, pages, page, kv_heads, dim, table, stride, width, ONE, requests, tokens, heads,
                               ctypes.byref(rules or _rules()), workspace, nbytes, None, None)


@pytest.mark.parametrize("kw,code,text", [
    (dict(dim=80), -1, b"head_dim"), (dict(page=24), -1, b"page size"), (dict(page=256), -1, b"page size"), (dict(heads=3, kv_heads=2), -1, b"multiple"),
    (dict(dtype=3), -1, b"fp16 or bf16"), (dict(cache_dtype=0), -1, b"int8 or e4m3"), (dict(stride=1), -1, b"row stride"), (dict(table=None), -1, b"block table"),
    (dict(workspace=None), -3, b"workspace"), (dict(nbytes=64), -3, b"workspace"), (dict(st=4), -1, b"strides"), (dict(q=ctypes.c_void_p(8)), -1, b"16-byte"),
    (dict(width=1 << 27, stride=1 << 27), -1, b"2^30"), (dict(rules=dict(window=-2)), -1, b"window"), (dict(rules=dict(softcap=-2.0)), -1, b"softcap"),
    (dict(rules=dict(softmax_scale=-1.0)), -1, b"softmax_scale"), (dict(rules=dict(distance_bias=16, bias_radius=5000)), -1, b"radius"), (dict(tokens=-1), -1, b"bad shape")])
def test_cache_attn_refusals(lib, kw, code, text):
    kw = dict(kw)
    if "rules" in kw:
        kw["rules"] = _rules(**kw["rules"])
    assert _cache(lib, **kw) == code and text in lib.stof_last_error()


def test_cache_attn_of_nothing(lib):
    assert _cache(lib, requests=0) == 0 and _cache(lib, tokens=0) == 0
    assert lib.stof_cache_attn_workspace_bytes(0, 1, 2, 1, 64, 16, 4) == 0
    assert lib.stof_cache_attn_workspace_bytes(4, 1, 8, 2, 64, 16, 64) > 0


def _append(lib, cache_dtype=3, pages=4, page=16, kv_heads=1, dim=64, dtype=0, st=64, tokens=1, k=ONE, slots=ONE):
    s = (ctypes.c_longlong * 3)(st, st, st)
    return lib.stof_cache_append(ONE, ONE, ONE, ONE, cache_dtype, pages, page, kv_heads, dim, k, ONE, dtype, s, s, slots, tokens, None, None)


@pytest.mark.parametrize("kw,text", [
    (dict(cache_dtype=0), b"int8 or e4m3"), (dict(page=8), b"page size"), (dict(dim=32), b"head_dim"), (dict(dtype=1), b"fp16 or bf16"), (dict(st=4), b"strides"),
    (dict(k=None), b"null"), (dict(slots=None), b"null"), (dict(k=ctypes.c_void_p(8)), b"16-byte"), (dict(pages=1 << 28), b"32-bit slots"), (dict(tokens=-1), b"bad shape"),
    (dict(kv_heads=0), b"bad shape")])
def test_cache_append_refusals(lib, kw, text):
    assert _append(lib, **kw) == -1 and text in lib.stof_last_error()


def test_cache_append_refuses_one_page_for_keys_and_values(lib):
    assert _append(lib) == -1 and b"of their own" in lib.stof_last_error()


def test_cache_append_of_nothing(lib):
    assert _append(lib, tokens=0) == 0


@pytest.mark.parametrize("kw,text", [
    (dict(page=10), b"page size"), (dict(requests=-1), b"negative"), (dict(width=-1), b"negative"), (dict(stride=1), b"row stride"), (dict(count=None), b"null"),
    (dict(slots=None), b"null"), (dict(lengths=None), b"null")])
def test_page_tables_refusals(lib, kw, text):
    a = dict(lengths=ONE, requests=2, stride=4, width=4, count=ONE, page=16, slots=ONE)
    a.update(kw)
    rc = lib.stof_page_tables(a["lengths"], ONE, a["requests"], ONE, a["stride"], a["width"], ONE, 8, a["count"], a["page"], a["slots"], 4, ONE, ONE, ONE, None, None)
    assert rc == -1 and text in lib.stof_last_error()


def test_operators_refuse_cpu_tensors(lib):
    import stof_b200
    x = torch.zeros(1, 2, 8, 64, dtype=torch.float16)
    pages, scales = torch.zeros(4, 2, 16, 64, dtype=torch.int8), torch.zeros(4, 2)
    i32 = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(stof_b200.StofError, match="CUDA"):
        stof_b200.scored_attention(x, x, x)
    with pytest.raises(stof_b200.StofError, match="CUDA"):
        stof_b200.cache_attention(x, pages, pages, scales, scales, i32[None], i32)
    with pytest.raises(stof_b200.StofError, match="CUDA"):
        stof_b200.cache_append(pages, pages, scales, scales, x[0], x[0], i32)
    with pytest.raises(stof_b200.StofError, match="CUDA"):
        stof_b200.page_tables(i32, i32, i32[None], i32, i32, 16, 0)


def test_restated_attention_equals_torch():
    """Where torch's own masked softmax says the same."""
    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(2, 4, 20, 64, generator=g), torch.randn(2, 2, 30, 64, generator=g), torch.randn(2, 2, 30, 64, generator=g))
    kk, vv = k.repeat_interleave(2, 1).double(), v.repeat_interleave(2, 1).double()
    on = torch.ones(20, 30, dtype=torch.bool).tril(10)
    want = torch.softmax((q.double() @ kk.transpose(2, 3) / 8).masked_fill(~on, -float("inf")), 3) @ vv
    assert torch.allclose(os_.scored_attention(q, k, v, causal=True), want, atol=1e-12)


def test_restated_append_and_cache_attention_agree_with_unquantised():
    """int8 entries within half a step of what was written; attention over them as over those values."""
    g = torch.Generator().manual_seed(2)
    pages, scales = torch.zeros(5, 2, 16, 64, dtype=torch.int8), torch.zeros(5, 2)
    x = torch.randn(40, 2, 64, generator=g).half()
    slots = torch.tensor([3 * 16 + i for i in range(16)] + [16 + i for i in range(16)] + [i for i in range(8)], dtype=torch.int32)
    os_.cache_append(pages, scales, x, slots)
    rows = os_.cache_rows(pages, scales, torch.tensor([3, 1, 0]), 40, 1)
    step = torch.cat((scales[3, 1].repeat(16), scales[1, 1].repeat(16), scales[0, 1].repeat(8))).double()[:, None]
    assert bool(((rows - x[:, 1].double()).abs() <= step * 0.5001).all())


def test_restated_page_tables():
    table, stack, slots, starts, count, missing = os_.page_tables([17, 0, 40], [16, 20, 0], [[5, -1, -1], [2, 3, -1], [-1, -1, -1]], [7, 8, -1, -1], 2, 16, 43)
    assert missing == 0 and starts == [0, 1, 1, 41] and count == 0
    assert table[0][:2] == [5, 3] and table[2] == [2, 8, 7]
    assert slots[:2] == [3 * 16, 2 * 16] and slots[41:] == [-1, -1]


def test_cache_attn_refuses_rows_beyond_32_bits(lib):
    assert _cache(lib, heads=64, kv_heads=1, tokens=(1 << 24) + 1) == -1 and b"2^30" in lib.stof_last_error()
    assert lib.stof_cache_attn_workspace_bytes(1, (1 << 24) + 1, 64, 1, 64, 16, 4) == 0


def test_page_tables_refuse_tables_beyond_32_bits(lib):
    rc = lib.stof_page_tables(ONE, ONE, 1 << 16, ONE, 1 << 15, 1 << 15, ONE, 8, ONE, 16, ONE, 4, ONE, ONE, ONE, None, None)
    assert rc == -1 and b"2^31 entries" in lib.stof_last_error()
