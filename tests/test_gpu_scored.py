"""Attention by formula and rules, the paged 8-bit cache and its tables, against their definitions in 64 bits."""
import math

import pytest
import torch

from oracle import scored as os_

pytestmark = pytest.mark.gpu
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def _rand(shape, seed, scale=1.0, dtype=torch.float16):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype)


def _bound(want, v_max, dtype):
    """What rounding allows, in absolute terms.  u = eps / 2 of the type.  The output is rounded once (u |want|).  P is rounded once for
    the product: u relative to every p, so u sum(p |v|) / sum(p) <= u max|v|.  Scores up to 64 in units of log2 carry fp32 errors of a few
    2^-24 * 64, the exponentials of at most 1e-4 (the polynomial one), the tanh 7e-6 relative of up to 60: together below 6e-4 of
    sum(p |v|) / sum(p).  In fp16 a small P loses relative accuracy below 2^-14: 2^-25 absolute each, beside a largest P of at least 2^-1."""
    u = torch.finfo(dtype).eps / 2
    return u * want.abs() + (u + 6e-4) * v_max + 1e-6


def _check(got, want, v, dtype):
    assert got.dtype == dtype and got.shape == want.shape
    assert bool(torch.isfinite(got).all())
    err = (got.double().cpu() - want).abs()
    over = err - _bound(want, float(v.abs().max()), dtype)
    assert float(over.max()) <= 0, f"off by {float(err.max()):.3e}, bound exceeded by {float(over.max()):.3e}"


def _status():
    from stof_b200 import _lib
    torch.cuda.synchronize()
    _lib.check_status(torch.device("cuda"), "test")


def _both(q, k, v, dtype=torch.float16, **rules):
    import stof_b200
    dev = {n: (x.cuda() if isinstance(x, torch.Tensor) else x) for n, x in rules.items()}
    got = stof_b200.scored_attention(q.cuda(), k.cuda(), v.cuda(), **dev)
    _status()
    vmax = v.clone()
    if rules.get("key_lens") is not None:
        for b in range(v.shape[0]):
            vmax[b, :, int(rules["key_lens"][b]):] = 0
    _check(got, os_.scored_attention(q, k, v, **rules), vmax.double(), dtype)
    return got


def _lens(values):
    return torch.tensor(values, dtype=torch.int32)


def _table(heads, radius, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(heads, 2 * radius + 1, generator=g)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("q_len,k_len", [(1, 1), (1, 130), (127, 127), (128, 128), (129, 257), (300, 300)])
def test_scored_plain_and_causal(dim, dtype, q_len, k_len):
    t = TYPES[dtype]
    q, k, v = _rand((2, 2, q_len, dim), 1, 2.0, t), _rand((2, 2, k_len, dim), 2, 1.0, t), _rand((2, 2, k_len, dim), 3, 1.0, t)
    _both(q, k, v, t)
    _both(q, k, v, t, causal=True)


def _rules(name, B, H, Sk):
    g = torch.Generator().manual_seed(7)
    docs = torch.randint(1, 90, (B, Sk), generator=g).cumsum(1) // 1500
    return {
        "cap": dict(softcap=30.0), "cap far": dict(softcap=1.5), "cap middle": dict(softcap=14.0), "cap tiny": dict(softcap=1e-3), "cap huge": dict(softcap=1e6), "slopes": dict(slopes=torch.rand(H, generator=g)),
        "slopes causal": dict(slopes=torch.rand(H, generator=g), causal=True), "table": dict(distance_bias=_table(H, 20, 5)),
        "table 0": dict(distance_bias=_table(H, 0, 5)), "table wide causal": dict(distance_bias=_table(H, 2048, 6), causal=True),
        "everything": dict(softcap=20.0, slopes=torch.rand(H, generator=g), distance_bias=_table(H, 33, 8), causal=True, window=150,
                           prefix_lens=_lens([min(70, Sk)] + [0] * (B - 1)), key_lens=_lens([Sk] + [Sk - 3] * (B - 1)), documents=docs.int()),
        "window": dict(window=40), "window causal": dict(window=140, causal=True), "window 1": dict(window=1), "window wide": dict(window=1 << 40, causal=True),
        "prefix": dict(causal=True, prefix_lens=_lens([0] + [min(200, Sk)] * (B - 1))),
        "prefix past the keys": dict(causal=True, prefix_lens=_lens([10 * Sk] + [-5] * (B - 1))),
        "window prefix": dict(causal=True, window=30, prefix_lens=_lens([min(5, Sk)] + [min(129, Sk)] * (B - 1))),
        "documents": dict(documents=docs.int()), "documents causal": dict(documents=docs.int(), causal=True),
        "documents shuffled": dict(documents=torch.randint(-2, 3, (B, Sk), generator=g).int()),
        "one document": dict(documents=torch.full((B, Sk), 4, dtype=torch.int32)),
        "padded": dict(key_lens=_lens([Sk] + [max(1, Sk // 2)] * (B - 1))), "padded to nothing": dict(key_lens=_lens([0] + [1] * (B - 1))),
        "padded beyond": dict(key_lens=_lens([Sk + 100] + [-7] * (B - 1))), "padded causal": dict(key_lens=_lens([128] + [Sk - 1] * (B - 1)), causal=True),
    }[name]


ALL_RULES = ["cap", "cap far", "cap middle", "cap tiny", "cap huge", "slopes", "slopes causal", "table", "table 0", "table wide causal", "everything", "window", "window causal", "window 1", "window wide",
             "prefix", "prefix past the keys", "window prefix", "documents", "documents causal", "documents shuffled", "one document", "padded",
             "padded to nothing", "padded beyond", "padded causal"]


@pytest.mark.parametrize("name", ALL_RULES)
@pytest.mark.parametrize("dim,dtype,q_len,k_len", [(64, "fp16", 333, 333), (128, "bf16", 140, 400)])
def test_scored_rules(name, dim, dtype, q_len, k_len):
    t = TYPES[dtype]
    q, k, v = _rand((2, 4, q_len, dim), 11, 2.0, t), _rand((2, 2, k_len, dim), 12, 1.0, t), _rand((2, 2, k_len, dim), 13, 1.0, t)
    _both(q, k, v, t, **_rules(name, 2, 4, k_len))


@pytest.mark.parametrize("name", ["slopes causal", "table", "window causal", "window prefix", "documents causal", "padded causal", "everything"])
@pytest.mark.parametrize("dim,dtype", [(64, "bf16"), (128, "fp16")])
def test_scored_rules_two_stretches_per_block(name, dim, dtype):
    """Enough heads that a block takes 256 rows: the two stretches want different tiles."""
    t = TYPES[dtype]
    q, k, v = _rand((2, 40, 500, dim), 21, 2.0, t), _rand((2, 2, 650, dim), 22, 1.0, t), _rand((2, 2, 650, dim), 23, 1.0, t)
    rules = _rules(name, 2, 40, 650)
    import stof_b200
    dev = {n: (x.cuda() if isinstance(x, torch.Tensor) else x) for n, x in rules.items()}
    got = stof_b200.scored_attention(q.cuda(), k.cuda(), v.cuda(), **dev)
    _status()
    for h in (0, 19, 20, 39):                            # the definition head by head is slow: both K/V heads, first and last of a group
        one = {n: (x[h:h + 1] if n in ("slopes", "distance_bias") else x) for n, x in rules.items()}
        _check(got[:, h:h + 1], os_.scored_attention(q[:, h:h + 1], k[:, h // 20:h // 20 + 1], v[:, h // 20:h // 20 + 1], **one), v.double(), t)


def test_scored_more_queries_than_keys():
    """Positions of the first queries are negative: nothing for them under a causal mask."""
    q, k, v = _rand((1, 2, 200, 64), 31, 2.0), _rand((1, 2, 70, 64), 32), _rand((1, 2, 70, 64), 33)
    assert not _both(q, k, v, causal=True)[:, :, :130].any()
    _both(q, k, v, window=50)
    _both(q, k, v, slopes=torch.tensor([0.5, 0.1]))


def test_scored_without_keys_or_queries():
    import stof_b200
    q = _rand((1, 2, 5, 64), 1).cuda()
    none = torch.empty(1, 2, 0, 64, dtype=torch.float16, device="cuda")
    assert not stof_b200.scored_attention(q, none, none).any()
    assert stof_b200.scored_attention(none, q, q).shape == (1, 2, 0, 64)
    assert stof_b200.scored_attention(q[:0], q[:0], q[:0]).shape == (0, 2, 5, 64)


def test_scored_padding_may_hold_anything():
    q, k, v = _rand((2, 2, 300, 64), 41, 2.0), _rand((2, 2, 300, 64), 42), _rand((2, 2, 300, 64), 43)
    lens = _lens([200, 129])
    clean = _both(q, k, v, key_lens=lens)
    for b, n in enumerate(lens.tolist()):
        k[b, :, n:] = math.nan
        v[b, :, n:] = math.nan
        v[b, :, n::2] = math.inf
    import stof_b200
    got = stof_b200.scored_attention(q.cuda(), k.cuda(), v.cuda(), key_lens=lens.cuda())
    _status()
    assert torch.equal(got, clean)


def test_scored_lowest_and_infinite_bias():
    """A bias of the type's lowest values keeps its row a softmax; minus infinity takes keys out, a row of nothing else is zero."""
    q, k, v = _rand((1, 2, 140, 64), 51, 2.0), _rand((1, 2, 140, 64), 52), _rand((1, 2, 140, 64), 53)
    low = torch.full((2, 41), -65504.0)
    _both(q, k, v, distance_bias=low)
    half = _table(2, 20, 9)
    half[0, :20] = -math.inf
    half[1] = -math.inf
    got = _both(q, k, v, distance_bias=half)
    assert not got[:, 1].any()


def test_scored_nan_comes_out():
    import stof_b200
    q, k, v = _rand((1, 2, 140, 64), 51, 2.0), _rand((1, 2, 140, 64), 52), _rand((1, 2, 140, 64), 53)
    q[0, 1, 7] = math.nan
    got = stof_b200.scored_attention(q.cuda(), k.cuda(), v.cuda(), causal=True).cpu()
    _status()
    assert bool(torch.isnan(got[0, 1, 7]).all()) and int(torch.isnan(got).sum()) == 64


@pytest.mark.parametrize("dim", [64, 128])
def test_scored_layouts(dim):
    """Slices of a fused projection, expanded heads, odd strides and addresses: the same bits as packed tensors."""
    import stof_b200
    B, H, S = 2, 4, 150
    qkv = _rand((B, S, 3, H, dim), 61).cuda()
    q, k, v = (qkv[:, :, i].transpose(1, 2) for i in range(3))
    want = stof_b200.scored_attention(q.contiguous(), k.contiguous(), v.contiguous(), causal=True)
    out = torch.zeros(B, S, H, dim, dtype=torch.float16, device="cuda")
    got = stof_b200.scored_attention(q, k, v, causal=True, out=out.transpose(1, 2))
    assert got.data_ptr() == out.data_ptr() and torch.equal(out.transpose(1, 2), want)
    wide = torch.zeros(B, H, S, dim + 3, dtype=torch.float16, device="cuda")
    wide[..., 1:dim + 1] = q
    assert torch.equal(stof_b200.scored_attention(wide[..., 1:dim + 1], k, v, causal=True), want)
    flat = torch.zeros(k.numel() + 1, dtype=torch.float16, device="cuda")
    flat[1:] = k.contiguous().view(-1)
    assert torch.equal(stof_b200.scored_attention(q, flat[1:].view(B, H, S, dim), v, causal=True), want)
    assert torch.equal(stof_b200.scored_attention(q, k.mT.contiguous().mT, v, causal=True), want)
    one = k[:, :1]
    assert torch.equal(stof_b200.scored_attention(q, one.expand(B, H, S, dim), v, causal=True),
                       stof_b200.scored_attention(q, one.expand(B, H, S, dim).contiguous(), v, causal=True))
    assert torch.equal(stof_b200.scored_attention(q[:1].expand(B, H, S, dim), k, v)[0], stof_b200.scored_attention(q[:1], k[:1], v[:1])[0])
    docs = (torch.arange(2 * S, device="cuda").view(S, 2) // 40).int().t().contiguous().t()           # (S, 2): its columns are strided
    assert torch.equal(stof_b200.scored_attention(q, k, v, documents=docs.t()), stof_b200.scored_attention(q, k, v, documents=docs.t().contiguous()))
    _status()


def test_scored_equals_the_row_wise_operator():
    import stof_b200
    q, k, v = (_rand((2, 3, 256, 64), i).cuda() for i in range(3))
    want = stof_b200.rowwise_attn_full(q, k, v, True).view(2, 256, 3, 64).transpose(1, 2)
    got = stof_b200.scored_attention(q, k, v, causal=True)
    assert float((got.float() - want.float()).abs().max()) <= 4e-3


# ------------------------------------------------------------------------------------------ the cache
def _cache(lengths, heads, page, dim, entry, seed, spare=3, width=None):
    """Pages in random order with random entries; what lies behind a request's keys is NaN where the type has one."""
    g = torch.Generator().manual_seed(seed)
    blocks = [-(-n // page) for n in lengths]
    pages = sum(blocks) + spare
    order = torch.randperm(pages, generator=g).tolist()
    table = torch.zeros(len(lengths), width or max(max(blocks), 1), dtype=torch.int32)
    most = os_.ENTRY_MAX[entry]

    def entries():
        x = (torch.randn(pages, heads, page, dim, generator=g) * most / 4).clamp(-most, most)
        return (x.round() if entry == torch.int8 else x).to(entry)

    k, v = entries(), entries()
    for b, n in enumerate(lengths):
        for i in range(blocks[b]):
            table[b, i] = order.pop()
        if n % page and entry != torch.int8:
            for x in (k, v):
                x.view(torch.uint8)[table[b, blocks[b] - 1].item(), :, n % page:] = 0x7F
    scales = [(torch.rand(pages, heads, generator=g) + 0.5) * 4 / most for _ in range(2)]
    return k, v, *scales, table, torch.tensor(lengths, dtype=torch.int32)


def _both_cache(q, cache, **rules):
    import stof_b200
    k, v, ks, vs, table, lengths = cache
    dev = {n: (x.cuda() if isinstance(x, torch.Tensor) else x) for n, x in rules.items()}
    got = stof_b200.cache_attention(q.cuda(), *(x.cuda() for x in cache), **dev)
    _status()
    finite = torch.where(torch.isnan(v.float()), 0.0, v.float())
    _check(got, os_.cache_attention(q, *cache, **rules), finite.double() * vs.double()[:, :, None, None], q.dtype)
    return got


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("entry", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("heads,kv_heads,tokens,dtype", [(2, 2, 1, "fp16"), (8, 2, 1, "bf16"), (8, 1, 2, "fp16"), (6, 2, 7, "bf16")])
def test_cache_attention(dim, entry, page, heads, kv_heads, tokens, dtype):
    lengths = [1, page, page + 1, 0, 333, 63, 64, 700]
    _both_cache(_rand((len(lengths), tokens, heads, dim), 71, 2.0, TYPES[dtype]), _cache(lengths, kv_heads, page, dim, entry, 72))


@pytest.mark.parametrize("rules", [dict(softcap=3.0), dict(softcap=50.0), dict(softcap=1e6), dict(softcap=1e-3), dict(window=1), dict(window=70), dict(slopes=torch.tensor([0.5, 0.01, 0.2, 0.0])),
                                   dict(distance_bias=_table(4, 30, 5)), dict(distance_bias=_table(4, 0, 5)), dict(softmax_scale=0.3),
                                   dict(softcap=20.0, window=200, slopes=torch.tensor([0.5, 0.01, 0.2, 0.0]), distance_bias=_table(4, 128, 6))])
@pytest.mark.parametrize("tokens", [1, 3])
def test_cache_attention_rules(rules, tokens):
    lengths = [500, 2, 1, 130, 64]                       # shorter than the new tokens, too: those in front of the request see nothing
    _both_cache(_rand((5, tokens, 4, 128), 81, 2.0, torch.bfloat16), _cache(lengths, 2, 32, 128, torch.float8_e4m3fn, 82), **rules)


def test_cache_attention_long_and_short_requests():
    """Requests over several thread blocks, several requests in one; more requests than a block has threads."""
    _both_cache(_rand((2, 1, 4, 64), 91, 2.0), _cache([9000, 5], 1, 64, 64, torch.int8, 92))
    g = torch.Generator().manual_seed(3)
    lengths = [int(x) for x in torch.randint(0, 90, (300,), generator=g)]
    _both_cache(_rand((300, 1, 2, 64), 93, 2.0), _cache(lengths, 2, 16, 64, torch.int8, 94))


def test_cache_attention_uneven_scales():
    """P is rounded relative to the largest scale a warp has met, whichever page comes first."""
    k, v, ks, vs, table, lengths = _cache([320], 1, 16, 64, torch.int8, 95)
    for order in (1.0, -1.0):
        vs[table[0].long(), 0] = torch.exp2(order * torch.linspace(-12, 12, table.shape[1])) / 32
        _both_cache(_rand((1, 1, 2, 64), 96, 2.0), (k, v, ks, vs, table, lengths))
    vs[table[0, :10].long()] = 0.0
    _both_cache(_rand((1, 1, 2, 64), 96, 2.0), (k, v, ks, vs, table, lengths))
    ks[:] = 0.0
    _both_cache(_rand((1, 1, 2, 64), 96, 2.0), (k, v, ks, vs, table, lengths))


def test_cache_attention_large_bf16_queries():
    """bf16 has fp32's range; the products run in fp16."""
    cache = _cache([200, 77], 2, 32, 64, torch.int8, 97)
    q = _rand((2, 1, 4, 64), 98, 1.0)
    big = (q.float() * 2.0 ** 100).bfloat16()
    got = _both_cache(big, cache, softmax_scale=2.0 ** -102)
    assert float((got.float() - _both_cache(q.bfloat16(), cache, softmax_scale=0.25).float()).abs().max()) == 0


def test_cache_attention_nan_comes_out_and_stays_in_its_row():
    import stof_b200
    cache = _cache([200, 77], 2, 32, 64, torch.int8, 97)
    q = _rand((2, 1, 4, 64), 98, 1.0)
    clean = stof_b200.cache_attention(q.cuda(), *(x.cuda() for x in cache))
    q[0, 0, 2] = math.nan
    got = stof_b200.cache_attention(q.cuda(), *(x.cuda() for x in cache))
    _status()
    assert bool(torch.isnan(got[0, 0, 2]).all())
    clean[0, 0, 2] = got[0, 0, 2] = 0
    assert torch.equal(got, clean)


def test_cache_attention_reports_bad_pages():
    import stof_b200
    from stof_b200 import _lib
    q = _rand((2, 1, 2, 64), 1)
    k, v, ks, vs, table, lengths = _cache([200, 40], 2, 16, 64, torch.int8, 2)
    table[0, 3] = 1 << 20
    table[0, 5] = -1
    stof_b200.cache_attention(q.cuda(), *(x.cuda() for x in (k, v, ks, vs, table, lengths)))
    torch.cuda.synchronize()
    with pytest.raises(stof_b200.StofError, match="status 2"):
        _lib.check_status(torch.device("cuda"), "test")
    # behind a request's need the table may hold anything, and the table may be wider than it has to be
    wide = torch.full((2, 40), -5, dtype=torch.int32)
    table[0, 3] = table[0, 5] = 0
    wide[0, :13], wide[1, :3] = table[0, :13], table[1, :3]
    _both_cache(q, (k, v, ks, vs, wide, lengths))
    # lengths beyond the table count to its end
    full = stof_b200.cache_attention(q.cuda(), *(x.cuda() for x in (k, v, ks, vs, table[:, :3].contiguous(), torch.tensor([48, 40], dtype=torch.int32))))
    over = stof_b200.cache_attention(q.cuda(), *(x.cuda() for x in (k, v, ks, vs, table[:, :3].contiguous(), torch.tensor([2 ** 31 - 1, 40], dtype=torch.int32))))
    _status()
    assert torch.equal(full, over)


def test_cache_attention_layouts():
    import stof_b200
    cache = [x.cuda() for x in _cache([200, 77], 2, 32, 64, torch.int8, 97)]
    q = _rand((2, 3, 4, 64), 98, 1.0).cuda()
    want = stof_b200.cache_attention(q, *cache)
    fused = torch.zeros(2, 3, 8, 64, dtype=torch.float16, device="cuda")
    fused[:, :, 2:6] = q
    out = torch.zeros(2, 3, 10, 64, dtype=torch.float16, device="cuda")
    got = stof_b200.cache_attention(fused[:, :, 2:6], *cache, out=out[:, :, 3:7])
    assert torch.equal(got, want) and not out[:, :, :3].any() and not out[:, :, 7:].any()
    odd = torch.zeros(2, 3, 4, 65, dtype=torch.float16, device="cuda")
    odd[..., 1:] = q
    assert torch.equal(stof_b200.cache_attention(odd[..., 1:], *cache), want)
    wide = torch.full((2, 9), 1, dtype=torch.int32, device="cuda")
    wide[:, :cache[4].shape[1]] = cache[4]
    assert torch.equal(stof_b200.cache_attention(q, *cache[:4], wide[:, :cache[4].shape[1]], cache[5]), want)
    assert stof_b200.cache_attention(q[:, :0], *cache).shape == (2, 0, 4, 64)
    assert stof_b200.cache_attention(q[:0], *cache[:4], cache[4][:0], cache[5][:0]).shape == (0, 3, 4, 64)
    empty = torch.zeros(2, 0, dtype=torch.int32, device="cuda")
    assert not stof_b200.cache_attention(q, *cache[:4], empty, torch.zeros(2, dtype=torch.int32, device="cuda")).any()
    _status()


# ------------------------------------------------------------------------------------------ writes
def _append_both(cache, k, v, slots):
    import stof_b200
    dev = [x.cuda() for x in cache[:4]]
    stof_b200.cache_append(*dev, k.cuda(), v.cuda(), slots.cuda())
    _status()
    want = [x.clone() for x in cache[:4]]
    os_.cache_append(want[0], want[2], k, slots)
    os_.cache_append(want[1], want[3], v, slots)
    for got, ref in zip(dev, want):
        got = got.cpu()
        if got.dtype == torch.float8_e4m3fn:
            got, ref = got.view(torch.uint8), ref.view(torch.uint8)
        assert torch.equal(got, ref)
    return dev


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("entry", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
def test_cache_append_bit_for_bit(dim, entry, dtype, page):
    """Tokens of a step, prompts over several pages and short runs inside pages, scales that grow and scales that stay."""
    cache = _cache([page * 12], 3, page, dim, entry, 101)
    cache[0].view(torch.uint8)[0, 0, 0, 0] = 1           # (no NaN: what is in front of a run is rounded again)
    table = cache[4][0].tolist()
    slots = [table[0] * page + 5, table[1] * page, table[2] * page + page - 1]
    slots += [table[3] * page + i for i in range(3, page)] + [table[4] * page + i for i in range(page)] + [table[5] * page + i for i in range(7)]
    slots += [-1, -1] + [table[6] * page + i for i in range(1, 6)] + [-3] + [table[7] * page + i for i in range(2, 6)]
    g = torch.Generator().manual_seed(5)
    k, v = (torch.randn(len(slots), 3, dim, generator=g) * (torch.rand(len(slots), 1, 1, generator=g) * 6) for _ in range(2))
    k[1] = 0.0                                           # a scale of 0
    _append_both(cache, k.to(TYPES[dtype]), v.to(TYPES[dtype]), torch.tensor(slots, dtype=torch.int32))


def test_cache_append_many_tokens():
    """More tokens than a launch of small chunks takes."""
    page, tokens = 16, 1500
    cache = _cache([tokens + 10], 2, page, 64, torch.int8, 103)
    at = torch.arange(10, 10 + tokens)
    slots = cache[4][0][at // page] * page + at % page
    k, v = _rand((tokens, 2, 64), 104, 3.0), _rand((tokens, 2, 64), 105, 3.0)
    _append_both(cache, k, v, slots.int())


def test_cache_append_layouts_and_refused_slots():
    import stof_b200
    from stof_b200 import _lib
    cache = _cache([64], 2, 16, 64, torch.int8, 106)
    qkv = _rand((5, 3, 2, 64), 107)
    slots = torch.arange(16, 21, dtype=torch.int32)
    dev = _append_both(cache, qkv[:, 1], qkv[:, 2], slots)
    other = [x.cuda() for x in cache[:4]]
    whole = qkv.cuda()
    stof_b200.cache_append(*other, whole[:, 1], whole[:, 2], slots.cuda())
    assert all(torch.equal(a, b) for a, b in zip(dev, other))
    odd = torch.zeros(5, 2, 65, dtype=torch.float16, device="cuda")
    odd[..., 1:] = whole[:, 1]
    other = [x.cuda() for x in cache[:4]]
    stof_b200.cache_append(*other, odd[..., 1:], whole[:, 2], torch.stack((slots, slots), 1).cuda()[:, 0])
    assert all(torch.equal(a, b) for a, b in zip(dev, other))
    stof_b200.cache_append(*other, whole[:0, 1], whole[:0, 2], slots[:0].cuda())
    _status()
    before = [x.clone() for x in other]
    stof_b200.cache_append(*other, whole[:, 1], whole[:, 2], torch.full((5,), cache[0].shape[0] * 16, dtype=torch.int32, device="cuda"))
    torch.cuda.synchronize()
    with pytest.raises(stof_b200.StofError, match="status 2"):
        _lib.check_status(torch.device("cuda"), "test")
    assert all(torch.equal(a, b) for a, b in zip(before, other))


# ------------------------------------------------------------------------------------------ tables
def _tables_both(lengths, held, table, stack, count, size, new_tokens):
    import stof_b200
    t, s = torch.tensor(table, dtype=torch.int32).view(len(lengths), -1 if table else 4).cuda(), torch.tensor(stack, dtype=torch.int32).cuda()
    i32 = lambda x: torch.tensor(x, dtype=torch.int32).cuda()
    slots, starts, left, missing = stof_b200.page_tables(i32(lengths), i32(held), t, s, i32([count]), size, new_tokens)
    _status()
    want = os_.page_tables(lengths, held, table, stack, count, size, new_tokens)
    assert t.tolist() == want[0] and s.tolist() == want[1]
    assert slots.tolist() == want[2] and starts.tolist() == want[3] and left.item() == want[4] and missing.item() == want[5]
    return want


def _pool(held, width, size, spare, seed):
    import random
    r = random.Random(seed)
    pages = list(range(sum(-(-h // size) for h in held) + spare))
    r.shuffle(pages)
    table = [[pages.pop() for _ in range(-(-h // size))] + [-1] * (width - -(-h // size)) for h in held]
    used = sum(-(-h // size) for h in held)
    return table, pages + [-9] * used, len(pages)


@pytest.mark.parametrize("requests", [1, 2, 31, 33, 400, 1025, 2100])
@pytest.mark.parametrize("size", [16, 128])
def test_page_tables(requests, size):
    import random
    r = random.Random(requests)
    longest = 40 * size
    held = [r.choice([0, 1, size, size + 1, r.randint(0, longest)]) for _ in range(requests)]
    lengths = [r.choice([0, h, h + 1, h + size, r.randint(0, longest)]) for h in held]
    lengths = [min(x, longest) for x in lengths]
    table, stack, count = _pool(held, 40, size, sum(-(-x // size) for x in lengths), 1)
    fresh = sum(max(0, b - a) for a, b in zip(held, lengths))
    assert _tables_both(lengths, held, table, stack, count, size, fresh)[5] == 0
    _tables_both(lengths, held, table, stack, count, size, fresh + 77)
    _tables_both(lengths, held, table, stack, count, size, fresh // 2)


def test_page_tables_take_back_what_was_given():
    """The stack is empty: the pages taken are those that another request gives back in the same call."""
    table, stack, count = _pool([160, 0], 10, 16, 0, 2)
    assert _tables_both([0, 160], [160, 0], table, stack, count, 16, 160)[5] == 0
    assert _tables_both([32, 128], [160, 0], table, stack, count, 16, 128)[5] == 0


@pytest.mark.parametrize("requests", [2, 500])
def test_page_tables_all_or_nothing(requests):
    held, lengths = [20] * requests, [40] * requests
    table, stack, count = _pool(held, 4, 16, requests - 1, 3)
    assert _tables_both(lengths, held, table, stack, count, 16, 20 * requests)[5] == 1
    table, stack, count = _pool(held, 4, 16, 4 * requests, 3)
    assert _tables_both([16 * 5] * requests, held, table, stack, count, 16, 60 * requests)[5] == requests
    # given back twice: the stack has no room
    assert _tables_both([0] * requests, held, table, stack[:count], count, 16, 0)[5] < 0
    # lengths that are none
    _tables_both([-5] * requests, [-1] * requests, table, stack, count, 16, 4)
    _tables_both([2 ** 31 - 1] * requests, held, table, stack, count, 16, 4)


def test_page_tables_of_nobody():
    assert _tables_both([], [], [], [3, 4], 2, 16, 3)[2] == [-1, -1, -1]


# ------------------------------------------------------------------------------------------ refusals of the Python entry points
def _scored_args():
    x = _rand((2, 4, 32, 64), 1).cuda()
    return dict(q=x, k=x[:, :2].contiguous(), v=x[:, :2].contiguous())


@pytest.mark.parametrize("change,text", [
    (lambda a: a.update(q=a["q"].float()), "float16 or bfloat16"), (lambda a: a.update(k=a["k"].bfloat16()), "one type"), (lambda a: a.update(v=a["v"][:, :1]), "one shape"),
    (lambda a: a.update(q=a["q"][0]), "must be"), (lambda a: a.update(q=a["q"][..., :32], k=a["k"][..., :32], v=a["v"][..., :32]), "head size"),
    (lambda a: a.update(q=a["q"][:, :3]), "multiple"), (lambda a: a.update(q=a["q"][:1]), "batch"), (lambda a: a.update(softcap=0.0), "softcap"),
    (lambda a: a.update(softcap=float("nan")), "softcap"), (lambda a: a.update(window=0), "window"), (lambda a: a.update(window=-3), "window"),
    (lambda a: a.update(softmax_scale=-1.0), "softmax_scale"), (lambda a: a.update(slopes=torch.ones(3).cuda()), "slopes"),
    (lambda a: a.update(slopes=torch.ones(4).half().cuda()), "slopes"), (lambda a: a.update(distance_bias=torch.ones(4, 4).cuda()), "distance_bias"),
    (lambda a: a.update(distance_bias=torch.ones(4, 4099).cuda()), "2048"), (lambda a: a.update(documents=torch.zeros(2, 31, dtype=torch.int32).cuda()), "documents"),
    (lambda a: a.update(documents=torch.zeros(2, 32, dtype=torch.int64).cuda()), "documents"), (lambda a: a.update(key_lens=torch.ones(2).cuda()), "key_lens"),
    (lambda a: a.update(key_lens=torch.ones(3, dtype=torch.int32).cuda()), "key_lens"), (lambda a: a.update(prefix_lens=torch.ones(2, dtype=torch.int32).cuda()), "causal"),
    (lambda a: a.update(out=a["q"]), "overlap"), (lambda a: a.update(out=torch.empty(2, 4, 32, 64).cuda()), "out must"), (lambda a: a.update(slopes=torch.ones(4)), "CUDA"),
    (lambda a: a.update(out=torch.empty(2, 4, 32, 65, dtype=torch.float16).cuda()[..., 1:]), "multiples of 16")])
def test_scored_refusals(change, text):
    import stof_b200
    a = _scored_args()
    change(a)
    with pytest.raises(stof_b200.StofError, match=text):
        stof_b200.scored_attention(a.pop("q"), a.pop("k"), a.pop("v"), **a)


@pytest.mark.parametrize("change,text", [
    (lambda a: a.update(q=a["q"][0]), "must be"), (lambda a: a.update(q=a["q"].float()), "float16 or bfloat16"), (lambda a: a.update(k_pages=a["k_pages"].half()), "int8 or float8"),
    (lambda a: a.update(v_pages=a["v_pages"][:4]), "one type and shape"), (lambda a: a.update(k_scales=a["k_scales"].half()), "scales"),
    (lambda a: a.update(k_pages=a["k_pages"].transpose(0, 1), v_pages=a["v_pages"].transpose(0, 1)), "contiguous"), (lambda a: a.update(lengths=a["lengths"].long()), "lengths"),
    (lambda a: a.update(block_table=a["block_table"].long()), "block_table"), (lambda a: a.update(block_table=a["block_table"][:1]), "block_table"),
    (lambda a: a.update(block_table=a["block_table"].t().contiguous().t()), "block_table"), (lambda a: a.update(q=a["q"][:, :, :3]), "multiple"),
    (lambda a: a.update(window=0), "window"), (lambda a: a.update(out=a["q"]), "overlap"),
    (lambda a: a.update(k_pages=a["k_pages"][:, :, :8].contiguous(), v_pages=a["v_pages"][:, :, :8].contiguous()), "page size")])
def test_cache_attention_refusals(change, text):
    import stof_b200
    k, v, ks, vs, table, lengths = (x.cuda() for x in _cache([40, 20], 2, 16, 64, torch.int8, 1))
    a = dict(q=_rand((2, 1, 4, 64), 1).cuda(), k_pages=k, v_pages=v, k_scales=ks, v_scales=vs, block_table=table, lengths=lengths)
    change(a)
    with pytest.raises(stof_b200.StofError, match=text):
        stof_b200.cache_attention(**a)


@pytest.mark.parametrize("change,text", [
    (lambda a: a.update(k=a["k"].float()), "float16 or bfloat16"), (lambda a: a.update(v=a["v"][:1]), "one type and shape"),
    (lambda a: a.update(k=a["k"][:, :1], v=a["v"][:, :1]), "as the cache is"), (lambda a: a.update(slots=a["slots"].long()), "slots"),
    (lambda a: a.update(slots=a["slots"][:1]), "slots"), (lambda a: a.update(slots=a["slots"].cpu()), "CUDA")])
def test_cache_append_refusals(change, text):
    import stof_b200
    k, v, ks, vs, *_ = (x.cuda() for x in _cache([40, 20], 2, 16, 64, torch.int8, 1))
    new = _rand((3, 2, 64), 1).cuda()
    a = dict(k_pages=k, v_pages=v, k_scales=ks, v_scales=vs, k=new, v=new, slots=torch.arange(3, dtype=torch.int32).cuda())
    change(a)
    with pytest.raises(stof_b200.StofError, match=text):
        stof_b200.cache_append(**a)


@pytest.mark.parametrize("change,text", [
    (lambda a: a.update(lengths=a["lengths"].long()), "lengths"), (lambda a: a.update(held=a["held"][:1]), "held"), (lambda a: a.update(new_tokens=-1), "new_tokens"),
    (lambda a: a.update(page_size=20), "page size"), (lambda a: a.update(free_count=a["held"]), "free_count"), (lambda a: a.update(free_pages=a["free_pages"][::2]), "free_pages"),
    (lambda a: a.update(block_table=a["block_table"].float()), "block_table")])
def test_page_tables_operator_refusals(change, text):
    import stof_b200
    i = lambda *x: torch.tensor(x, dtype=torch.int32).cuda()
    a = dict(lengths=i(3, 4), held=i(1, 1), block_table=i(0, 1).view(2, 1), free_pages=i(5, 6, 7, 8), free_count=i(4), page_size=16, new_tokens=5)
    change(a)
    with pytest.raises(stof_b200.StofError, match=text):
        stof_b200.page_tables(**a)
