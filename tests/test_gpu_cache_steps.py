"""`cache_attention` where a warp takes several steps: caches of so many keys that the pieces that thread blocks take are of two units of 128
keys and more.  Against the definition in 64 bits (on the GPU, whole requests at a time), with bounds from the keys that carry weight."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
MOST = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}


def _status():
    from stof_b200 import _lib
    torch.cuda.synchronize()
    _lib.check_status(torch.device("cuda"), "test")


def _steps(lengths, kv_heads, rows, dim):
    """Units of a piece, as the kernel deals them: the fewest steps that a warp of a full piece takes (row tiles of 8: one up to 8 rows)."""
    resident = torch.cuda.get_device_properties(0).multi_processor_count * (2 if rows > 8 else 4 if dim == 64 else 3)
    pairs = kv_heads * -(-rows // (16 if rows > 8 else 8))
    total, some = pairs * sum(-(-n // 128) for n in lengths), pairs * sum(n > 0 for n in lengths)
    target = max(resident - some // 2 if some < resident else resident, min(total // 16, 4 * resident))
    return max(-(-total // target), 1)


def _cache(lengths, kv_heads, page, dim, entry, seed):
    """Pages in random order with random entries and scales that make values of unit size."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    blocks = [-(-n // page) for n in lengths]
    pages = sum(blocks) + 3
    order = torch.randperm(pages, generator=g, device="cuda").int()
    table, at = torch.zeros(len(lengths), max(blocks), dtype=torch.int32, device="cuda"), 0
    for b, n in enumerate(blocks):
        table[b, :n] = order[at:at + n]
        at += n

    def entries():
        x = (torch.randn(pages, kv_heads, page, dim, generator=g, device="cuda") * (MOST[entry] / 4)).clamp(-MOST[entry], MOST[entry])
        return (x.round() if entry == torch.int8 else x).to(entry)

    scales = [(torch.rand(pages, kv_heads, generator=g, device="cuda") + 0.5) * 4 / MOST[entry] for _ in range(2)]
    return entries(), entries(), *scales, table, torch.tensor(lengths, dtype=torch.int32, device="cuda")


def _q(requests, tokens, heads, dim, dtype, seed, scale=2.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(requests, tokens, heads, dim, generator=g, device="cuda") * scale).to(dtype)


def _request(pages, scales, row, length):
    """(Hkv, length, D) float64 of one request, and every key's scale (Hkv, length)."""
    at = row[:-(-length // pages.shape[2])].long()
    x = pages.view(torch.int8)[at].view(pages.dtype).float().double().transpose(0, 1).flatten(1, 2)[:, :length]
    s = scales[at].double().t().repeat_interleave(pages.shape[2], 1)[:, :length]
    return x * s[..., None], s


def _check(q, cache, **rules):
    """What rounding allows.  With u = 2^-11 or 2^-8 of the output's type: the output is rounded once, u |o|.  Every p is rounded to fp16
    for the product, together with V's scale: 2^-11 of sum(p |v|), and 2^-25 each where it is that small beside a largest p |scale| of
    a half at least, so n 2^-24 max(p |scale|) max|entry|.  Sums in fp32: 2^-14 of sum(p |v|) is more than chains of a hundred make
    of it.  A score is off by 2^-20 of the sum of its parts' magnitudes (products of 128 terms added in fp32, a few factors), a capped
    one by 3e-6 of itself and 3e-7 of the cap; its p by as much relative, and so the sums that it is in.  A p of 2^-126 of its row's largest
    and below is no normal fp32 number and counts as 0 (to 2^-125: the reference that it is held to may be a rounding off)."""
    import stof_b200
    kp, vp, ks, vs, table, lengths = cache
    got = stof_b200.cache_attention(q, *cache, **rules)
    _status()
    B, T, H, D = q.shape
    N = kp.shape[1]
    group, window, cap, slopes, bias = H // N, rules.get("window"), rules.get("softcap"), rules.get("slopes"), rules.get("distance_bias")
    scale, u = rules.get("softmax_scale", D ** -0.5), torch.finfo(q.dtype).eps / 2
    assert got.shape == q.shape and got.dtype == q.dtype and bool(torch.isfinite(got).all())
    for b, length in enumerate(lengths.tolist()):
        if length == 0:
            assert not got[b].any()
            continue
        k, _ = _request(kp, ks, table[b], length)
        v, v_scale = _request(vp, vs, table[b], length)
        qd = q[b].double().transpose(0, 1).reshape(N, group * T, D)                          # heads of a K/V head, tokens inside
        x, off = scale * (qd @ k.transpose(1, 2)), scale * (qd.abs() @ k.abs().transpose(1, 2)) * 2.0 ** -20
        if cap:
            x = cap * torch.tanh(x / cap)
            off = off + 3e-6 * x.abs() + 3e-7 * cap
        pos = (torch.arange(T, device="cuda") + length - T).repeat(group)
        away = torch.arange(length, device="cuda")[None, :] - pos[:, None]
        add = torch.zeros(H, T, length, dtype=torch.float64, device="cuda")
        if slopes is not None:
            add = add + slopes.double().view(H, 1, 1) * away.view(group, T, length)[0]
        if bias is not None:
            radius = bias.shape[1] // 2
            add = add + bias.double()[:, away.view(group, T, length)[0].clamp(-radius, radius) + radius]
        add = add.view(N, group * T, length)
        x, off = x + add, off + add.abs() * 2.0 ** -20
        on = (away <= 0) & (pos >= 0)[:, None]
        if window is not None:
            on &= away > -window
        x = x.masked_fill(~on, -math.inf)
        none = ~on.any(1)
        x[:, none] = 0.0
        p = torch.softmax(x, 2)
        p[:, none] = 0.0
        off = torch.where(p > 0, off, 0.0)
        want, size = p @ v, p @ v.abs()
        allow = u * want.abs() + (2.0 ** -11 + 2.0 ** -14) * size + (p * off) @ v.abs() + want.abs() * (p * off).sum(2, keepdim=True) \
            + length * 2.0 ** -24 * (p * v_scale.abs()[:, None]).amax(2, keepdim=True) * MOST[vp.dtype] + 2.0 ** -25 \
            + torch.where(p < p.amax(2, keepdim=True) * 2.0 ** -125, p, 0.0) @ v.abs()
        mine = got[b].double().transpose(0, 1).reshape(N, group * T, D)
        over = (mine - want).abs() - allow
        assert float(over.max()) <= 0, f"request {b}: off by {float((mine - want).abs().max()):.3e}, bound exceeded by {float(over.max()):.3e}"
    return got


LONG = [4000, 1, 4100, 0, 2049, 3333, 5000, 4224]


@pytest.mark.parametrize("dim,heads,kv_heads,tokens,dtype", [(64, 8, 8, 1, torch.float16), (64, 8, 8, 4, torch.bfloat16), (128, 16, 8, 2, torch.bfloat16), (64, 16, 4, 5, torch.float16),
                                                             (128, 32, 8, 6, torch.float16)])
@pytest.mark.parametrize("entry,page", [(torch.int8, 16), (torch.float8_e4m3fn, 64), (torch.int8, 128)])
def test_several_steps(dim, heads, kv_heads, tokens, dtype, entry, page):
    assert _steps(LONG, kv_heads, tokens * heads // kv_heads, dim) >= 2
    _check(_q(len(LONG), tokens, heads, dim, dtype, 1), _cache(LONG, kv_heads, page, dim, entry, 2))


@pytest.mark.parametrize("rules", [dict(softcap=3.0), dict(softcap=30.0), dict(window=1000), dict(window=2500, softcap=40.0), dict(slopes=True), dict(slopes=True, window=3000), dict(bias=128),
                                   dict(bias=2048, softcap=5.0)])
@pytest.mark.parametrize("tokens", [1, 3])
def test_several_steps_under_rules(rules, tokens):
    """(slopes up to one a key: the references of rows move at every step)"""
    lengths = LONG * 3
    assert _steps([min(n, rules.get("window", n)) for n in lengths], 8, tokens, 64) >= 2
    rules, g = dict(rules), torch.Generator(device="cuda").manual_seed(3)
    if rules.pop("slopes", False):
        rules["slopes"] = torch.exp2(-torch.arange(8, device="cuda") * 1.5)
    if "bias" in rules:
        rules["distance_bias"] = torch.randn(8, 2 * rules.pop("bias") + 1, generator=g, device="cuda")
    _check(_q(len(lengths), tokens, 8, 64, torch.float16, 4), _cache(lengths, 8, 32, 64, torch.float8_e4m3fn, 5), **rules)


def test_largest_p_beside_largest_scale_stays_in_fp16():
    """P may be 2^8 before a row's reference moves; V's scale beside it must leave the product inside fp16.  Scores of the last 128 keys are 8
    units of log2 above those in front, their page's scale is 256 times the other's; entries are 0 here and there."""
    lengths = [256] * 16
    assert _steps(lengths, 20, 1, 64) >= 2
    kp, vp, ks, vs, table, n = _cache(lengths, 20, 128, 64, torch.int8, 11)
    ks.zero_()
    vs[table[:, 0].long()] = 1.0 / 64
    vs[table[:, 1].long()] = 256.0 / 64
    bias = torch.zeros(20, 2 * 200 + 1, device="cuda")
    bias[:, 200 - 127:] = 8.0 / 1.4426950408889634 * (1 - 1e-6)
    _check(_q(16, 1, 20, 64, torch.bfloat16, 12), (kp, vp, ks, vs, table, n), distance_bias=bias)


@pytest.mark.parametrize("ratio", [12, 18, 24, 40, 100])
@pytest.mark.parametrize("tokens", [1, 3])
def test_a_large_scale_without_weight_takes_no_digits(ratio, tokens):
    """The first pages' V scales are 2^ratio times the others', their scores e^-120 of them: what carries weight keeps its digits."""
    lengths = [768] * 16
    assert _steps(lengths, 8, tokens, 64) >= 2
    kp, vp, ks, vs, table, n = _cache(lengths, 8, 16, 64, torch.int8, 13)
    vs[table[:, :9].long()] = 2.0 ** (ratio - 5)
    bias = torch.zeros(8, 2 * 600 + 1, device="cuda")
    bias[:, 0] = -120.0
    _check(_q(16, tokens, 8, 64, torch.bfloat16, 14), (kp, vp, ks, vs, table, n), distance_bias=bias)


@pytest.mark.parametrize("dim,heads,tokens,entry", [(64, 8, 1, torch.int8), (64, 16, 3, torch.float8_e4m3fn), (128, 16, 1, torch.float8_e4m3fn), (128, 32, 5, torch.int8)])
@pytest.mark.parametrize("spread", [4, 20, 60])
def test_scales_of_any_size_in_any_order(dim, heads, tokens, entry, spread):
    """V scales of 2^-spread to 2^spread, rising, falling and mixed, zeros among them, and scores that favour small scales, large ones or none."""
    lengths = [4000, 1, 900, 0, 2049, 3333, 5000, 4224]
    assert _steps(lengths, 8, tokens * heads // 8, dim) >= 2
    kp, vp, ks, vs, table, n = _cache(lengths, 8, 32, dim, entry, 15)
    width = table.shape[1]
    size = torch.linspace(-1, 1, width, device="cuda")
    q = _q(8, tokens, heads, dim, torch.bfloat16, 16)
    for order in (size, -size, torch.rand(width, device="cuda", generator=torch.Generator(device="cuda").manual_seed(17)) * 2 - 1):
        by_page = torch.zeros(vs.shape[0], device="cuda")
        for b, length in enumerate(lengths):
            blocks = -(-length // 32)
            by_page[table[b, :blocks].long()] = order[:blocks]
        scales = torch.exp2(by_page * spread)[:, None].expand_as(vs).contiguous()
        scales[::7] = 0.0
        for slope in (0.0, 0.05):
            _check(q, (kp, vp, ks, scales / 64, table, n), slopes=torch.full((heads,), slope, device="cuda"))


def test_pages_of_scale_zero_in_front():
    """Rows that have seen keys but no values yet."""
    lengths = [768] * 16
    kp, vp, ks, vs, table, n = _cache(lengths, 8, 16, 64, torch.int8, 18)
    for scale in (2.0 ** -100, 2.0 ** -20, 1.0, 2.0 ** 90):
        vs[table[:, :20].long()] = 0.0
        vs[table[:, 20:].long()] = scale
        _check(_q(16, 1, 8, 64, torch.bfloat16, 19), (kp, vp, ks, vs, table, n))
        vs[table.long()] = 0.0
        assert not _check(_q(16, 1, 8, 64, torch.bfloat16, 19), (kp, vp, ks, vs, table, n)).any()


def test_nan_and_infinite_scales_reach_who_sees_them():
    import stof_b200
    lengths = [768] * 16
    kp, vp, ks, vs, table, n = _cache(lengths, 8, 16, 64, torch.int8, 20)
    q = _q(16, 3, 8, 64, torch.float16, 21)
    clean = stof_b200.cache_attention(q, kp, vp, ks, vs, table, n)
    for bad in (math.nan, math.inf):
        for scales in (ks, vs):
            broken = scales.clone()
            broken[table[3, 7].long(), 5] = bad
            args = (kp, vp, broken, vs, table, n) if scales is ks else (kp, vp, ks, broken, table, n)
            got = stof_b200.cache_attention(q, *args)
            _status()
            assert not bool(torch.isfinite(got[3, :, 5]).any())
            got[3, :, 5] = clean[3, :, 5]
            assert torch.equal(got, clean)
    # a page that begins behind the first of three tokens: that token does not see its scale
    kp, vp, ks, vs, table, n = _cache([50] * 8, 2, 16, 64, torch.int8, 22)
    q = _q(8, 3, 2, 64, torch.float16, 23)
    clean = stof_b200.cache_attention(q, kp, vp, ks, vs, table, n)
    vs[table[:, 3].long()] = math.nan
    got = stof_b200.cache_attention(q, kp, vp, ks, vs, table, n)
    _status()
    assert torch.equal(got[:, 0], clean[:, 0]) and not bool(torch.isfinite(got[:, 1:]).any())


@pytest.mark.parametrize("low", [-1e4, -1e9, -1e30, -3e38])
@pytest.mark.parametrize("tokens", [1, 3])
def test_scores_far_below_the_first_ones_lose_nothing(low, tokens):
    """A table that masks far keys by a low value: the reference that the first steps leave must not take the digits of the later scores."""
    lengths = [768] * 16
    assert _steps(lengths, 8, tokens, 64) >= 2
    cache = _cache(lengths, 8, 16, 64, torch.int8, 24)
    bias = torch.randn(8, 2 * 600 + 1, device="cuda")
    for reach in (600, 350, 40):                         # keys at this distance and beyond
        bias[:, :601 - reach] = low
        _check(_q(16, tokens, 8, 64, torch.float16, 25), cache, distance_bias=bias)


def test_first_pages_of_huge_scores():
    """The same by K's scales: scores of the first pages at -1e5 and below, of those behind them near zero."""
    lengths = [768] * 16
    kp, vp, ks, vs, table, n = _cache(lengths, 8, 16, 64, torch.int8, 26)
    q = _q(16, 1, 8, 64, torch.float16, 27).abs() + 0.5
    kp[table[:, :11].long()] = -100
    for big in (1e2, 1e6):
        ks[table[:, :11].long()] = big
        _check(q, (kp, vp, ks, vs, table, n))


@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 30, 4097, 4096, 4095])
@pytest.mark.parametrize("tokens", [1, 5])
def test_windows_longer_than_any_request_at_the_c_entry(window, tokens):
    """Requests of nothing, shorter than the new tokens and long, whatever the window is taken from."""
    import ctypes

    from stof_b200 import _lib
    lengths = [0, 1, 4000, 2, 4096, 300]
    q, cache = _q(6, tokens, 4, 64, torch.float16, 28), _cache(lengths, 2, 32, 64, torch.int8, 29)
    want = _check(q, cache)
    kp, vp, ks, vs, table, n = cache
    assert table.shape[1] * 32 == 4096
    L, out = _lib.lib(), torch.full_like(q, 7.0)
    rules = _lib.ScoreRules(softmax_scale=0.125, window=window)
    st = _lib.strides3(q.stride()[:3])
    size = L.stof_cache_attn_workspace_bytes(6, tokens, 4, 2, 64, 32, 128)
    space = torch.empty(size, dtype=torch.uint8, device="cuda")
    at = lambda t: ctypes.c_void_p(t.data_ptr())
    rc = L.stof_cache_attn(at(q), at(out), _lib.STOF_DTYPE_F16, st, st, at(kp), at(vp), at(ks), at(vs), _lib.STOF_DTYPE_INT8, kp.shape[0], 32, 2, 64, at(table), 128, 128,
                           at(n), 6, tokens, 4, ctypes.byref(rules), at(space), size, at(_lib.status_word(torch.device("cuda"))), ctypes.c_void_p(torch.cuda.current_stream().cuda_stream))
    assert rc == 0, L.stof_last_error()
    _status()
    if window >= 4096:
        assert torch.equal(out, want)
    else:
        assert torch.equal(out, _check(q, cache, window=window))


@pytest.mark.parametrize("tokens", [1, 4])
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("window", [1, 17, 100, 700])
def test_pages_in_front_of_the_window_may_be_anything(tokens, page, window):
    """Given back and marked, or somebody else's by now, with scales and entries of any kind."""
    lengths = [3000, 129, 128, 1000, 5, 2047]
    q = _q(6, tokens, 4, 64, torch.float16, 30)
    kp, vp, ks, vs, table, n = _cache(lengths, 2, page, 64, torch.float8_e4m3fn, 31)
    want = _check(q, (kp, vp, ks, vs, table, n), window=window)
    marked, other = table.clone(), table.clone()
    # a page of NaN under scales of NaN
    spare = [i for i in range(kp.shape[0]) if i not in set(table.flatten().tolist())]
    for x in (kp, vp):
        x.view(torch.uint8)[spare[0]] = 0x7F
    for x in (ks, vs):
        x[spare[0]] = math.nan
    for b, length in enumerate(lengths):
        hidden = max(length - tokens - window + 1, 0) // page
        marked[b, :hidden], other[b, :hidden] = -1, spare[0]
    import stof_b200
    for t in (marked, other):
        got = stof_b200.cache_attention(q, kp, vp, ks, vs, t, n, window=window)
        _status()
        assert torch.equal(got, want)


@pytest.mark.parametrize("low", [100, 120, 122, 124, 126, 140])
@pytest.mark.parametrize("up", [-90, -20])
@pytest.mark.parametrize("ratio", [110, 129, 131, 133, 140])
def test_a_large_scale_under_little_weight(low, up, ratio):
    """Values of 2^up at full weight, then values 2^ratio larger at 2^-low of it: neither factor of the second product may leave fp32 alone."""
    lengths = [256] * 16
    kp, vp, ks, vs, table, n = _cache(lengths, 20, 128, 64, torch.int8, 32)
    ks.zero_()
    vs[table[:, 0].long()] = 2.0 ** up / 64
    vs[table[:, 1].long()] = 2.0 ** (up + ratio) / 64
    bias = torch.zeros(20, 2 * 200 + 1, device="cuda")
    bias[:, 200 - 127:] = -low * math.log(2)
    _check(_q(16, 1, 20, 64, torch.bfloat16, 33), (kp, vp, ks, vs, table, n), distance_bias=bias)


@pytest.mark.parametrize("low", [-1e3, -1e9, -3e38])
@pytest.mark.parametrize("spread", [4, 30])
def test_low_scores_under_scales_of_any_size(low, spread):
    """What the first steps leave at scores that masks make is in no way of what carries weight, large scales among it."""
    lengths = [4000, 1500, 900, 0, 2049, 3333, 5000, 4224]
    assert _steps(lengths, 8, 1, 64) >= 2
    kp, vp, ks, vs, table, n = _cache(lengths, 8, 32, 64, torch.int8, 34)
    g = torch.Generator(device="cuda").manual_seed(35)
    vs = vs * torch.exp2((torch.rand(vs.shape, generator=g, device="cuda") * 2 - 1) * spread)
    bias = torch.randn(8, 2 * 2000 + 1, generator=g, device="cuda")
    for reach in (2000, 1400, 700, 33):                  # keys at this distance and beyond
        bias[:, :2001 - reach] = low
        _check(_q(8, 1, 8, 64, torch.bfloat16, 36), (kp, vp, ks, vs, table, n), distance_bias=bias)
        _check(_q(8, 1, 8, 64, torch.bfloat16, 36), (kp, vp, ks, vs, table, n), distance_bias=bias, slopes=torch.full((8,), 0.04, device="cuda"))


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("tokens,window", [(1, 1), (1, 70), (3, 70), (2, 333)])
def test_values_in_front_of_the_window_take_no_part(dim, tokens, window):
    """A NaN leaves the results when the window leaves it, not when it leaves the page."""
    import stof_b200
    lengths = [600, 129, 75, 40, 350]
    q = _q(5, tokens, 4, dim, torch.float16, 37)
    kp, vp, ks, vs, table, n = _cache(lengths, 2, 64, dim, torch.float8_e4m3fn, 38)
    want = _check(q, (kp, vp, ks, vs, table, n), window=window)
    for b, length in enumerate(lengths):
        for key in range(max(length - tokens - window + 1, 0)):
            page = table[b, key // 64].item()
            for x in (kp, vp):
                x.view(torch.uint8)[page, :, key % 64] = 0x7F
    got = stof_b200.cache_attention(q, kp, vp, ks, vs, table, n, window=window)
    _status()
    assert torch.equal(got, want)


def test_a_captured_call_follows_lengths_and_scales():
    """Captured over requests of five tokens, replayed over thousands: pieces, steps and references are found at every replay."""
    import stof_b200
    kp, vp, ks, vs, table, n = _cache([4000] * 12, 8, 32, 64, torch.int8, 39)
    q = _q(12, 1, 8, 64, torch.bfloat16, 40)
    n.fill_(5)
    stof_b200.cache_attention(q, kp, vp, ks, vs, table, n, window=3000)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = stof_b200.cache_attention(q, kp, vp, ks, vs, table, n, window=3000)
    g = torch.Generator(device="cuda").manual_seed(41)
    for _ in range(3):
        n.copy_(torch.randint(0, 4001, (12,), generator=g, device="cuda").int())
        vs.copy_(torch.exp2(torch.randn(vs.shape, generator=g, device="cuda") * 8) / 64)
        graph.replay()
        assert torch.equal(out, _check(q, (kp, vp, ks, vs, table, n), window=3000))
