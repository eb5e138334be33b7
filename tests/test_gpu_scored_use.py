"""The operators of `stof_b200.scored` as programs use them: on other streams, from threads, in graphs, far into memory; and that the
shapes reach the kernels they are meant for."""
import threading

import pytest
import torch

from oracle import scored as os_
from test_gpu_scored import TYPES, _cache, _check, _rand, _rules, _status

pytestmark = pytest.mark.gpu


def _kernels(call):
    from torch.profiler import ProfilerActivity, profile
    call()
    torch.cuda.synchronize()
    with profile(activities=[ProfilerActivity.CUDA]) as record:
        call()
        torch.cuda.synchronize()
    names = [e.name for e in record.events() if "stof::" in e.name]
    if not names:
        pytest.skip("the profiler records no kernels here")
    return names


@pytest.mark.parametrize("batch,heads,q_len,dim,kernel", [(1, 40, 500, 128, "scored_attn_kernel<128, 2,"), (2, 40, 500, 128, "scored_attn_kernel<128, 1,"),
                                                          (1, 4, 500, 128, "scored_attn_kernel<128, 1,"), (8, 40, 500, 64, "scored_attn_kernel<64, 1,")])
def test_shapes_run_on_the_kernels_that_the_tests_take_them_for(batch, heads, q_len, dim, kernel):
    import stof_b200
    if torch.cuda.get_device_properties(0).multi_processor_count != 148:
        pytest.skip("the sizes are those of 148 SMs")
    q, k = torch.zeros(batch, heads, q_len, dim, dtype=torch.float16, device="cuda"), torch.zeros(batch, heads, q_len, dim, dtype=torch.float16, device="cuda")
    assert kernel in _kernels(lambda: stof_b200.scored_attention(q, k, k))[-1]


@pytest.mark.parametrize("name", ["cap", "cap far", "cap middle", "slopes causal", "table", "table wide causal", "window", "window causal", "window prefix", "prefix", "documents",
                                  "documents causal", "documents shuffled", "padded", "padded causal", "padded to nothing", "everything"])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("q_len,k_len", [(500, 500), (400, 777)])
def test_two_stretches_that_share_their_tiles(name, dtype, q_len, k_len):
    """One batch of 40 heads of 128: a block takes 256 rows, whose stretches want different tiles, or (400) the second of them few rows."""
    import stof_b200
    t = TYPES[dtype]
    q, k, v = _rand((1, 40, q_len, 128), 21, 2.0, t), _rand((1, 2, k_len, 128), 22, 1.0, t), _rand((1, 2, k_len, 128), 23, 1.0, t)
    rules = _rules(name, 1, 40, k_len)
    dev = {n: (x.cuda() if isinstance(x, torch.Tensor) else x) for n, x in rules.items()}
    got = stof_b200.scored_attention(q.cuda(), k.cuda(), v.cuda(), **dev)
    _status()
    for h in (0, 20, 39):
        one = {n: (x[h:h + 1] if n in ("slopes", "distance_bias") else x) for n, x in rules.items()}
        _check(got[:, h:h + 1], os_.scored_attention(q[:, h:h + 1], k[:, h // 20:h // 20 + 1], v[:, h // 20:h // 20 + 1], **one), v.double(), t)


def _calls():
    """name -> a call that gives its outputs as a list, and the outputs that it has to give."""
    import stof_b200
    q, k, v = (_rand((2, 4, 333, 64), i).cuda() for i in range(3))
    docs = (torch.arange(666, device="cuda").view(2, 333) // 70).int()
    cache = [x.cuda() for x in _cache([300, 77, 5], 2, 16, 64, torch.int8, 7)]
    one = _rand((3, 2, 4, 64), 8).cuda()
    kv = _rand((40, 2, 64), 9).cuda()
    slots = torch.arange(16, 56, dtype=torch.int32, device="cuda")
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")
    lengths, held, table, stack, count = i32(40, 0, 7), i32(10, 30, 0), i32(0, -1, -1, 1, 2, -1, -1, -1, -1).view(3, 3), i32(5, 6, 7, -1, -1), i32(3)

    def append():
        pages = [x.clone() for x in cache[:4]]
        stof_b200.cache_append(*pages, kv, kv, slots)
        return pages

    def tables():
        t, s = table.clone(), stack.clone()
        return [t, s, *stof_b200.page_tables(lengths, held, t, s, count, 16, 40)]

    return {"scored": lambda: [stof_b200.scored_attention(q, k, v, causal=True, softcap=20.0, documents=docs)],
            "cache": lambda: [stof_b200.cache_attention(one, *cache, window=100)], "append": append, "tables": tables}


@pytest.mark.parametrize("name", ["scored", "cache", "append", "tables"])
def test_another_stream_and_a_graph(name):
    call = _calls()[name]
    want = call()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(2_000_000)                     # the work before it on its stream is not done when the call is made
        got = call()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
    for x in got:
        x.view(torch.uint8).zero_()
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    _status()


def test_two_graphs_at_once_do_not_share_a_workspace():
    """Two captured calls over long requests, replayed on two streams at the same time: each has partial results of its own."""
    import stof_b200
    caches = [[x.cuda() for x in _cache([6000, 3000], 2, 64, 64, torch.int8, 40 + i)] for i in range(2)]
    qs = [_rand((2, 1, 4, 64), 50 + i).cuda() for i in range(2)]
    want = [stof_b200.cache_attention(q, *c) for q, c in zip(qs, caches)]
    graphs, got, streams = [], [], [torch.cuda.Stream() for _ in range(2)]
    for q, c in zip(qs, caches):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            got.append([stof_b200.cache_attention(q, *c) for _ in range(8)])
    torch.cuda.synchronize()
    for _ in range(10):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(w, x) for w, xs in zip(want, got) for x in xs)
    _status()


def test_threads_call_at_once():
    calls = _calls()
    want = {n: f() for n, f in calls.items()}
    torch.cuda.synchronize()
    failed = []

    def work(name):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(30):
                    got = calls[name]()
                torch.cuda.current_stream().synchronize()
                if not all(torch.equal(a, b) for a, b in zip(want[name], got)):
                    failed.append(name)
        except Exception as error:
            failed.append(f"{name}: {error!r}")

    threads = [threading.Thread(target=work, args=(n,)) for n in list(calls) * 2]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed
    _status()


def test_the_same_twice_gives_the_same_bits():
    for name, call in _calls().items():
        a, b = call(), call()
        assert all(torch.equal(x, y) for x, y in zip(a, b)), name
    import stof_b200
    cache = [x.cuda() for x in _cache([9000, 2000, 5], 2, 64, 128, torch.float8_e4m3fn, 7)]
    q = _rand((3, 1, 8, 128), 8).cuda()
    first = stof_b200.cache_attention(q, *cache)
    assert all(torch.equal(first, stof_b200.cache_attention(q, *cache)) for _ in range(5))


def test_a_page_behind_two_gigabytes():
    """Entries whose byte offset passes 2^31 and 2^32."""
    import stof_b200
    pages = 2 ** 32 // (8 * 128 * 128) + 3
    k = torch.empty(pages, 8, 128, 128, dtype=torch.int8, device="cuda")
    ks = torch.zeros(pages, 8, device="cuda")
    x, y = _rand((200, 8, 128), 1).cuda(), _rand((200, 8, 128), 2).cuda()
    where = [pages - 1, pages // 2 + 2]
    slots = torch.cat([p * 128 + torch.arange(n) for p, n in zip(where, (128, 72))]).int().cuda()
    v = torch.empty_like(k)
    vs = torch.zeros_like(ks)
    stof_b200.cache_append(k, v, ks, vs, x, y, slots)
    small = [torch.zeros(2, 8, 128, 128, dtype=torch.int8, device="cuda") for _ in range(2)] + [torch.zeros(2, 8, device="cuda") for _ in range(2)]
    stof_b200.cache_append(*small, x, y, torch.arange(200, dtype=torch.int32, device="cuda"))
    q = _rand((1, 1, 8, 128), 3).cuda()
    length = torch.tensor([200], dtype=torch.int32, device="cuda")
    far = stof_b200.cache_attention(q, k, v, ks, vs, torch.tensor([where], dtype=torch.int32, device="cuda"), length)
    near = stof_b200.cache_attention(q, *small, torch.tensor([[0, 1]], dtype=torch.int32, device="cuda"), length)
    _status()
    assert torch.equal(far, near)


def test_strides_behind_two_gigabytes():
    import stof_b200
    flats = [torch.empty(2 ** 31 + 2 ** 20, dtype=torch.float16, device="cuda") for _ in range(2)]
    q, k, v = (_rand((2, 2, 130, 64), i).cuda() for i in range(3))
    views = []
    for i, x in enumerate((q, k, v, torch.zeros_like(q))):
        view = flats[i // 3][i * 40000:].as_strided((2, 2, 130, 64), (2 ** 31 + 64, 130 * 64, 64, 1))
        view.copy_(x)
        views.append(view)
    want = stof_b200.scored_attention(q, k, v, causal=True)
    stof_b200.scored_attention(*views[:3], causal=True, out=views[3])
    _status()
    assert torch.equal(views[3], want)


def test_operators_as_the_first_cuda_call_of_a_thread():
    calls = _calls()
    for f in calls.values():
        f()
    failed = []

    def first():
        for name, f in calls.items():
            try:
                f()
            except Exception as error:
                failed.append(f"{name}: {error!r}")

    t = threading.Thread(target=first)
    t.start()
    t.join()
    torch.cuda.synchronize()
    assert not failed


def test_rows_behind_the_last_query_stay_as_they_are():
    """The rows leave in boxes of 32: a last box that the sequence does not fill writes nothing behind it."""
    import stof_b200
    for dim in (64, 128):
        out = torch.full((2, 2, 160, dim), 7.0, dtype=torch.float16, device="cuda")
        q = _rand((2, 2, 133, dim), 1).cuda()
        stof_b200.scored_attention(q, q, q, out=out[:, :, :133])
        assert bool((out[:, :, 133:] == 7.0).all())
        assert torch.equal(out[:, :, :133], stof_b200.scored_attention(q, q, q))


def test_a_reported_failure_mutes_the_operators():
    """A non-zero status word keeps them from writing, as it does the others."""
    import stof_b200
    from stof_b200 import _lib
    q = _rand((1, 2, 64, 64), 1).cuda()
    out = torch.full_like(q, 3.0)
    cache = [x.cuda() for x in _cache([40], 2, 16, 64, torch.int8, 1)]
    word = _lib.status_word(torch.device("cuda"))
    word.fill_(1)
    before = [x.clone() for x in cache[:4]]
    stof_b200.scored_attention(q, q, q, out=out)
    stof_b200.cache_append(*cache[:4], q[0, :, :48].transpose(0, 1), q[0, :, :48].transpose(0, 1), torch.arange(48, dtype=torch.int32, device="cuda"))
    one = torch.full((1, 1, 2, 64), 3.0, dtype=torch.float16, device="cuda")
    stof_b200.cache_attention(q[:, :, :1].transpose(1, 2), *cache, out=one)
    torch.cuda.synchronize()
    word.zero_()
    assert bool((out == 3.0).all()) and bool((one == 3.0).all()) and all(torch.equal(a, b) for a, b in zip(before, cache[:4]))


def test_generation_refuses_before_it_changes_the_cache():
    import stof_b200
    from test_gpu_generation import HEADS, HID, _weights
    enc = stof_b200.gpt2_stack([stof_b200.EncoderWeights.from_dict(w, "cuda") for w in _weights(1)], HEADS)
    cache = stof_b200.GenerationCache(1, HEADS, 2, 300000)
    lengths = torch.tensor([5, 0], dtype=torch.int32, device="cuda")
    for x, match in ((torch.zeros(5, HID, dtype=torch.bfloat16, device="cuda"), "float16"), (torch.zeros(131073, HID, dtype=torch.float16, device="cuda"), "131072")):
        with pytest.raises(stof_b200.StofError, match=match):
            enc.prefill(x, cache, lengths)
    with pytest.raises(stof_b200.StofError, match="float16"):
        enc.step(torch.zeros(2, 1, HID, device="cuda"), cache)
    cache.check()
    assert cache.lengths.tolist() == [0, 0]


MASKS = {"causal": dict(causal=True), "window": dict(window=40), "window causal": dict(window=70, causal=True),
         "prefix": dict(causal=True, prefix_lens=torch.tensor([77, 0], dtype=torch.int32)), "padded": dict(key_lens=torch.tensor([100, 301], dtype=torch.int32)),
         "padded to nothing": dict(causal=True, key_lens=torch.tensor([0, 33], dtype=torch.int32))}


@pytest.mark.parametrize("mask", MASKS)
@pytest.mark.parametrize("cap", [1e-38, 1e-3, 1.5, 6.0, 14.0, 50.0, 1e6, 3e38])
@pytest.mark.parametrize("dim,dtype,q_len,k_len", [(64, "fp16", 333, 333), (128, "bf16", 300, 400), (64, "bf16", 400, 301)])
def test_the_cap_alone_under_masks(mask, cap, dim, dtype, q_len, k_len):
    """From scores near zero to far behind the cap in one tensor: the polynomials and the exact form, with scores that the mask takes."""
    from test_gpu_scored import _both
    t = TYPES[dtype]
    q, k, v = _rand((2, 2, q_len, dim), 31, 2.0, t), _rand((2, 1, k_len, dim), 32, 1.0, t), _rand((2, 1, k_len, dim), 33, 1.0, t)
    q[:, 1] *= 0.01
    q[:, :, 64:128] = 0                                  # whole warps of rows that score zero everywhere
    _both(q, k, v, t, softcap=cap, **MASKS[mask])


@pytest.mark.parametrize("junk", [float("nan"), float("inf"), -float("inf"), 6e4])
@pytest.mark.parametrize("dim", [64, 128])
def test_the_cap_alone_over_junk_behind_the_keys(junk, dim):
    from test_gpu_scored import _both
    q, k, v = _rand((2, 2, 260, dim), 34, 2.0), _rand((2, 2, 260, dim), 35), _rand((2, 2, 260, dim), 36)
    clean = [x.clone() for x in (k, v)]
    for x in (k, v):
        x[0, :, 130:] = junk
        x[1, :, 7:] = junk
    lens = torch.tensor([130, 7], dtype=torch.int32)
    for x in clean:
        x[0, :, 130:] = 0
        x[1, :, 7:] = 0
    import stof_b200
    got = stof_b200.scored_attention(q.cuda(), k.cuda(), v.cuda(), softcap=30.0, key_lens=lens.cuda())
    _status()
    _check(got, os_.scored_attention(q, *clean, softcap=30.0, key_lens=lens), clean[1].double(), torch.float16)


@pytest.mark.parametrize("rules", [{}, dict(causal=True), dict(window=30), dict(causal=True, softcap=9.0), dict(causal=True, slopes=torch.tensor([0.5, 0.01])),
                                   dict(window=200, distance_bias=torch.linspace(-1, 1, 2 * 17).view(2, 17)), dict(causal=True, prefix_lens=torch.tensor([50, 1], dtype=torch.int32))])
@pytest.mark.parametrize("dim,dtype", [(64, "bf16"), (128, "fp16")])
def test_more_queries_than_keys(rules, dim, dtype):
    """The first queries sit in front of the first key."""
    from test_gpu_scored import _both
    t = TYPES[dtype]
    _both(_rand((2, 2, 401, dim), 41, 2.0, t), _rand((2, 2, 170, dim), 42, 1.0, t), _rand((2, 2, 170, dim), 43, 1.0, t), t, **rules)


def test_append_refuses_one_page_for_keys_and_values():
    import stof_b200
    k, _, ks, vs = [x.cuda() for x in _cache([40], 2, 16, 64, torch.int8, 1)][:4]
    x, slots = _rand((5, 2, 64), 1).cuda(), torch.arange(5, dtype=torch.int32, device="cuda")
    with pytest.raises(stof_b200.StofError, match="of their own"):
        stof_b200.cache_append(k, k, ks, vs, x, x, slots)
    with pytest.raises(stof_b200.StofError, match="of their own"):
        stof_b200.cache_append(k, k.clone(), ks, ks, x, x, slots)


@pytest.mark.parametrize("cap", [1e-38, 1e-3, 1.5, 14.0, 3e38])
@pytest.mark.parametrize("rules", [{}, dict(window=33), dict(slopes=torch.tensor([0.5, 0.0, 0.1, 2.0])), dict(window=60, slopes=torch.tensor([0.5, 0.0, 0.1, 2.0]))])
def test_cache_caps_windows_and_slopes_together(cap, rules):
    import stof_b200
    cache = _cache([300, 3, 40, 0], 2, 32, 64, torch.int8, 5)
    for tokens in (1, 5):
        q = _rand((4, tokens, 4, 64), 6, 2.0)
        dev = {n: (x.cuda() if isinstance(x, torch.Tensor) else x) for n, x in rules.items()}
        got = stof_b200.cache_attention(q.cuda(), *(x.cuda() for x in cache), softcap=cap, **dev)
        _status()
        want = os_.cache_attention(q, *cache, softcap=cap, **rules)
        v_max = (cache[1].double().abs() * cache[3].double()[:, :, None, None]).max()
        _check(got, want, v_max.view(1), torch.float16)
