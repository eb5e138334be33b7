"""`cache_append`, `scored_attention` and the stacks' generation at values and in orders that their other tests leave out."""
import math

import pytest
import torch

from oracle import scored as os_
from test_gpu_scored import _both, _both_cache, _cache, _rand, _status

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("entry", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("side", [0, 1])
@pytest.mark.parametrize("first,count", [(0, 40), (3, 2), (17, 20), (0, 1)])
def test_an_appended_nan_comes_out_of_attention(entry, dtype, side, first, count):
    """Prompts (a block's run) and steps (a warp's): who sees the page gets NaN, the other request and the other heads what they had."""
    import stof_b200
    cache = [x.cuda() for x in _cache([first + count, 50], 2, 16, 64, entry, 1)]
    for b, length in enumerate((first + count, 50)):         # (what lies behind the keys may be anything, here it is not)
        for x in cache[:2]:
            x.view(torch.uint8)[cache[4][b, -(-length // 16) - 1].item(), :, length % 16 or 16:] = 0
    x = [_rand((count, 2, 64), 2 + i, 1.0, dtype).cuda() for i in range(2)]
    at = first + torch.arange(count, device="cuda")
    slots = (cache[4][0][at // 16] * 16 + at % 16).int()
    q = _rand((2, 1, 4, 64), 4).cuda()

    def outputs(bad):
        mine = [t.clone() for t in cache]
        rows = [t.clone() for t in x]
        if bad:
            rows[side][count // 2, 1, 5] = math.nan
        stof_b200.cache_append(*mine[:4], *rows, slots)
        return stof_b200.cache_attention(q, *mine), mine

    (clean, _), (got, mine) = outputs(False), outputs(True)
    _status()
    seen = got[0, 0, 2:]                                     # of head 1
    if side == 0 or entry == torch.int8:
        assert bool(torch.isnan(seen).all())
    else:
        assert bool(torch.isnan(seen[:, 5]).all())
    assert torch.equal(got[1], clean[1]) and torch.equal(got[0, 0, :2], clean[0, 0, :2])
    # a run that begins the pages again leaves nothing of it
    at = torch.arange(first + count, device="cuda")
    rows = _rand((first + count, 2, 64), 9, 1.0, dtype).cuda()
    stof_b200.cache_append(*mine[:4], rows, rows, (cache[4][0][at // 16] * 16 + at % 16).int())
    assert bool(torch.isfinite(stof_b200.cache_attention(q, *mine)).all())


@pytest.mark.parametrize("low", [torch.finfo(torch.float32).min, -3e38, -1e30])
def test_a_table_of_the_lowest_value_masks_as_a_low_score_does(low):
    """Keys under it have no weight beside others, and a row of nothing else is a softmax over them: scores next to it lose all their digits,
    in 64 bits too, so that all keys count alike."""
    q, k, v = _rand((1, 2, 300, 64), 51, 2.0), _rand((1, 2, 300, 64), 52), _rand((1, 2, 300, 64), 53)
    g = torch.Generator().manual_seed(5)
    near = torch.randn(2, 2 * 200 + 1, generator=g)
    near[:, :120] = low                                      # 81 and more behind
    near[1, 300:] = low                                      # 99 and more ahead
    for table in (near, torch.full((2, 41), low)):
        for rules in (dict(), dict(causal=True), dict(softcap=20.0), dict(slopes=torch.tensor([0.25, 0.0]))):
            _both(q, k, v, distance_bias=table, **rules)
    lengths = [300, 1, 500]
    for table in (near, torch.full((2, 41), low)):
        for rules in (dict(), dict(window=130), dict(softcap=20.0), dict(slopes=torch.tensor([0.25, 0.0]))):
            _both_cache(_rand((3, 3, 2, 64), 54, 2.0), _cache(lengths, 1, 32, 64, torch.int8, 55), distance_bias=table, **rules)
    far = torch.full((2, 2 * 20 + 1), low)
    far[:, :15] = 0.5                                        # what is near is masked, what is far is not
    _both(q, k, v, causal=True, distance_bias=far)
    _both_cache(_rand((3, 3, 2, 64), 54, 2.0), _cache(lengths, 1, 32, 64, torch.int8, 55), distance_bias=far)


def _stack():
    import stof_b200
    from test_gpu_generation import HEADS, _weights
    return stof_b200.gpt2_stack([stof_b200.EncoderWeights.from_dict(w, "cuda") for w in _weights(1)], HEADS), stof_b200.GenerationCache(1, HEADS, 3, 100, page_size=16)


def _i32(*x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def test_negative_lengths_are_no_lengths():
    """A request let go with a negative length holds nothing: what comes into its row next is as in a fresh cache."""
    x, y = _rand((30, 256), 1).cuda(), _rand((3, 1, 256), 2).cuda()
    results = []
    for gone in (None, _i32(-1, 0, -7)):
        stack, cache = _stack()
        if gone is not None:
            stack.prefill(_rand((33, 256), 3).cuda(), cache, _i32(20, 0, 13))
            cache.resize(gone, 0)
            assert cache.lengths.tolist() == [0, 0, 0]
        results.append((stack.prefill(x, cache, _i32(12, 18, -3)), stack.step(y, cache)[:2], cache.lengths.tolist()))
        cache.check()
    _status()
    assert torch.equal(results[0][0], results[1][0]) and torch.equal(results[0][1], results[1][1])
    assert results[0][2] == results[1][2] == [13, 19, 0]


@pytest.mark.parametrize("lengths", [(25, 0, 10), (20, 0, 0, ), (20, 31, 0), (-1, 30, 30)])
def test_prompts_that_cannot_be_served_change_nothing(lengths):
    """More tokens for a request that holds some; more tokens than there are."""
    import stof_b200
    stack, cache = _stack()
    stack.prefill(_rand((20, 256), 1).cuda(), cache, _i32(15, 0, 5))
    cache.check()
    before = [x.view(torch.int8).clone() if x.dtype == torch.float8_e4m3fn else x.clone() for x in (cache.k_pages, cache.v_pages, cache.k_scales, cache.v_scales, cache.block_table,
                                                                                                      cache.free_pages, cache.free_count, cache.lengths)]
    stack.prefill(_rand((30, 256), 2).cuda(), cache, _i32(*lengths))
    after = [cache.k_pages.view(torch.int8), cache.v_pages.view(torch.int8), cache.k_scales, cache.v_scales, cache.block_table, cache.free_pages, cache.free_count, cache.lengths]
    assert all(torch.equal(a, b) for a, b in zip(before, after))
    with pytest.raises(stof_b200.StofError, match="1 calls of prefill changed nothing"):
        cache.check()
    cache.check()
    # what follows is served: fewer tokens for one, none for another, a prompt for the third, tokens behind the last prompt
    y = stack.prefill(_rand((30, 256), 2).cuda(), cache, _i32(10, 12, 0))
    cache.check()
    assert cache.lengths.tolist() == [10, 12, 0]
    other, fresh = _stack()
    assert torch.equal(other.prefill(_rand((30, 256), 2).cuda(), fresh, _i32(0, 12, 0))[:12], y[:12])


def test_prompts_refuse_other_numbers_of_lengths():
    import stof_b200
    stack, cache = _stack()
    for bad in (_i32(1, 2), _i32(5), torch.zeros(3, 1, dtype=torch.int32, device="cuda")):
        with pytest.raises(stof_b200.StofError, match="lengths"):
            stack.prefill(_rand((5, 256), 1).cuda(), cache, bad)
    assert cache.lengths.tolist() == [0, 0, 0]


def test_prompts_and_steps_of_nothing():
    """Requests that leave while none come; no new tokens."""
    stack, cache = _stack()
    stack.prefill(_rand((20, 256), 1).cuda(), cache, _i32(15, 0, 5))
    assert stack.prefill(_rand((0, 256), 1).cuda(), cache, _i32(0, 0, 5)).shape == (0, 256)
    assert cache.lengths.tolist() == [0, 0, 5]
    assert stack.step(_rand((3, 0, 256), 1).cuda(), cache).shape == (3, 0, 256)
    cache.check()
    _status()
    assert cache.lengths.tolist() == [0, 0, 5]


SHAPES = {"scored_attn_kernel<128, 2,": (1, 40, 500, 128), "scored_attn_kernel<128, 1,": (2, 40, 500, 128), "scored_attn_kernel<64, 1,": (8, 40, 500, 64)}
RECORD = """
import sys
import torch
from torch.profiler import ProfilerActivity, profile
import stof_b200
for shape in {shapes}:
    q = torch.zeros(shape, dtype=torch.float16, device="cuda")
    stof_b200.scored_attention(q, q, q)
    torch.cuda.synchronize()
    with profile(activities=[ProfilerActivity.CUDA]) as record:
        stof_b200.scored_attention(q, q, q)
        torch.cuda.synchronize()
    print("|".join(e.name for e in record.events() if "stof::" in e.name))
"""


def test_shapes_run_on_their_kernels_in_a_process_of_its_own():
    """(late in a long process the profiler records nothing): the shapes of the tests of two stretches that share their tiles take that kernel, those
    of twice the batch do not."""
    import os
    import subprocess
    import sys

    import stof_b200
    if torch.cuda.get_device_properties(0).multi_processor_count != 148:
        pytest.skip("the sizes are those of 148 SMs")
    path = os.path.dirname(os.path.dirname(os.path.abspath(stof_b200.__file__)))
    run = subprocess.run([sys.executable, "-c", RECORD.format(shapes=list(SHAPES.values()))], env={**os.environ, "PYTHONPATH": path}, capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stderr
    names = run.stdout.strip("\n").split("\n")
    assert len(names) == len(SHAPES) and all(kernel in name for kernel, name in zip(SHAPES, names)), names


@pytest.mark.parametrize("rules", [dict(), dict(causal=True), dict(slopes=torch.tensor([0.25, 0.1, 0.0, 0.02]))])
def test_a_large_cap_beside_one_row_of_huge_scores(rules):
    """The row's neighbours, whose scores are of size one, keep their digits under a cap of a million."""
    q, k, v = (_rand((1, 4, 200, 64), 61 + i, 1.5, torch.bfloat16) for i in range(3))
    q[0, :, 70] *= 1e6
    _both(q, k, v, torch.bfloat16, softcap=1e6, **rules)
    rules = {n: x for n, x in rules.items() if n != "causal"}
    q = _rand((2, 2, 4, 64), 64, 1.5, torch.bfloat16)
    q[:, 1, 2] *= 1e6
    _both_cache(q, _cache([300, 77], 1, 32, 64, torch.int8, 65), softcap=1e6, **rules)


@pytest.mark.parametrize("power", [100, 60, 50, 30, 15, -15, -30, -60, -100])
@pytest.mark.parametrize("cap", [1e-3, 2.0, 20.0, 1e6, 1e12, 1e20, 3e38])
def test_caps_under_scales_far_from_one(power, cap):
    """Queries of 2^power under a softmax_scale that takes it back: the cap's polynomial is of the raw score, whose powers may leave fp32."""
    q, k, v = (_rand((1, 2, 200, 64), 71 + i, 1.5, torch.bfloat16) for i in range(3))
    big = (q.float() * 2.0 ** power).bfloat16()
    for rules in (dict(), dict(causal=True, slopes=torch.tensor([0.25, 0.02]))):
        _both(big, k, v, torch.bfloat16, softcap=cap, softmax_scale=2.0 ** (-power - 3), **rules)
        rules.pop("causal", None)
        _both_cache(big[0].transpose(0, 1)[:4].reshape(2, 2, 2, 64), _cache([300, 77], 1, 32, 64, torch.int8, 65), softcap=cap, softmax_scale=2.0 ** (-power - 3), **rules)


@pytest.mark.parametrize("dim,dtype", [(64, torch.float16), (128, torch.bfloat16)])
def test_documents_over_the_longest_row(dim, dtype):
    """131072 packed tokens, the most that documents may name: rows at the beginning, at tiles' borders and at the end."""
    import stof_b200
    n = 131072
    g = torch.Generator().manual_seed(81)
    docs = torch.randint(1, 9000, (64,), generator=g).cumsum(0)
    docs = torch.searchsorted(docs, torch.arange(n), right=True).int()
    q, k, v = (_rand((1, h, n, dim), 82 + i, 1.5, dtype) for i, h in enumerate((2, 1, 1)))
    slopes = torch.tensor([0.01, 0.0])
    got = stof_b200.scored_attention(q.cuda(), k.cuda(), v.cuda(), causal=True, documents=docs[None].cuda(), slopes=slopes.cuda()).cpu()
    _status()
    border = [int(i) for i in (docs[1:] != docs[:-1]).nonzero()[:40:5, 0]]
    for row in [0, 1, 127, 128, 65535, 65536, 131071, *border, *(i + 1 for i in border)]:
        first = int((docs == docs[row]).nonzero()[0, 0])
        for h in range(2):
            x = os_.changed_scores(q[0, h, row:row + 1], k[0, 0, first:row + 1], torch.tensor([row - first]), scale=dim ** -0.5, slope=slopes[h])
            want = torch.softmax(x, 1) @ v[0, 0, first:row + 1].double()
            u = torch.finfo(dtype).eps / 2
            assert bool(((got[0, h, row].double() - want[0]).abs() <= u * want[0].abs() + (u + 6e-4) * float(v.abs().max()) + 1e-6).all()), (row, h)
