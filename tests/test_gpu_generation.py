"""A GPT-2 stack that generates: prompts and single tokens through page tables, the cache's writes and both attentions, against the same
layers in plain arithmetic."""
import pytest
import torch
import torch.nn.functional as F

from oracle import scored as os_

pytestmark = pytest.mark.gpu
HID, HEADS, FFN = 256, 4, 512


def _rand(shape, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).half()


def _weights(layers):
    shapes = {"Wqkv": (HID, 3 * HID), "bqkv": (3 * HID,), "Wo": (HID, HID), "bo": (HID,), "g1": (HID,), "b1": (HID,), "W1": (HID, FFN), "bi1": (FFN,), "W2": (FFN, HID),
              "bi2": (HID,), "g2": (HID,), "b2": (HID,)}
    return [{k: (_rand(s, 100 * i + j, s[0] ** -0.5 if len(s) == 2 else 0.1) + (1 if k[0] == "g" else 0)) for j, (k, s) in enumerate(shapes.items())} for i in range(layers)]


class Plain:
    """The requests one by one on the CPU; keys and values rounded as the cache rounds them, the operators' outputs to fp16."""

    def __init__(self, weights, entries, page, eps):
        self.w, self.entries, self.page, self.eps = weights, entries, page, eps
        self.cache = {}

    def request(self, r):
        if r not in self.cache:
            one = lambda: (torch.zeros(40, HEADS, self.page, 64, dtype=torch.int8).view(self.entries), torch.zeros(40, HEADS))
            self.cache[r] = [[one(), one()] for _ in self.w]
        return self.cache[r]

    def run(self, r, x, held, prompt, **rules):
        n = x.shape[0]
        for w, (kc, vc) in zip(self.w, self.request(r)):
            qkv = (x.double() @ w["Wqkv"].double() + w["bqkv"].double()).half()
            q, k, v = qkv.view(n, 3, HEADS, 64).unbind(1)
            slots = torch.arange(held, held + n)
            os_.cache_append(*kc, k, slots)
            os_.cache_append(*vc, v, slots)
            if prompt:
                o = os_.scored_attention(*(t.transpose(0, 1)[None] for t in (q, k, v)), causal=True, **rules)[0].transpose(0, 1)
            else:
                table = torch.arange(40, dtype=torch.int32)[None]
                o = os_.cache_attention(q[None], kc[0], vc[0], kc[1], vc[1], table, torch.tensor([held + n]), **rules)[0]
            ln = lambda y, g, b: F.layer_norm(y, (HID,), w[g].double(), w[b].double(), self.eps).half()
            x = ln(o.reshape(n, HID).half().double() @ w["Wo"].double() + w["bo"].double() + x.double(), "g1", "b1")
            inner = F.gelu(x.double() @ w["W1"].double() + w["bi1"].double(), approximate="tanh").half()
            x = ln(inner.double() @ w["W2"].double() + w["bi2"].double() + x.double(), "g2", "b2")
        return x


# Each layer rounds to fp16 at six places (qkv, attention, the two LayerNorms, the inner activation, P); a difference of one fp16 step
# in k or v may move an entry by one of its own steps (int8: amax / 127, half of what rounding to entries costs anyway; e4m3: 2^-3 of
# the entry).  Unit-variance states: 6 roundings of 2^-11 of values up to 4 a layer, gains of about one, two layers: 0.024; entries
# that flip are few, each weighted by its share of a softmax.
TOLERANCE = 0.03


@pytest.mark.parametrize("entries,page", [(torch.int8, 16), (torch.float8_e4m3fn, 32)])
@pytest.mark.parametrize("rules", [{}, dict(softcap=20.0, slopes=torch.tensor([0.5, 0.25, 0.125, 0.0625]))])
def test_prompts_and_steps(entries, page, rules):
    import stof_b200
    from stof_b200 import _lib
    weights = _weights(2)
    enc = stof_b200.gpt2_stack([stof_b200.EncoderWeights.from_dict(w, "cuda") for w in weights], HEADS)
    cache = stof_b200.GenerationCache(2, HEADS, 4, 300, page_size=page, entries=entries)
    plain = Plain(weights, entries, page, enc.eps)
    dev = {k: (v.cuda() if isinstance(v, torch.Tensor) else v) for k, v in rules.items()}
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")

    def close(got, want):
        assert float((got.float().cpu() - want.float()).abs().max()) <= TOLERANCE

    # two prompts come in, of the first and the third request
    x = _rand((150, HID), 1)
    got = enc.prefill(x.cuda(), cache, i32(130, 0, 20, 0), **dev)
    close(got[:130], plain.run(0, x[:130], 0, True, **rules))
    close(got[130:], plain.run(2, x[130:], 0, True, **rules))
    held = [130, 0, 20, 0]
    for step in range(3):                                # one token each, then two
        n = 1 if step < 2 else 2
        x = _rand((4, n, HID), 10 + step)
        got = enc.step(x.cuda(), cache, **dev)
        for r in (0, 2):
            close(got[r], plain.run(r, x[r], held[r], False, **rules))
            held[r] += n
    assert cache.lengths.tolist() == held
    # the first is done, the fourth comes in while the third stays
    before = int(cache.free_count.item())
    x = _rand((40, HID), 20)
    got = enc.prefill(x.cuda(), cache, i32(0, 0, held[2], 40), **dev)
    close(got, plain.run(3, x, 0, True, **rules))
    assert int(cache.free_count.item()) == before + -(-held[0] // page) - -(-40 // page)
    x = _rand((4, 1, HID), 30)
    got = enc.step(x.cuda(), cache, **dev)
    close(got[2], plain.run(2, x[2], held[2], False, **rules))
    close(got[3], plain.run(3, x[3], 40, False, **rules))
    cache.check()
    torch.cuda.synchronize()
    _lib.check_status(torch.device("cuda"), "generation")


def test_captured_step_is_replayed():
    """A step recorded into a graph goes on from where the cache is: as many replays as eager steps give the same bits."""
    import stof_b200
    weights = [stof_b200.EncoderWeights.from_dict(w, "cuda") for w in _weights(2)]
    enc = stof_b200.gpt2_stack(weights, HEADS)
    prompt, lengths = _rand((60, HID), 1).cuda(), torch.tensor([40, 20, 0], dtype=torch.int32, device="cuda")
    inputs = [_rand((3, 1, HID), 50 + i).cuda() for i in range(40)]
    outs = []
    for graphed in (False, True):
        cache = stof_b200.GenerationCache(2, HEADS, 3, 200, page_size=16)
        enc.prefill(prompt, cache, lengths)
        x = inputs[0].clone()
        got = []
        if graphed:
            warm = stof_b200.GenerationCache(2, HEADS, 3, 200, page_size=16)
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                enc.step(x, warm)
            torch.cuda.current_stream().wait_stream(side)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                out = enc.step(x, cache)
        for t in inputs:
            x.copy_(t)
            if graphed:
                graph.replay()
            else:
                out = enc.step(x, cache)
            got.append(out[:2].clone())
        outs.append((got, cache.lengths.tolist(), cache.free_count.tolist()))
        cache.check()
    assert outs[0][1:] == outs[1][1:] and outs[0][1] == [80, 60, 0]
    assert all(torch.equal(a, b) for a, b in zip(outs[0][0], outs[1][0]))


def test_missing_pages_change_nothing():
    import stof_b200
    enc = stof_b200.gpt2_stack([stof_b200.EncoderWeights.from_dict(w, "cuda") for w in _weights(1)], HEADS)
    cache = stof_b200.GenerationCache(1, HEADS, 2, 100, pages=3, page_size=16)
    enc.prefill(_rand((30, HID), 1).cuda(), cache, torch.tensor([30, 0], dtype=torch.int32, device="cuda"))
    cache.check()
    pages = cache.k_pages.view(torch.int8).clone()
    enc.prefill(_rand((40, HID), 2).cuda(), cache, torch.tensor([30, 40], dtype=torch.int32, device="cuda"))
    with pytest.raises(stof_b200.StofError, match="2 pages short"):
        cache.check()
    assert cache.lengths.tolist() == [30, 0] and int(cache.free_count.item()) == 1 and torch.equal(cache.k_pages.view(torch.int8), pages)


def test_generation_refusals():
    import stof_b200
    enc = stof_b200.gpt2_stack([stof_b200.EncoderWeights.from_dict(w, "cuda") for w in _weights(1)], HEADS)
    with pytest.raises(stof_b200.StofError, match="entries"):
        stof_b200.GenerationCache(1, HEADS, 2, 100, entries=torch.float16)
    with pytest.raises(stof_b200.StofError, match="page_size"):
        stof_b200.GenerationCache(1, HEADS, 2, 100, page_size=20)
    for cache in (stof_b200.GenerationCache(2, HEADS, 2, 100), stof_b200.GenerationCache(1, 2, 2, 100)):
        with pytest.raises(stof_b200.StofError, match="generation"):
            enc.step(_rand((2, 1, HID), 1).cuda(), cache)
