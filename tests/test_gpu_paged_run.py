"""The paged cache's operators together, as a server runs them over a small Llama: prompts, greedy decoding, a beam
search with its forks and a speculative step with its tree, each row's logits against the same text run alone, token by
token, in a cache of its own.

Tolerances, of the logits' rms. Attention's sums differ in their last bits between the two, and that flips roundings.

Dense weights over an f32 cache: each of 13 products of up to 512 terms is off by 512 * 2^-24 = 3e-5 at most, 4e-4 in
all, and scores of up to 10 make 1e-3 of what feeds them. Over a 16-bit cache a flip is a step of a key or a value, and a
flip early in a text flips others behind it: at the end the two runs round apart. Two roundings differ by
step / sqrt(6), 0.72 * 2^-7 * 0.41 = 2.3e-3 of a bf16 value in the mean; scores of a standard deviation of 0.64 (weights
of 0.05 over 256 units: q and k of 0.8, 64 products of them over 8) make 1.5e-3 of the weights, together 2.7e-3, two
layers and a gain of two behind them 7.8e-3, and the largest of 40000 values is at 4.5 times that: 3.5e-2; fp16 an
eighth, and the f32 bound beside it.

Quantized weights: a step of a Q8_K block is its largest of 256 values / 127. Roundings apart differ by
step / sqrt(6) = 3.2e-3 of that largest value: 1e-2 of the rms where it is 3 times it, 2.6e-2 for the product of gate and
up, whose largest is 8 times it. The squares of what a layer adds: the values 1, the scores 2, the output's product 1, gate
and up with a gain of two 4, down 6.8, in 1e-4: 1.5e-3; two layers and the head 3.1e-3, 5.5e-2 rms, 0.25 at 4.5 times that.
A row that is wrong altogether is off by 1.4 rms and 6 at its largest.
"""
import numpy as np
import pytest
import torch

from inference_amd import PagedKVCache, QMatMul, beam_select, qmm, reorder_rows
from inference_amd.llama_decode import DecodeSession, LlamaConfig, LlamaWeights, rope_tables
from inference_amd.paged import tree_masks
from oracle import paged

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
PAGE, WIDE, PAGES = 16, 8, 60


@pytest.fixture(scope="module", params=["quantized", "dense"])
def model(request):
    cfg = LlamaConfig(layers=2, hidden=256, ffn=512, heads=4, kv_heads=2, head_dim=64, vocab=700)
    w = LlamaWeights.random(cfg, 5, DEV, std=0.05)
    cos, sin = rope_tables(cfg, WIDE * PAGE)
    dense = {}
    if request.param == "dense":
        for t in [t for lw in w.layers for t in lw.values()] + [w.head]:
            dense[id(t)] = t.dequantize()

    def product(t, x):
        return x @ dense[id(t)].t() if dense else QMatMul(t).forward(x)
    return cfg, w, torch.from_numpy(cos).to(DEV), torch.from_numpy(sin).to(DEV), product, bool(dense)


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def norm(x, w, eps):
    out = torch.empty_like(x)
    qmm._check(qmm.lib().qmm_rms_norm(x.data_ptr(), x.shape[0], x.shape[1], x.shape[1], w.data_ptr(), eps,
                                      out.data_ptr(), x.shape[1], qmm._stream(DEV)))
    return out


def forward(model, cache, tokens, starts, masks=None, depths=None):
    """Logits of a step's rows, whose keys and values are appended in every layer."""
    cfg, w, cos, sin, product, _ = model
    x = w.embed[tokens.long()].contiguous()
    n = x.shape[0]
    for li, lw in enumerate(w.layers):
        h = norm(x, w.attn_norm[li], cfg.eps)
        q, k, v = (product(lw[p], h).view(n, -1, cfg.head_dim) for p in "qkv")
        q = cache.append(li, k, v, starts, q=q, cos=cos, sin=sin, depths=depths)
        x = x + product(lw["o"], cache.attention(li, q, starts, masks=masks).view(n, -1))
        h = norm(x, w.ffn_norm[li], cfg.eps)
        g, u = product(lw["gate"], h), product(lw["up"], h)
        x = x + product(lw["down"], torch.nn.functional.silu(g) * u)
    return product(w.head, norm(x, w.final_norm, cfg.eps))


def empty(model, slots, dtype=torch.float32):
    cfg = model[0]
    return PagedKVCache.empty(cfg.layers, PAGES, cfg.kv_heads, PAGE, cfg.head_dim, slots, WIDE, dtype, DEV)


def alone(model, text, dtype=torch.float32):
    """Logits of every position of a text, token by token."""
    c = empty(model, 1, dtype)
    out = []
    for t in text:
        assert int(c.fork(ints([0]), reserve=1)) == 0
        out.append(forward(model, c, ints([t]), ints([0, 1]))[0])
        c.accept(None, ints([1]))
    return torch.stack(out)


@pytest.fixture
def close(model, request):
    dtype = request.node.callspec.params.get("dtype", torch.float32)
    tol = 0.25 if not model[5] else {torch.float32: 1e-3, torch.float16: 5.4e-3, torch.bfloat16: 3.5e-2}[dtype]

    def check(got, want):
        rms = float(want.double().square().mean().sqrt())
        assert float((got - want).abs().max()) <= tol * rms
    return check


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_ragged_prompts_and_greedy_tokens(model, close, dtype):
    cfg = model[0]
    texts = [list(range(3, 40)), [9], [500, 2, 77, 8, 100] * 4]
    c = empty(model, 3, dtype)
    assert int(c.fork(ints([0, 1, 2]), reserve=len(texts[0]))) == 0
    starts = ints(np.cumsum([0] + [len(t) for t in texts]).tolist())
    logits = forward(model, c, ints(sum(texts, [])), starts)
    c.accept(None, ints([len(t) for t in texts]))
    at = 0
    for t in texts:
        close(logits[at:at + len(t)], alone(model, t, dtype))
        at += len(t)
    last = logits[starts[1:].long() - 1]
    for _ in range(6):
        new = last.argmax(-1)
        for t, x in zip(texts, new.tolist()):
            t.append(x)
        assert int(c.fork(ints([0, 1, 2]), reserve=1)) == 0
        last = forward(model, c, new.int(), ints([0, 1, 2, 3]))
        c.accept(None, ints([1, 1, 1]))
    for t, row in zip(texts, last):
        close(row, alone(model, t, dtype)[-1])
    if dtype == torch.float32 and not model[5]:  # (the decode session's steps: the same logits)
        s = DecodeSession(model[1], 64)
        s.reset(texts[1])
        history = torch.zeros((len(texts[1]), cfg.vocab), device=DEV)
        s.tokens[:len(texts[1])] = ints(texts[1])
        s.prompt_len = len(texts[1])
        s.run(len(texts[1]), use_graph=False, history=history)
        close(history, alone(model, texts[1]))


def test_beam_search(model, close):
    cfg = model[0]
    searches, beams, steps = 2, 3, 8
    rows = searches * beams
    c = empty(model, rows)
    prompts = [[5, 6, 7, 8, 9, 10, 11, 12, 13, 14, 15, 16, 17, 18], [400]]
    text = torch.zeros((rows, 64), dtype=torch.int32, device=DEV)
    # the prompts once each, in the first beam's slot
    assert int(c.fork(ints(list(range(rows))), reserve=16)) == 0
    starts, tokens = [0], []
    for s in range(searches):
        tokens += prompts[s]
        starts += [len(tokens)] * beams
        text[s * beams:(s + 1) * beams, :len(prompts[s])] = ints(prompts[s])
    logits = forward(model, c, ints(tokens), ints(starts))
    n = [len(prompts[r // beams]) for r in range(rows)]
    c.accept(None, ints([n[r] if r % beams == 0 else 0 for r in range(rows)]))
    full = torch.zeros((rows, cfg.vocab), device=DEV)
    for s in range(searches):
        full[s * beams] = logits[starts[s * beams + 1] - 1]
    scores = torch.full((rows,), float("-inf"), device=DEV)
    scores[::beams] = 0.0
    finished = torch.zeros(rows, dtype=torch.int32, device=DEV)
    eos = int(full[0].argsort(descending=True)[1])  # (a beam of the first step ends)
    for step in range(steps):
        want = paged.beam(full.cpu().numpy(), scores.cpu().numpy(), beams, beams, finished.cpu().numpy(), eos)
        new, parents, best, over = beam_select(full, scores, beams, beams, finished=finished, eos=eos)
        np.testing.assert_array_equal(new.cpu().numpy(), want[0])
        np.testing.assert_array_equal(parents.cpu().numpy(), want[1])
        parents = parents.view(-1)
        assert int(c.fork(parents, reserve=1)) == 0
        text = reorder_rows(text, parents)
        text[torch.arange(rows), torch.tensor([n[r] + step for r in range(rows)])] = new.view(-1)
        scores, finished = best.view(-1).contiguous(), over.view(-1).contiguous()
        full = forward(model, c, new.view(-1).clamp_min(0), ints(list(range(rows + 1))))
        c.accept(None, ints([1] * rows))
        # every page is counted once for each beam that has it
        table, refs = c.table.cpu().numpy(), c.refs.cpu().numpy()
        count = np.zeros(PAGES, int)
        np.add.at(count, table[table >= 0], 1)
        np.testing.assert_array_equal(refs, count)
        if step in (0, steps - 1):
            for r in range(rows):
                if float(scores[r]) > -np.inf:
                    close(full[r], alone(model, text[r, :n[r] + step + 1].tolist())[-1])
    assert bool(finished.any())


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_speculative_step(model, close, dtype):
    """Two texts with drafted trees: each node's logits are its path's, and after the accepted paths have moved up the
    next token's are the accepted text's. Then the pool is packed, and nothing changes."""
    texts = [[7, 1, 300, 4, 5, 6, 44, 8, 9, 10, 3, 2], [600, 13]]
    trees = [[-1, -1, 0, 0, 1, 2, 2, 5], [-1, 0, 0, 1]]
    drafts = [[20, 21, 22, 23, 24, 25, 26, 27], [30, 31, 32, 33]]
    paths = [[0, 2, 5, 7], [0, 2]]
    c = empty(model, 3, dtype)
    assert int(c.fork(ints([-1, 1, 2]), reserve=20)) == 0  # (slot 0 stays empty)
    forward(model, c, ints(texts[0] + texts[1]), ints([0, 0, 12, 14]))
    c.accept(None, ints([0, 12, 2]))
    masks, depths = tree_masks(trees)
    starts = ints([0, 0, 8, 12])
    logits = forward(model, c, ints(drafts[0] + drafts[1]), starts, masks.to(DEV), depths.to(DEV))
    first = 0
    for text, tree, draft in zip(texts, trees, drafts):
        for j in range(len(tree)):
            path, k = [], j
            while k >= 0:
                path.insert(0, draft[k])
                k = tree[k]
            close(logits[first + j], alone(model, text + path, dtype)[-1])
        first += len(tree)
    path = torch.zeros((3, 4), dtype=torch.int32, device=DEV)
    path[1], path[2, :2] = ints(paths[0]), ints(paths[1])
    c.accept(path, ints([0, 4, 2]))
    assert c.lens.tolist() == [0, 16, 4]
    accepted = [t + [d[i] for i in p] for t, d, p in zip(texts, drafts, paths)]
    for packed in (False, True):
        if packed:
            c.fork(ints([0, 1, 2]), reserve=0)
            assert int(c.compact()) == 2 and int(c.refs[2:].abs().sum()) == 0
        assert int(c.fork(ints([-1, 1, 2]), reserve=1)) == 0
        got = forward(model, c, ints([50, 51]), ints([0, 0, 1, 2]))
        for row, t, x in zip(got, accepted, (50, 51)):
            close(row, alone(model, t + [x], dtype)[-1])
