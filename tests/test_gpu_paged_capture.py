"""Whole steps over a cache in pages, captured and replayed, beside the same steps run eagerly on a cache of their own: a
beam search's, a drafted tree's, and the packing of the pool between them. Every list, page and result has the same bits
after each replay."""
import numpy as np
import pytest
import torch

from inference_amd import PagedKVCache, beam_select, reorder_rows
from inference_amd.paged import tree_masks

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
LAYERS, KV, HEADS, DIM, PAGE, WIDE, PAGES = 2, 2, 8, 64, 16, 8, 48
VOCAB = HEADS * DIM
SEARCHES, BEAMS = 2, 3
ROWS = SEARCHES * BEAMS
TREE = [-1, -1, 0, 0, 2, 3, 3, 5, 1]
PATH = [0, 3, 5, 7]


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


class Run:
    """A cache and all that a step keeps, with rows made of the tokens by tables in place of a model."""

    def __init__(self, dtype):
        g = torch.Generator(device=DEV).manual_seed(3)
        self.q, self.k, self.v = (torch.randn((VOCAB, h, DIM), device=DEV, generator=g) for h in (HEADS, KV, KV))
        a = torch.arange(WIDE * PAGE, device=DEV)[:, None] * 100.0 ** (-torch.arange(DIM, device=DEV) % (DIM // 2) / DIM)
        self.cos, self.sin = a.cos().contiguous(), a.sin().contiguous()
        self.c = PagedKVCache.empty(LAYERS, PAGES, KV, PAGE, DIM, ROWS, WIDE, dtype, DEV)
        self.parents, self.tokens, self.one = ints(list(range(ROWS))), ints([5, 9, 9, 5, 9, 9]), ints([1] * ROWS)
        self.starts, self.drafts = ints(list(range(ROWS + 1))), ints([i * len(TREE) for i in range(ROWS + 1)])
        self.scores = torch.zeros(ROWS, device=DEV)
        self.finished, self.short = ints([0] * ROWS), ints([0])
        self.text = torch.zeros((ROWS, 64), dtype=torch.int32, device=DEV)
        self.moved, self.used = torch.zeros_like(self.text), ints([0])
        masks, depths = tree_masks([TREE] * ROWS)
        self.masks, self.depths = masks.to(DEV), depths.to(DEV)
        self.path, self.counts = ints([PATH] * ROWS), ints([4, 1, 0, 3, 2, 4])
        self.out = torch.zeros((ROWS * len(TREE), HEADS, DIM), device=DEV)

    def layers(self, tokens, starts, masks=None, depths=None, most=1):
        t = tokens.long()
        x = 0.0
        for layer in range(LAYERS):
            q = self.c.append(layer, self.k[t] + layer, self.v[t] - layer, starts, q=self.q[t] + x, cos=self.cos,
                              sin=self.sin, depths=depths)
            x = self.c.attention(layer, q, starts, masks=masks, max_rows=most)
        return x

    def beam(self):
        self.c.fork(self.parents, reserve=1, shortage=self.short)
        logits = self.layers(self.tokens, self.starts).view(ROWS, VOCAB) * 4
        self.c.accept(None, self.one)
        new, parents, scores, over = beam_select(logits, self.scores, BEAMS, BEAMS, finished=self.finished, eos=7)
        reorder_rows(self.text, parents.view(-1), out=self.moved)
        self.text.copy_(self.moved)
        self.text[:, :1] += new.view(-1, 1)
        self.tokens.copy_(new.view(-1)), self.parents.copy_(parents.view(-1))
        self.scores.copy_(scores.view(-1)), self.finished.copy_(over.view(-1))

    def tree(self):
        self.c.fork(self.parents, reserve=len(TREE), shortage=self.short)
        rows = ((self.tokens[:, None] + torch.arange(len(TREE), device=DEV) * 31) % VOCAB).int().view(-1)
        self.out.copy_(self.layers(rows, self.drafts, self.masks, self.depths, len(TREE)))
        self.c.accept(self.path, self.counts)
        self.parents.copy_(torch.arange(ROWS, device=DEV))

    def pack(self):
        self.c.fork(self.parents, shortage=self.short)
        self.parents.copy_(torch.arange(ROWS, device=DEV))
        self.used.copy_(self.c.compact())

    def state(self):
        return [self.c.table, self.c.lens, self.c.refs, self.c.k, self.c.v, self.parents, self.tokens, self.scores,
                self.finished, self.short, self.text, self.moved, self.used, self.out]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_captured_steps(dtype):
    eager, other = Run(dtype), Run(dtype)
    graphs = {}
    for name in ("beam", "tree", "pack"):
        getattr(other, name)()  # (the kernels are loaded before the capture)
    torch.cuda.synchronize()
    other = Run(dtype)
    for name in ("beam", "tree", "pack"):
        graphs[name] = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graphs[name]):
            getattr(other, name)()
    for name in "beam beam beam tree beam pack beam tree pack beam beam tree beam pack".split():
        graphs[name].replay()
        getattr(eager, name)()
        torch.cuda.synchronize()
        for a, b in zip(eager.state(), other.state()):
            assert torch.equal(a, b)
        assert int(eager.short) == 0
        table, refs = eager.c.table.cpu().numpy(), eager.c.refs.cpu().numpy()
        want = np.zeros(PAGES, int)
        np.add.at(want, table[table >= 0], 1)
        np.testing.assert_array_equal(refs, want)
        if name == "pack":
            assert int(eager.used) == int((refs != 0).sum()) and not refs[int(eager.used):].any()
    assert int(eager.c.lens.max()) >= 16
