"""paged_attn where the scores of the keys are chosen: growing along the keys, and one key far above the others. Every sequence of
the batch has the same pages, so that there are work items enough for each to take all of its keys in one range."""

import pytest
import torch

from q4llm import ops

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
IDS = ["f32", "f16", "bf16"]
# tokens of a sequence and query heads of a KV head: rows of one wave, of two waves side by side, of all four
FORMS = [(1, 1), (5, 4), (40, 4)]
FORM_IDS = ["1x1", "5x4", "40x4"]


class Line:
    """`batch` sequences of n keys on the same pages. Key j has the score scores[j] with every query (q and k have one dim that is not
    zero, q's is 1), and the values v [n, n_kv, hd]."""

    def __init__(self, dev, dt, scores, v, batch, rows, g):
        n, n_kv, hd = v.shape
        ct = torch.bfloat16 if dt == torch.bfloat16 else torch.float16
        pages = -(-n // 16)
        k = torch.zeros(pages * 16, n_kv, hd)
        k[:n, :, 0] = scores[:, None]
        vv = torch.zeros(pages * 16, n_kv, hd)
        vv[:n] = v
        order = torch.randperm(pages, generator=torch.Generator().manual_seed(n))
        self.k, self.v = (torch.empty(pages, 16, n_kv, hd, dtype=ct, device=dev) for _ in range(2))
        for c, x in ((self.k, k), (self.v, vv)):
            c[order.to(dev)] = x.unflatten(0, (pages, 16)).to(ct).to(dev)
        self.table = order.int().to(dev)[None].repeat(batch, 1)
        self.lens = torch.full((batch,), n, dtype=torch.int32, device=dev)
        self.q = torch.zeros(batch * rows, n_kv * g, hd, dtype=dt, device=dev)
        self.q[..., 0] = 1
        # in 64 bits, of the values as the cache holds them: [rows, n_kv, hd]
        s, w = k[:n, 0, 0].to(ct).double(), v.to(ct).double()
        seen = torch.arange(n)[None] <= torch.arange(n - rows, n)[:, None]
        p = torch.softmax(torch.where(seen, s, float("-inf")), -1)
        self.ref = torch.einsum("rn,nhd->rhd", p, w)
        self.size = torch.einsum("rn,nhd->rhd", p, w.abs())
        self.top = w.abs().amax(0)
        self.most = s.abs().max().item()
        self.shape, self.dt, self.n = (batch, rows, n_kv, g, hd), dt, n

    def check(self, err):
        """err: of the result, relative to sum p |v|, and absolute."""
        got = ops.paged_attn(self.q, self.k, self.v, self.table, self.lens, 1.0)
        got = got.unflatten(1, self.shape[2:]).unflatten(0, self.shape[:2]).cpu().double()
        ref, size = (x[None, :, :, None] for x in (self.ref, self.size))
        half = torch.finfo(self.dt).eps / 2
        tol = err[0] * size + err[1] * self.top[None, None, :, None]
        tol = tol + half * (ref.abs() + tol) + torch.finfo(self.dt).smallest_normal * torch.finfo(self.dt).eps
        worst = ((got - ref).abs() / tol).max().item()
        assert worst <= 1, worst  # a NaN fails as well


def weight_step(dt):
    """The rounding of a softmax weight relative to itself."""
    return 2.0 ** -22 if dt == torch.float32 else torch.finfo(dt).eps / 2


@pytest.mark.parametrize("dt", DTYPES, ids=IDS)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("rows,g", FORMS, ids=FORM_IDS)
def test_scores_that_grow_along_the_keys(dev, dt, hd, rows, g):
    """Every block of keys has a new maximum, by more than the 2^8 up to which the sums are not rescaled."""
    n, n_kv = 2048, 16
    gen = torch.Generator().manual_seed(hd + rows)
    line = Line(dev, dt, torch.arange(n) * (400.0 / n), torch.randn(n, n_kv, hd, generator=gen), 32, rows, g)
    # scores: the exponent's factor and product are rounded, twice 2^-24 of the largest score each for a weight and the sum; a weight
    # and the sum of weights are rounded, exp2 and the sums over n keys in fp32
    line.check((2 * line.most * 2.0 ** -22 + 2 * weight_step(dt) + (n + 40) * U, 0.0))


@pytest.mark.parametrize("dt", DTYPES, ids=IDS)
@pytest.mark.parametrize("rows,g", FORMS, ids=FORM_IDS)
@pytest.mark.parametrize("above", [14.0, 16.0, 17.375, 18.0, 22.0])
def test_one_key_far_above_the_others(dev, dt, rows, g, above):
    """The first key draws most of the attention and has the value 0 in even dims: what is left there is the share of 16384 others,
    each far below a weight of 1."""
    n, n_kv, hd = 16385, 8, 64
    gen = torch.Generator().manual_seed(rows)
    v = torch.randn(n, n_kv, hd, generator=gen)
    v[..., ::2] = 1 + 0.125 * torch.rand(n, n_kv, hd // 2, generator=gen)
    v[0, :, ::2] = 0
    scores = 0.05 * torch.rand(n, generator=gen)
    scores[0] = above
    line = Line(dev, dt, scores, v, 64, rows, g)
    # as above; and with an fp16 cache a weight is off by 2^-25, half of fp16's smallest step, where the largest one is 2^12 or more
    line.check((2 * line.most * 2.0 ** -22 + 2 * weight_step(dt) + (n + 40) * U, 0.0 if dt == torch.bfloat16 else n * 2.0 ** -37))


@pytest.mark.parametrize("dt", DTYPES, ids=IDS)
@pytest.mark.parametrize("rows,g", FORMS, ids=FORM_IDS)
def test_scores_near_the_limit_of_fp16_caches(dev, dt, rows, g):
    """Scores up to 9 million, where those of two keys are equal or thousands apart: the values of the highest ones."""
    n, n_kv, hd = 700, 16, 64
    gen = torch.Generator().manual_seed(7 * rows)
    ct = torch.bfloat16 if dt == torch.bfloat16 else torch.float16
    scores = ((torch.rand(n, generator=gen) * 2 - 1) * 60000).to(ct).float()
    line = Line(dev, dt, scores, torch.randn(n, n_kv, hd, generator=gen), 32, rows, g)
    line.q *= 150
    s, w = scores.double(), line.v.cpu()  # (of the pages: the reference is built from the same values as Line's)
    assert w.isfinite().all() and s.abs().max() * 150 < 1e7
    seen = torch.arange(n)[None] <= torch.arange(n - rows, n)[:, None]
    top = torch.where(seen, s, float("-inf"))
    top = (top == top.amax(-1, keepdim=True)).double()
    p = top / top.sum(-1, keepdim=True)
    order = torch.randperm(-(-n // 16), generator=torch.Generator().manual_seed(n))
    v = w[order].flatten(0, 1)[:n].double()
    line.ref, line.size = (torch.einsum("rn,nhd->rhd", p, x) for x in (v, v.abs()))
    # equal scores have equal weights, and all others none: the sums of at most n equal weights, and the quotient
    line.check((2 * weight_step(dt) + (n + 40) * U, 0.0))
