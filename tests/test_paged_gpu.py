"""The operators of batched serving over a paged cache, each against a plain 64-bit computation: rope_rotate,
paged_kv_append, paged_attn and spec_verify, and a run of them together.

Error bounds count roundings: u(t) = finfo(t).eps / 2 is a rounding to t, U = 2^-24 one to fp32."""

import math

import pytest
import torch

from q4llm import ops
from q4llm.rope import Rope

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
IDS = ["f32", "f16", "bf16"]


def half_step(dt):
    return torch.finfo(dt).eps / 2


def cache_of(dt):
    return torch.bfloat16 if dt == torch.bfloat16 else torch.float16


def freqs(rot, dev, base=500000.0):
    return (base ** (-torch.arange(0, rot, 2, dtype=torch.float64) / max(rot, 1))).float().to(dev)


def i32(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


# ------------------------------------------------------------------------------------------------ rotation


def rotated(x, pos, rope, inverse=False):
    """(x rotated in 64 bits, the bound of an fp32 computation's error), on the CPU."""
    x, f = x.cpu().double(), rope.inv_freq.cpu().double()
    h = f.numel()
    pos = pos.cpu().double()
    t = pos[:, None, None] * f
    c, s = rope.mscale * torch.cos(t), rope.mscale * torch.sin(t) * (-1 if inverse else 1)
    a, b = (x[..., 0:2 * h:2], x[..., 1:2 * h:2]) if rope.interleaved else (x[..., :h], x[..., h:2 * h])
    p, q = a * c - b * s, b * c + a * s
    # cos and sin: the fraction of a revolution rounded to fp32 (2^-26 of one), the function itself within two roundings,
    # mscale; angle in fp64: position * 2^-52; then two products and a sum
    e = rope.mscale * (a.abs() + b.abs()) * (2 * math.pi * 2.0 ** -26 + 4 * U + 2 * U + 3 * U) + \
        rope.mscale * (a.abs() + b.abs()) * (pos.abs() * 2.0 ** -51)[:, None, None]
    out, err = x.clone(), torch.zeros_like(x)
    if rope.interleaved:
        out[..., 0:2 * h:2], out[..., 1:2 * h:2] = p, q
        err[..., 0:2 * h:2] = err[..., 1:2 * h:2] = e
    else:
        out[..., :h], out[..., h:2 * h] = p, q
        err[..., :h] = err[..., h:2 * h] = e
    return out, err


def check_rounded(got, ref, err, dt):
    """got (of type dt) is ref within err and the rounding to dt (subnormal steps included)."""
    tiny = torch.finfo(dt).smallest_normal * torch.finfo(dt).eps
    tol = err + half_step(dt) * (ref.abs() + err) + tiny
    bad = (got.cpu().double() - ref).abs() - tol
    assert (bad <= 0).all(), bad.max()


@pytest.mark.parametrize("dt", DTYPES, ids=IDS)
@pytest.mark.parametrize("interleaved", [False, True], ids=["half", "inter"])
@pytest.mark.parametrize("t,h,hd,rot", [(1, 1, 2, 2), (1, 32, 128, 128), (7, 5, 64, 32), (33, 3, 80, 80), (5, 4, 80, 38),
                                        (3, 2, 96, 30), (2, 3, 256, 256), (1200, 9, 64, 64), (4, 2, 1024, 1024),
                                        (3, 2, 10, 6), (6, 4, 64, 0), (9, 3, 80, 40), (9, 3, 100, 100)])
def test_rope_rotate(dev, dt, interleaved, t, h, hd, rot):
    g = torch.Generator().manual_seed(t * 7 + hd)
    x = torch.randn(t, h, hd, generator=g).to(dt).to(dev)
    pos = torch.randint(0, 1 << 20, (t,), generator=g).int().to(dev)
    rope = Rope(freqs(rot, dev), interleaved, 1.2)
    ref, err = rotated(x, pos, rope)
    got = ops.rope_rotate(x, pos, rope)
    check_rounded(got, ref, err, dt)
    assert torch.equal(got[..., rot:], x[..., rot:])
    back, err = rotated(x, pos, rope, inverse=True)
    check_rounded(ops.rope_rotate(x, pos, rope, inverse=True), back, err, dt)
    # in place: the same bits
    y = x.clone()
    assert ops.rope_rotate(y, pos, rope, out=y) is y and torch.equal(y, got)


@pytest.mark.parametrize("dt", DTYPES, ids=IDS)
def test_large_calls_go_around_the_caches_with_the_same_bits(dev, dt):
    """Past 32 MB the loads and stores bypass the caches: what they give is what the same tokens give in small calls."""
    t, n_q, n_kv, hd = (20000 if dt == torch.float32 else 40000), 4, 2, 64
    g = torch.Generator().manual_seed(1)
    qkv = torch.randn(t, n_q + 2 * n_kv, hd, generator=g).to(dt).to(dev)
    pos = torch.arange(t, dtype=torch.int32, device=dev)
    rope = Rope(freqs(hd, dev))
    assert qkv.numel() * qkv.element_size() > 32 << 20
    big = ops.rope_rotate(qkv, pos, rope)
    assert all(torch.equal(ops.rope_rotate(qkv[i:i + 5000], pos[i:i + 5000], rope), big[i:i + 5000]) for i in range(0, t, 5000))
    table = torch.randperm(t // 16, generator=g).int().to(dev)[None]
    caches = [torch.zeros(t // 16, 16, n_kv, hd, dtype=cache_of(dt), device=dev) for _ in range(4)]
    q = ops.paged_kv_append(qkv[:, n_q:n_q + n_kv], qkv[:, n_q + n_kv:], *caches[:2], table, i32([t], dev), rope=rope, q=qkv[:, :n_q])
    assert torch.equal(q, big[:, :n_q])
    for i in range(0, t, 5000):
        s = qkv[i:i + 5000]
        ops.paged_kv_append(s[:, n_q:n_q + n_kv], s[:, n_q + n_kv:], *caches[2:], table, i32([i + 5000], dev), rope=rope)
    assert torch.equal(caches[0], caches[2]) and torch.equal(caches[1], caches[3])


def test_rope_far_and_negative_positions(dev):
    pos = i32([0, -1, -12345, (1 << 31) - 1, -(1 << 31), 1 << 24, 16777217], dev)
    x = torch.randn(7, 3, 128, generator=torch.Generator().manual_seed(3)).to(dev)
    rope = Rope(freqs(128, dev))
    ref, err = rotated(x, pos, rope)
    check_rounded(ops.rope_rotate(x, pos, rope), ref, err, torch.float32)
    assert torch.equal(ops.rope_rotate(x, pos, rope)[0], x[0])


@pytest.mark.parametrize("dt", DTYPES, ids=IDS)
@pytest.mark.parametrize("interleaved", [False, True], ids=["half", "inter"])
def test_rope_strides_and_special_values(dev, dt, interleaved):
    """Slices of a wider row, a start off 16 bytes, heads outermost; dims that are not rotated are copied bit for bit."""
    g = torch.Generator().manual_seed(5)
    pos = torch.arange(11, dtype=torch.int32, device=dev) * 97
    rope = Rope(freqs(48, dev), interleaved)
    wide = torch.randn(11, 6 * 64 + 1, generator=g).to(dt).to(dev)
    heads_first = torch.randn(6, 11, 64, generator=g).to(dt).to(dev)
    one = torch.randn(1, 1, 64, generator=g).to(dt).to(dev).expand(11, 6, 64)
    for x in (wide[:, 1:].unflatten(1, (6, 64)), wide[:, :-1].unflatten(1, (6, 64))[:, 2:5], heads_first.transpose(0, 1), one):
        ref, err = rotated(x, pos, rope)
        check_rounded(ops.rope_rotate(x, pos, rope), ref, err, dt)
        out = torch.full((x.shape[1], 11, 80), 7.0, dtype=dt, device=dev)
        view = out[:, :, 16:].transpose(0, 1)
        ops.rope_rotate(x, pos, rope, out=view)
        check_rounded(view, ref, err, dt)
        assert (out[:, :, :16] == 7).all()
    x = heads_first.transpose(0, 1).clone()
    x[..., 48:] = torch.tensor([float("nan"), float("inf"), -0.0, -float("inf")] * 4, dtype=dt)
    y = ops.rope_rotate(x, pos, rope)
    bits = torch.int32 if dt == torch.float32 else torch.int16
    assert torch.equal(y[..., 48:].contiguous().view(bits), x[..., 48:].contiguous().view(bits))
    assert torch.isfinite(y[..., :48]).all()


def test_rope_rotation_is_its_gradient(dev):
    """<w, R x> differentiated by x is R^-1 w (times mscale^2 of an inverse: the rotation is orthogonal up to mscale): against
    differences along random directions, in which R is linear."""
    g = torch.Generator().manual_seed(9)
    x, w, d = (torch.randn(5, 3, 64, generator=g).to(dev) for _ in range(3))
    pos = i32([0, 5, 999, 70000, 3], dev)
    for inter in (False, True):
        rope = Rope(freqs(64, dev), inter, 1.1)
        grad = ops.rope_rotate(w, pos, rope, inverse=True).double()
        f = lambda y: (ops.rope_rotate(y, pos, rope).double() * w.double()).sum()  # noqa: E731
        diff = (f(x + d) - f(x - d)) / 2
        # 960 terms, each off by a few fp32 roundings of values below 16
        assert abs(diff - (grad * d.double()).sum()).item() <= 960 * 16 * 16 * U


# ------------------------------------------------------------------------------------------------ paged batches


class Batch:
    """Sequences of `lens` keys, the last rows[b] of them this step's, on shuffled pages; the first `shared` positions
    on pages that all hold. Unused rows of the pool hold NaN."""

    def __init__(self, dev, dt, hd, n_kv, page, lens, rows, shared=0, ragged=False, seed=0, spare=2, pages=None, extra=0):
        self.g = g = torch.Generator().manual_seed(seed)
        self.dev, self.dt, self.hd, self.n_kv, self.page, self.shared = dev, dt, hd, n_kv, page, shared
        self.lens, self.rows, self.extra = list(lens), list(rows), extra
        n = len(lens)
        ct = cache_of(dt)
        most = max(max(-(-x // page) for x in lens), -(-shared // page), 1) + 1
        sp = -(-shared // page)
        own = [max(0, -(-x // page) - shared // page) for x in lens]
        total = sp + sum(own) + spare
        order = torch.randperm(total, generator=g).tolist()
        self.shared_pages = order[:sp]
        table = [[-7] * most for _ in lens]  # entries that no key is in: not pages
        at = sp
        for b in range(n):
            f = shared // page
            table[b][f:f + own[b]] = order[at:at + own[b]]
            at += own[b]
        self.table = table
        k = torch.full((total, page, n_kv, hd), float("nan"))
        v = torch.full((total, page, n_kv, hd), float("nan"))
        for j in range(shared):
            p = self.shared_pages[j // page]
            k[p, j % page], v[p, j % page] = torch.randn(2, n_kv, hd, generator=g)
        for b in range(n):
            for j in range(shared, lens[b]):
                p = table[b][j // page]
                k[p, j % page], v[p, j % page] = torch.randn(2, n_kv, hd, generator=g)
        self.k, self.v = k.to(ct).to(dev), v.to(ct).to(dev)
        self.tokens = sum(rows) + extra
        self.cu = None
        if ragged:
            self.cu = i32([sum(rows[:i]) for i in range(n + 1)], dev)
        self.page_table, self.seq_lens = i32(table, dev), i32(lens, dev)
        self.sp = i32(self.shared_pages, dev) if shared else None

    def keys(self, b):
        """(k, v) [len, n_kv, hd] of sequence b in 64 bits on the CPU."""
        kk, vv = self.k.cpu().double(), self.v.cpu().double()
        at = [(self.shared_pages[j // self.page] if j < self.shared else self.table[b][j // self.page], j % self.page)
              for j in range(self.lens[b])]
        if not at:
            return kk[:0, 0], vv[:0, 0]
        p, o = torch.tensor(at).t()
        return kk[p, o], vv[p, o]

    def attn(self, q, scale, **kw):
        return ops.paged_attn(q, self.k, self.v, self.page_table, self.seq_lens, scale, cu_q=self.cu, shared_pages=self.sp,
                              shared_len=self.shared, **kw)

    def reference(self, q, scale, L=None):
        """(o, error bound) [tokens, n_q, hd] in 64 bits; rows of no sequence: NaN."""
        q = q.cpu().double()
        n_q = q.shape[1]
        g = n_q // self.n_kv
        o = torch.full(q.shape, float("nan"), dtype=torch.float64)
        err = torch.zeros_like(o)
        at = 0
        # of a weight: both it and the sum of weights are rounded (fp32: two fp16 terms leave 2^-22)
        u = 2.0 ** -22 if self.dt == torch.float32 else half_step(self.dt)
        for b, r in enumerate(self.rows):
            k, v = self.keys(b)
            end = min(self.lens[b], L if L is not None else self.lens[b])
            for i in range(r):
                n = min(max(self.lens[b] - r + i + 1, 0), end)
                if n == 0:
                    o[at] = 0
                    at += 1
                    continue
                kk, vv = (x[:n].repeat_interleave(g, 1) for x in (k, v))
                s = torch.einsum("hd,nhd->hn", q[at], kk) * scale
                p = torch.softmax(s, -1)
                o[at] = torch.einsum("hn,nhd->hd", p, vv)
                # scores: products of q in two fp16 terms, hd sums; the exponent's own rounding; then the weight's
                # (twice), exp2, and sums over n keys in fp32
                size = abs(scale) * torch.einsum("hd,nhd->hn", q[at].abs(), kk.abs()).amax(-1)
                ds = size * (2.0 ** -22 + (self.hd + 4) * U)
                e = 2 * ds + 2 * u + (n + 40) * U
                # weights below fp16's normal range are off by 2^-25 of the largest
                low = 0.0 if self.dt == torch.bfloat16 else n * 2.0 ** -25 * vv.abs().amax(0)
                err[at] = torch.einsum("hn,nhd->hd", p, vv.abs()) * e[:, None] + low
                at += 1
        return o, err

    def check(self, q, scale, got=None, L=None, **kw):
        got = self.attn(q, scale, L=L, **kw) if got is None else got
        ref, err = self.reference(q, scale, L)
        n = sum(self.rows)
        check_rounded(got.unflatten(1, (q.shape[1], self.hd))[:n], ref[:n], err[:n], self.dt)
        return got

    def q(self, n_q):
        return torch.randn(self.tokens, n_q, self.hd, generator=self.g).to(self.dt).to(self.dev)


# ------------------------------------------------------------------------------------------------ append

APPENDS = [  # page, lens, rows, ragged
    (16, [1], [1], False), (16, [17, 5, 32], [1, 1, 1], False), (7, [20, 3, 9], [3, 3, 3], False),
    (24, [100, 0, 31, 64], [40, 0, 31, 1], True), (1, [4, 9], [2, 9], True), (64, [3, 700], [1, 650], True),
    (8, [5] * 70, [1] * 70, True)]


@pytest.mark.parametrize("dt", DTYPES, ids=IDS)
@pytest.mark.parametrize("page,lens,rows,ragged", APPENDS)
@pytest.mark.parametrize("n_q,n_kv,hd,rot,inter", [(6, 2, 128, 128, False), (5, 5, 64, 32, True), (3, 1, 80, 38, False), (2, 3, 80, 40, False),
                                                   (2, 2, 64, None, False)])
def test_paged_kv_append(dev, dt, page, lens, rows, ragged, n_q, n_kv, hd, rot, inter):
    b = Batch(dev, dt, hd, n_kv, page, lens, rows, ragged=ragged, seed=len(lens) + page, extra=2 if ragged else 0)
    t = b.tokens
    qkv = torch.randn(t, (n_q + 2 * n_kv) * hd, generator=b.g).to(dt).to(dev)
    q, k, v = (x.unflatten(1, (-1, hd)) for x in qkv.split([n_q * hd, n_kv * hd, n_kv * hd], 1))
    rope = None if rot is None else Rope(freqs(rot, dev), inter, 1.05)
    pos = [x - r + i for x, r in zip(lens, rows) for i in range(r)]
    want_k, want_v = b.k.cpu().clone(), b.v.cpu().clone()
    q_out = torch.full((t, n_q, hd), 9.0, dtype=dt, device=dev)
    got = ops.paged_kv_append(k, v, b.k, b.v, b.page_table, b.seq_lens, cu_q=b.cu, rope=rope, q=q, q_out=q_out)
    assert got is q_out
    n = len(pos)
    p = torch.tensor(pos)
    exact = [(x[:n].cpu().double(), torch.zeros(n, x.shape[1], hd, dtype=torch.float64)) if rope is None else
             rotated(x[:n], p, rope) for x in (q, k)]
    check_rounded(q_out[:n], *exact[0], dt)
    assert (q_out[n:] == 9).all()  # tokens of no sequence
    seq = [s for s, r in enumerate(rows) for _ in range(r)]
    pages = torch.tensor([b.table[s][x // page] for s, x in zip(seq, pos)], dtype=torch.long)
    offs = p % page
    gk, gv = b.k.cpu(), b.v.cpu()
    check_rounded(gk[pages, offs], *exact[1], b.k.dtype)
    assert torch.equal(gv[pages, offs], v[:n].cpu().to(b.v.dtype))
    want_k[pages, offs], want_v[pages, offs] = gk[pages, offs], gv[pages, offs]
    for a, w in ((gk, want_k), (gv, want_v)):  # nothing else was written
        assert torch.equal(a.view(torch.int16), w.view(torch.int16))


def test_append_without_a_row(dev):
    """Negative positions, positions past the page list and entries that are no page write nothing; q is rotated where the
    position is one."""
    dt, hd, page = torch.float32, 64, 4
    kc = torch.full((3, page, 1, hd), 5.0, dtype=torch.float16, device=dev)
    vc = kc.clone()
    table = i32([[1, -1], [3, 0], [2, 1], [0, 0], [1, 1 << 30]], dev)
    lens = i32([5, 3, 9, 1, 6], dev)  # positions: 4 (page -1), 2 (page 3 of 3), 8 (past the list), 0, 5 (no page)
    x = torch.randn(5, 3, hd, generator=torch.Generator().manual_seed(1)).to(dev)
    rope = Rope(freqs(hd, dev))
    q = ops.paged_kv_append(x[:, :1], x[:, 1:2], kc, vc, table, lens, rope=rope, q=x[:, 2:])
    ref, err = rotated(x[:, 2:], torch.tensor([4, 2, 8, 0, 5]), rope)
    check_rounded(q, ref, err, dt)
    assert (kc[1:] == 5).all() and (vc[1:] == 5).all() and (kc[0, 1:] == 5).all()
    assert torch.equal(vc[0, 0, 0], x[3, 1].half())
    # more tokens than keys: the first ones have no position
    q_out = torch.full((4, 1, hd), 9.0, device=dev)
    ops.paged_kv_append(x[:4, :1], x[:4, 1:2], kc, vc, i32([[2]], dev), i32([3], dev), rope=rope, q=x[:4, 2:], q_out=q_out)
    assert (q_out[0] == 9).all() and (q_out[1:] != 9).any() and torch.equal(vc[2, :3, 0], x[1:4, 1].half())
    assert (kc[2, 3] == 5).all()


# ------------------------------------------------------------------------------------------------ attention

ATTN = [  # page, lens, rows, shared, ragged
    (16, [1], [1], 0, False),
    (16, [700], [1], 0, False),
    (16, [33, 64, 1, 200, 31, 32], [1] * 6, 0, False),
    (16, [0, 5, 0, 40], [1] * 4, 0, False),                # empty sequences in a padded batch
    (24, [300, 290, 301], [1] * 3, 256, False),            # a prefix that ends inside a page
    (7, [90, 64, 61, 200], [1] * 4, 60, False),            # pages of odd size
    (1, [40, 37], [1] * 2, 33, False),
    (16, [70, 20, 0, 64, 65], [1] * 5, 64, False),         # shorter than the prefix, empty, the prefix alone
    (32, [130, 140, 150], [5] * 3, 96, False),             # several tokens a sequence
    (16, [3, 40], [5] * 2, 0, False),                      # more tokens than keys
    (64, [530, 600, 513, 700], [18, 88, 1, 150], 512, True),  # prompts of different lengths behind a prefix
    (16, [75, 0, 90, 64, 33], [75, 0, 3, 1, 2], 0, True),
    (16, [100, 50], [80, 30], 40, True),                   # prompts that begin inside the prefix
    (8, [9] * 70, [1, 2] * 35, 3, True),
    (128, [2100, 1999], [1] * 2, 1900, False)]


@pytest.mark.parametrize("dt", DTYPES, ids=IDS)
@pytest.mark.parametrize("n_q,n_kv,hd", [(6, 2, 128), (4, 4, 64), (8, 1, 128)])
@pytest.mark.parametrize("page,lens,rows,shared,ragged", ATTN)
def test_paged_attn(dev, dt, n_q, n_kv, hd, page, lens, rows, shared, ragged):
    b = Batch(dev, dt, hd, n_kv, page, lens, rows, shared, ragged, seed=len(lens) * 3 + hd, extra=3 if ragged else 0)
    q = b.q(n_q)
    out = torch.full((b.tokens, n_q * hd), 9.0, dtype=dt, device=dev)
    b.check(q, hd ** -0.5, out=out)
    assert (out[sum(rows):] == 9).all()  # tokens of no sequence


@pytest.mark.parametrize("dt", DTYPES, ids=IDS)
@pytest.mark.parametrize("page,lens,rows,shared,ragged,n_q,n_kv,hd", [
    (16, [600, 650, 520, 0, 300], [1] * 5, 520, False, 6, 2, 128),          # one tile of the streaming form, empty, shorter
    (24, [700] * 9, [2] * 9, 640, False, 4, 2, 64),                          # 36 rows: two waves for the keys
    (7, [560 + i for i in range(40)], [1 + i % 3 for i in range(40)], 513, True, 3, 1, 64),
    (16, [900 + 9 * i for i in range(30)], [3] * 30, 800, False, 4, 1, 128),  # 360 rows: tiles of 128
    (64, [1500, 1400, 1290], [60, 1, 20], 1281, True, 8, 2, 128),
    (32, [515, 512, 100, 700], [4] * 4, 512, False, 4, 4, 128)])
def test_paged_attn_prefix_as_a_range_of_its_own(dev, dt, page, lens, rows, shared, ragged, n_q, n_kv, hd):
    b = Batch(dev, dt, hd, n_kv, page, lens, rows, shared, ragged, seed=shared, extra=2 if ragged else 0)
    q = b.q(n_q)
    out = torch.full((b.tokens, n_q * hd), 9.0, dtype=dt, device=dev)
    L = max(b.page_table.shape[1] * page, shared)
    ws = torch.full((ops.paged_attn_workspace_bytes(b.tokens, n_q, n_kv, hd, len(lens), L, shared),), 255, dtype=torch.uint8,
                    device=dev)
    b.check(q, hd ** -0.5, out=out, workspace=ws)
    assert (out[sum(rows):] == 9).all()
    # L at the prefix: no range of the sequences' own
    b.check(q, hd ** -0.5, L=shared)


def test_native_calls_and_python_wrappers_agree(dev, monkeypatch):
    """The same bits whichever of the two checks the arguments."""
    b = Batch(dev, torch.float16, 64, 2, 16, [200, 90, 150], [2, 2, 2], 64, seed=3)
    qkv = torch.randn(6, 8, 64, generator=b.g).half().to(dev)
    rope = Rope(freqs(64, dev), True, 1.25)
    pos = torch.arange(6, dtype=torch.int32, device=dev)
    tok, draft, target, u, _ = drafts(dev, 3, 2, 500, 4)
    k0, v0 = b.k.clone(), b.v.clone()

    def everything():
        b.k.copy_(k0)
        b.v.copy_(v0)
        r = [ops.rope_rotate(qkv, pos, rope), ops.rope_rotate(qkv, pos, rope, inverse=True)]
        r.append(ops.paged_kv_append(qkv[:, 4:6], qkv[:, 6:], b.k, b.v, b.page_table, b.seq_lens, rope=rope, q=qkv[:, :4]))
        assert ops.paged_kv_append(qkv[:, 4:6], qkv[:, 6:], b.k, b.v, b.page_table, b.seq_lens, rope=rope) is None
        r += [b.attn(r[-1], 0.125), b.attn(r[-1], 0.125, L=170), b.k.clone().view(torch.int16), b.v.clone().view(torch.int16)]
        r += [*ops.spec_verify(tok, draft, target, u), *ops.spec_verify(tok, None, target, u, n_draft=i32([1, 0, 2], dev))]
        return r

    assert all(getattr(ops, n) is not ops._left_to_python for n in ("_rope", "_append", "_paged", "_verify"))
    native = everything()
    for n in ("_rope", "_append", "_paged", "_verify"):
        monkeypatch.setattr(ops, n, ops._left_to_python)
    assert all(torch.equal(x, y) for x, y in zip(native, everything()))


@pytest.mark.parametrize("n_q,n_kv", [(64, 1), (20, 4), (7, 7), (48, 1)])
def test_paged_attn_group_sizes(dev, n_q, n_kv):
    b = Batch(dev, torch.float16, 64, n_kv, 16, [70, 100], [2, 2], 48, seed=n_q)
    b.check(b.q(n_q), 0.125)


@pytest.mark.parametrize("n_q,n_kv", [(1, 1), (3, 1), (10, 2)])
@pytest.mark.parametrize("n,shared", [(5, 130), (17, 520), (23, 520), (40, 520), (67, 520), (129, 130), (129, 520)])
def test_paged_attn_ragged_tails(dev, n, shared, n_q, n_kv):
    """Batches whose rows end inside a tile, the workspace full of NaN: every row of every range is written."""
    rows = [1 + (i * 7) % 3 for i in range(n)]
    b = Batch(dev, torch.float16, 64, n_kv, 8, [shared + 20 + 3 * (i % 40) for i in range(n)], rows, shared, True, seed=n, extra=1)
    q = b.q(n_q)
    L = b.page_table.shape[1] * 8
    ws = torch.full((ops.paged_attn_workspace_bytes(b.tokens, n_q, n_kv, 64, n, L, shared),), 255, dtype=torch.uint8, device=dev)
    b.check(q, 0.125, workspace=ws)


@pytest.mark.parametrize("dt", DTYPES, ids=IDS)
@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("n,rows,lens,shared,n_kv", [(70, 1, 540, 520, 8), (140, 1, 40, 0, 4), (3, 130, 400, 0, 64),
                                                     (3, 130, 500, 300, 64), (2, 300, 310, 0, 48)])
def test_paged_attn_more_tiles_than_places(dev, dt, ragged, n, rows, lens, shared, n_kv):
    """More tiles of rows and heads than the chip takes at once: those past whole rounds are split over it. The workspace is
    full of NaN, and a second call with other queries on it is right too."""
    r = [rows - (i % 2 if rows > 1 else 0) if ragged else rows for i in range(n)]
    b = Batch(dev, dt, 64, n_kv, 16, [lens + 5 * (i % 7) for i in range(n)], r, shared, ragged, seed=n)
    L = b.page_table.shape[1] * 16
    ws = torch.full((ops.paged_attn_workspace_bytes(b.tokens, n_kv, n_kv, 64, n, L, shared),), 255, dtype=torch.uint8, device=dev)
    for _ in range(2):
        b.check(b.q(n_kv), 0.125, workspace=ws if ws.numel() else None)


@pytest.mark.parametrize("dt", DTYPES, ids=IDS)
@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("n,rows,n_kv,hd", [(3, 1, 8, 64), (9, 1, 16, 64), (24, 1, 8, 128), (17, 1, 16, 64), (5, 40, 2, 64),
                                            (33, 3, 8, 64), (64, 2, 1, 64), (65, 2, 2, 64)])
def test_paged_attn_unequal_lengths(dev, dt, ragged, n, rows, n_kv, hd):
    """Sequences of unequal lengths, some empty, in every order of work: few and many of them, tiles that fill the places and
    tiles that have to be split over them twice."""
    r = [(0 if i % 11 == 4 else 1 + i % rows) if ragged else rows for i in range(n)]
    lens = [max(r[i], (37 * i * i + 300 * i) % (1900 if n < 10 else 700)) for i in range(n)]
    b = Batch(dev, dt, hd, n_kv, 16, lens, r, 0, ragged, seed=n)
    L = b.page_table.shape[1] * 16
    ws = torch.full((max(16, ops.paged_attn_workspace_bytes(b.tokens, n_kv, n_kv, hd, n, L, 0)),), 255, dtype=torch.uint8, device=dev)
    b.check(b.q(n_kv), 0.125, workspace=ws)


@pytest.mark.parametrize("dt", DTYPES, ids=IDS)
@pytest.mark.parametrize("n,n_q,n_kv", [(2, 4, 2), (70, 32, 32), (700, 32, 16)])
def test_paged_attn_shared_keys_alone(dev, dt, n, n_q, n_kv):
    """No key is a sequence's own: few tiles, whose shared keys are several ranges, and more tiles than compute units, whose
    shared keys are one."""
    b = Batch(dev, dt, 64, n_kv, 16, [520 + (i % 2) for i in range(n)], [1] * n, 512, seed=n)
    q = b.q(n_q)
    L = 512
    ws = torch.full((ops.paged_attn_workspace_bytes(n, n_q, n_kv, 64, n, L, 512),), 255, dtype=torch.uint8, device=dev)
    got = ops.paged_attn(q, b.k, b.v, b.page_table, b.seq_lens, 0.125, shared_pages=b.sp, shared_len=512, L=L, workspace=ws)
    at = torch.tensor(b.shared_pages, device=dev)
    k, v = (x[at].flatten(0, 1).double().repeat_interleave(n_q // n_kv, 1) for x in (b.k, b.v))  # [512, n_q, hd]
    s = torch.einsum("thd,jhd->thj", q.double().cpu(), k.cpu()) * 0.125
    ref = torch.einsum("thj,jhd->thd", s.softmax(-1), v.cpu()).flatten(1)
    # the weights' rounding and the result's, each half a step of at most max |v|; scores of 64 products in fp32, off by at
    # most 66 U sum |q k| scale < 66 U * 200 / 8 = 1e-4 (sum |q k| < 200: 64 normal pairs of mean 0.64), as is e^s
    assert (got.double().cpu() - ref).abs().max() <= (2 * half_step(dt) + 2e-4) * v.abs().max().item()


@pytest.mark.parametrize("scale", [-0.3, 0.0, 0.01, 2.0])
@pytest.mark.parametrize("dt", DTYPES, ids=IDS)
def test_paged_attn_scales(dev, dt, scale):
    b = Batch(dev, dt, 64, 2, 16, [90, 130], [1, 1], 64, seed=4)
    b.check(b.q(4), scale)


@pytest.mark.parametrize("dt", DTYPES, ids=IDS)
def test_paged_attn_strides_lengths_and_streams(dev, dt):
    """q as a slice of a fused row and off 16 bytes, a page table with a row pitch, L below the lengths, another stream."""
    b = Batch(dev, dt, 64, 2, 16, [100, 80, 33], [2, 2, 2], 32, seed=8)
    wide = torch.randn(6, 8 * 64 + 1, generator=b.g).to(dt).to(dev)
    for q in (wide[:, :-1].unflatten(1, (8, 64))[:, 2:6], wide[:, 1:].unflatten(1, (8, 64))):
        b.check(q, 0.125)
    q = b.q(4)
    want = b.check(q, 0.125)
    table = torch.full((3, 40), -3, dtype=torch.int32, device=dev)
    table[:, :b.page_table.shape[1]] = b.page_table
    plain, b.page_table = b.page_table, table[:, :plain_cols(b)]
    assert not b.page_table.is_contiguous() and torch.equal(b.attn(q, 0.125), want)
    b.page_table = plain
    for L in (32, 33, 64, 99):
        b.check(q, 0.125, L=L)
    s = torch.cuda.Stream(dev)
    s.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(s):
        got = b.attn(q, 0.125)
    torch.cuda.current_stream(dev).wait_stream(s)
    assert torch.equal(got, want)


def plain_cols(b):
    return b.page_table.shape[1]


def test_paged_attn_prefix_is_only_a_way_to_read(dev):
    """With the prefix's pages in every row of the table, reading them as shared or as each sequence's own agrees."""
    for dt in DTYPES:
        b = Batch(dev, dt, 128, 2, 16, [200, 150, 300], [1, 1, 1], 144, seed=2)
        b.page_table[:, :9] = b.sp
        b.table = b.page_table.tolist()
        q = b.q(6)
        b.check(q, 128 ** -0.5)
        own = ops.paged_attn(q, b.k, b.v, b.page_table, b.seq_lens, 128 ** -0.5)
        b.check(q, 128 ** -0.5, got=own)


def test_paged_attn_bad_pages_hold_no_keys(dev):
    """Entries outside the pool: their keys do not exist for the softmax; with none left a row is zero."""
    dt = torch.float16
    b = Batch(dev, dt, 64, 1, 16, [64, 48, 32], [1, 1, 1], seed=6)
    k, v = b.k.clone(), b.v.clone()
    table = b.page_table.clone()
    table[0, 1], table[1, 0], table[2, :2] = 1 << 30, -1, b.k.shape[0]
    q = b.q(2)
    got = ops.paged_attn(q, k, v, table, b.seq_lens, 0.125).unflatten(1, (2, 64)).cpu().double()
    for s, keep in ((0, list(range(16)) + list(range(32, 64))), (1, list(range(16, 48)))):
        kk, vv = (x[keep, 0] for x in b.keys(s))
        p = torch.softmax(q[s].cpu().double() @ kk.t() * 0.125, -1)
        assert ((got[s] - p @ vv).abs() <= 4 * half_step(dt) * (p @ vv.abs()) + 1e-5).all()
    assert (got[2] == 0).all()
    shared = i32([-1, b.table[0][1], 1 << 29], dev)  # two of three shared pages are none
    got = ops.paged_attn(q[:1], k, v, b.page_table[:1], i32([48], dev), 0.125, shared_pages=shared, shared_len=48)
    kk, vv = (x[16:32, 0] for x in b.keys(0))
    p = torch.softmax(q[0].cpu().double() @ kk.t() * 0.125, -1)
    assert ((got.unflatten(1, (2, 64))[0].cpu().double() - p @ vv).abs() <= 4 * half_step(dt) * (p @ vv.abs()) + 1e-5).all()


def test_paged_attn_nan_stays_in_its_row(dev):
    """A NaN query makes its own row NaN and no other; large scores neither overflow nor lose the others."""
    for dt in DTYPES:
        b = Batch(dev, dt, 128, 1, 16, [90, 70, 100], [1, 1, 1], 64, seed=3)
        q = b.q(4)
        q[1, 2, 5] = float("nan")
        got = b.attn(q, 0.1).unflatten(1, (4, 128))
        assert got[1, 2].isnan().all()
        ref, err = b.reference(q, 0.1)
        keep = torch.ones(3, 4, dtype=torch.bool)
        keep[1, 2] = False
        check_rounded(got.cpu()[keep], ref[keep], err[keep], dt)
        q = b.q(4) * 30
        b.check(q, 1.0)


@pytest.mark.parametrize("rows", [1, 9, 20, 40])
@pytest.mark.parametrize("dt", DTYPES, ids=IDS)
def test_paged_attn_many_small_weights(dev, dt, rows):
    """One key far above thousands of others: weights below fp16's normal range (2^-14) carry most of the sum."""
    b = Batch(dev, dt, 64, 1, 16, [3000], [rows], 2000, seed=rows)
    q = torch.ones(rows, 2, 64).to(dt).to(dev)
    b.k.copy_(torch.where(b.k.isnan(), b.k, torch.full_like(b.k, 0.25)))
    first = b.shared_pages[0]
    b.k[first, 3] = 0.25 + 10.5 / 8  # scores 2 and 2 + 10.5
    b.check(q, 0.125)


def test_paged_attn_cache_past_32_bits(dev):
    """Rows at byte offsets past 2^32 (and past 2^31 elements)."""
    n_kv, hd, page = 8, 128, 16
    pages = (1 << 32) // (page * n_kv * hd * 2) + 40
    k = torch.empty(pages, page, n_kv, hd, dtype=torch.bfloat16, device=dev)
    v = torch.empty_like(k)
    b = Batch(dev, torch.bfloat16, hd, n_kv, page, [100, 77], [1, 1], 32, seed=5)
    small = b.k.shape[0]
    at = pages - small
    k[at:], v[at:] = b.k, b.v
    k[:small], v[:small] = float("nan"), float("nan")
    q = b.q(8)
    want = b.attn(q, 0.09)
    table = torch.where(b.page_table >= 0, b.page_table + at, b.page_table)
    got = ops.paged_attn(q, k, v, table, b.seq_lens, 0.09, shared_pages=b.sp + at, shared_len=32)
    assert torch.equal(got, want)
    x = torch.randn(2, 2 * n_kv, hd, generator=b.g).bfloat16().to(dev)
    ops.paged_kv_append(x[:, :n_kv], x[:, n_kv:], k, v, table, b.seq_lens)
    for s, n in enumerate(b.lens):
        row = (table[s, (n - 1) // page], (n - 1) % page)
        assert torch.equal(k[row], x[s, :n_kv]) and torch.equal(v[row], x[s, n_kv:])


def test_paged_matches_the_dense_cache(dev):
    """One sequence: the paged operators against attn_bucket and rope_kv_write on the dense cache (fp32 angles there:
    positions are small)."""
    n_q, n_kv, hd, page, n = 6, 2, 128, 16, 150
    g = torch.Generator().manual_seed(12)
    qkv = torch.randn(n, (n_q + 2 * n_kv) * hd, generator=g).to(dev)
    f = freqs(hd, dev)
    t = torch.arange(256, device=dev)[:, None].float() * f
    cos, sin = (torch.cat([x, x], 1).contiguous() for x in (t.cos(), t.sin()))
    kd, vd = (torch.zeros(256, n_kv, hd, dtype=torch.float16, device=dev) for _ in range(2))
    start = i32([0], dev)
    dense = ops.rope_kv_write(qkv.clone(), cos, sin, kd, vd, n_q, n_kv, hd, start)[:, :n_q * hd].unflatten(1, (n_q, hd))
    kc, vc = (torch.zeros(12, page, n_kv, hd, dtype=torch.float16, device=dev) for _ in range(2))
    table = torch.randperm(12, generator=g)[:10].int().to(dev)[None]
    q, k, v = (x.unflatten(1, (-1, hd)) for x in qkv.split([n_q * hd, n_kv * hd, n_kv * hd], 1))
    lens = i32([n], dev)
    qr = ops.paged_kv_append(k, v, kc, vc, table, lens, rope=Rope(f), q=q)
    # fp32 angles: 150 * 2^-23 each, of values below 6
    assert (qr - dense).abs().max().item() <= 150 * 2.0 ** -23 * 12 + 12 * 8 * U
    rows = kc[table[0].long()].flatten(0, 1)[:n], vc[table[0].long()].flatten(0, 1)[:n]
    assert torch.equal(rows[1], vd[:n]) and (rows[0] - kd[:n]).abs().max().item() <= 8 * 2.0 ** -11
    kd[:n] = rows[0]
    a = ops.paged_attn(qr, kc, vc, table, lens, hd ** -0.5)
    c = ops.attn_bucket(qr, kd, vd, 256, start, hd ** -0.5)
    # both within 2 ds + .. of the exact result; scores below 12 in natural units, values below 6
    assert (a - c).abs().max().item() <= 2 * 6 * (2 * 12 * (2.0 ** -22 + 132 * U) + 200 * U)


# ------------------------------------------------------------------------------------------------ verification


def verified(tokens, draft, target, u, n_draft=None):
    """The rule in 64 bits, row by row."""
    b, k = tokens.shape
    v = target.shape[2]
    target, u = target.cpu().double(), u.cpu().double()
    draft = None if draft is None else draft.cpu().double()
    out, counts = [], []
    for r in range(b):
        n = k if n_draft is None else min(max(int(n_draft[r]), 0), k)
        a = 0
        while a < n:
            x = int(tokens[r, a])
            if not 0 <= x < v or not u[r, a] * (1.0 if draft is None else draft[r, a, x]) < target[r, a, x]:
                break
            a += 1
        w = target[r, a].clamp(min=0)
        if a < n:
            left = target[r, a] - (0 if draft is None else draft[r, a])
            if draft is None and 0 <= int(tokens[r, a]) < v:
                left[int(tokens[r, a])] = 0
            left = torch.where(left > 0, left, torch.zeros_like(left))
            w = left if left.sum() > 0 else w
        c = w.cumsum(0)
        if c[-1] > 0:
            over = (c > u[r, k] * c[-1]).nonzero()
            nxt = int(over[0]) if len(over) else int(w.nonzero()[-1])
        else:
            nxt = -1
        out.append([int(t) for t in tokens[r, :a]] + [nxt] + [-1] * (k - a))
        counts.append(a)
    return torch.tensor(out, dtype=torch.int32), torch.tensor(counts, dtype=torch.int32)


def drafts(dev, b, k, v, seed, near=0.5):
    g = torch.Generator().manual_seed(seed)
    z = torch.randn(b, k + 1, v, generator=g) * 2
    target = torch.softmax(z, -1)
    draft = torch.softmax(z[:, :k] + near * torch.randn(b, k, v, generator=g), -1)
    tokens = (torch.multinomial(draft.flatten(0, 1), 1, generator=g).view(b, k).int() if k else
              torch.zeros(b, 0, dtype=torch.int32))
    u = torch.rand(b, k + 1, generator=g)
    return [x.to(dev) for x in (tokens, draft, target, u)] + [g]


@pytest.mark.parametrize("given", [True, False])
@pytest.mark.parametrize("b,k,v", [(1, 1, 1), (1, 4, 7), (3, 1, 32000), (5, 8, 4096), (2, 3, 4097), (4, 5, 12289), (33, 2, 100),
                                   (2, 70, 257), (3, 0, 5000), (2, 2, 1500001)])
def test_spec_verify(dev, given, b, k, v):
    tokens, draft, target, u, g = drafts(dev, b, k, v, b * 100 + k)
    draft = draft if given else None
    n = torch.randint(0, k + 1, (b,), generator=g).int().to(dev)
    for nd in (None, n):
        got = ops.spec_verify(tokens, draft, target, u, n_draft=nd)
        want = verified(tokens, draft, target, u, nd)
        assert torch.equal(got[0].cpu(), want[0]) and torch.equal(got[1].cpu(), want[1])


def test_spec_verify_borders(dev):
    """Certain and impossible tokens, u at 0 and just below 1, running sums on the border, equal distributions, rows of zeros,
    weights that are no numbers, tokens and counts outside their range."""
    v = 6
    p = torch.tensor([0.25, 0.0, 0.25, 0.25, 0.25, 0.0])
    q = torch.tensor([0.5, 0.5, 0.0, 0.0, 0.0, 0.0])
    nan, inf = float("nan"), float("inf")
    top = 1 - 2.0 ** -24
    rows = [  # token, draft, target 0, target 1, u0, u1, drafts
        (0, q, p, p, 0.0, 0.0, 1), (0, q, p, p, 0.5, 0.0, 1), (0, q, p, p, 0.499999, 0.0, 1), (0, q, p, p, 0.75, 0.0, 1),
        (0, q, p, p, 0.75, top, 1), (0, q, p, p, 0.75, 0.5, 1), (1, q, p, p, 0.0, 0.3, 1), (2, q, p, p, 0.99, 0.25, 1),
        (2, q, p, p, 0.99, 0.75, 1), (2, q, p, p, 0.99, top, 1), (1, p, p, p, 0.5, 0.6, 1), (5, p, p, p, 0.0, 0.25, 1),
        (0, q, 0 * p, p, 0.1, 0.5, 1), (0, q, p, 0 * p, 0.1, 0.5, 1), (0, q, p, p, nan, 0.5, 1), (-1, q, p, p, 0.0, 0.5, 1),
        (6, q, p, p, 0.0, 0.5, 1), (1 << 30, q, p, p, 0.0, 0.5, 1), (0, q, p, p, 0.9, 0.5, 0), (0, q, p, p, 0.9, 0.5, -4),
        (0, q, p, p, 0.1, 0.5, 9), (0, q, torch.tensor([0.1, nan, 0.2, -1.0, nan, 0.7]), p, 0.9, 0.5, 1),
        (3, q, p, torch.tensor([nan, 0.5, -inf, 0.5, 0.0, nan]), 0.9, 0.5, 1), (0, q, p, p, 0.75, 1.0, 1)]
    tok = i32([[r[0]] for r in rows], dev)
    draft = torch.stack([r[1] for r in rows])[:, None].to(dev)
    target = torch.stack([torch.stack([r[2], r[3]]) for r in rows]).to(dev)
    u = torch.tensor([[r[4], r[5]] for r in rows], device=dev)
    n = i32([r[6] for r in rows], dev)
    clean = torch.where(target > 0, target, torch.zeros_like(target))  # no numbers and negative ones count as zero
    got = ops.spec_verify(tok, draft, target, u, n_draft=n)
    want = verified(tok, draft, clean, u, n)
    assert torch.equal(got[0].cpu(), want[0]) and torch.equal(got[1].cpu(), want[1])
    got = ops.spec_verify(tok, None, target, u, n_draft=n)
    want = verified(tok, None, clean, u, n)
    assert torch.equal(got[0].cpu(), want[0]) and torch.equal(got[1].cpu(), want[1])
    assert got[0].shape == (len(rows), 2) and v == target.shape[2]


def test_spec_verify_strides_and_unaligned_rows(dev):
    tokens, draft, target, u, _ = drafts(dev, 4, 3, 1001, 17)
    wide = torch.zeros(4, 4, 1003, device=dev)
    wide[..., 1:1002] = target
    first = draft.transpose(0, 1).contiguous().transpose(0, 1)
    both = torch.zeros(4, 9, dtype=torch.int32, device=dev)
    both[:, 2:5] = tokens
    got = ops.spec_verify(both[:, 2:5], first, wide[..., 1:1002], u)
    want = verified(tokens, draft, target, u)
    assert torch.equal(got[0].cpu(), want[0]) and torch.equal(got[1].cpu(), want[1])


def test_spec_verify_keeps_the_target_distribution(dev):
    """Over evenly spread uniforms the first token out has the target's distribution, whatever the draft's."""
    p, q = torch.tensor([0.5, 0.2, 0.2, 0.1]), torch.tensor([0.1, 0.6, 0.1, 0.2])
    m = 200
    grid = (torch.arange(m).double() + 0.5) / m
    total = torch.zeros(4, dtype=torch.float64)
    for x in range(4):
        u = torch.stack(torch.meshgrid(grid, grid, indexing="ij"), -1).view(-1, 2).float().to(dev)
        n = u.shape[0]
        tok = torch.full((n, 1), x, dtype=torch.int32, device=dev)
        out, _ = ops.spec_verify(tok, q.expand(n, 1, 4).to(dev), p.expand(n, 2, 4).to(dev), u)
        total += q[x].double() * torch.bincount(out[:, 0].long().cpu(), minlength=4).double() / n
    # a border between two grid points moves at most one of m steps, in the acceptance and in the draw
    assert (total - p.double()).abs().max().item() <= 2.0 / m


# ------------------------------------------------------------------------------------------------ graphs and together


def test_captured_calls_serve_later_steps(dev):
    """One capture of append and attention, replayed while lengths, tokens and pages change on the device; each replay
    equals the eager calls. Two graphs on one workspace."""
    dt, n_q, n_kv, hd, page = torch.float32, 4, 2, 64, 16
    b = Batch(dev, dt, hd, n_kv, page, [60, 33, 47], [1, 1, 1], 32, seed=21)
    b.page_table[:, 2:5] = i32([[0, 1, 2], [3, 4, 5], [6, 7, 8]], dev)
    pool = (9 + 3, page, n_kv, hd)
    k0, v0 = (torch.randn(pool, generator=b.g).half().to(dev) for _ in range(2))
    sp = i32([10, 11], dev)
    rope = Rope(freqs(hd, dev))
    qkv = torch.zeros(3, n_q + 2 * n_kv, hd, device=dev)
    lens = b.seq_lens.clone()
    L = 80
    ws = torch.empty(ops.paged_attn_workspace_bytes(3, n_q, n_kv, hd, 3, L, 32), dtype=torch.uint8, device=dev)
    kc, vc = k0.clone(), v0.clone()
    outs = [torch.zeros(3, n_q * hd, device=dev) for _ in range(2)]

    def step(kc, vc, out, scale):
        q = ops.paged_kv_append(qkv[:, n_q:n_q + n_kv], qkv[:, n_q + n_kv:], kc, vc, b.page_table, lens, rope=rope,
                                q=qkv[:, :n_q])
        ops.paged_attn(q, kc, vc, b.page_table, lens, scale, shared_pages=sp, shared_len=32, L=L, workspace=ws, out=out)

    step(k0.clone(), v0.clone(), outs[0].clone(), 0.1)
    torch.cuda.synchronize()
    graphs = []
    for out, scale in zip(outs, (0.125, 0.2)):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            step(kc, vc, out, scale)
    ke, ve = k0.clone(), v0.clone()
    kc.copy_(k0)
    vc.copy_(v0)
    for i in range(4):
        qkv.copy_(torch.randn(qkv.shape, generator=b.g))
        for g, out, scale in zip(graphs, outs, (0.125, 0.2)):
            g.replay()
            want = torch.zeros_like(out)
            step(ke, ve, want, scale)
            torch.cuda.synchronize()
            assert torch.equal(out, want) and torch.equal(kc, ke) and torch.equal(vc, ve)
        lens.add_(i32([1, 5, 0], dev))


def test_captured_verification(dev):
    tokens, draft, target, u, g = drafts(dev, 3, 4, 9000, 5)
    ws = torch.empty(ops.spec_verify_workspace_bytes(3, 4, 9000), dtype=torch.uint8, device=dev)
    ops.spec_verify(tokens, draft, target, u, workspace=ws)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.spec_verify(tokens, draft, target, u, workspace=ws)
    for seed in (6, 7, 8):
        t2, d2, p2, u2, _ = drafts(dev, 3, 4, 9000, seed)
        for a, x in ((tokens, t2), (draft, d2), (target, p2), (u, u2)):
            a.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        want = verified(tokens, draft, target, u)
        assert torch.equal(got[0].cpu(), want[0]) and torch.equal(got[1].cpu(), want[1])


def test_serving_a_batch_with_drafts(dev):
    """A one-layer model served in a batch behind a common prompt: the prefix once, prompts of different lengths, then rounds in
    which drafted tokens are appended, attended to, verified and, where refused, overwritten. Every round's target
    probabilities are those of the plain model on the tokens so far, and the tokens follow the rule."""
    n_q, n_kv, hd, page, vocab, dim, k = 4, 2, 64, 8, 300, 128, 3
    g = torch.Generator().manual_seed(31)
    embed = (torch.randn(vocab, dim, generator=g)).to(dev)
    wqkv = (torch.randn((n_q + 2 * n_kv) * hd, dim, generator=g) * dim ** -0.5).to(dev)
    wo = (torch.randn(vocab, n_q * hd, generator=g) * 0.4).to(dev)
    rope = Rope(freqs(hd, dev, 10000.0))
    scale = hd ** -0.5
    prefix = torch.randint(0, vocab, (21,), generator=g).tolist()
    prompts = [torch.randint(0, vocab, (n,), generator=g).tolist() for n in (1, 9, 4)]
    n = len(prompts)

    pool = 40
    kc, vc = (torch.full((pool, page, n_kv, hd), float("nan"), dtype=torch.float16, device=dev) for _ in range(2))
    order = torch.randperm(pool, generator=g).int()
    shared = order[:3].to(dev)  # 21 tokens on 3 pages of 8: the third belongs to the prefix alone past them
    table = order[3:3 + 3 * 8].view(3, 8).to(dev)
    table[:, :2] = shared[:2]

    def forward(tokens, lens, cu, table, shared_len):
        """tokens [T] of the batch -> target probabilities [T, vocab]."""
        qkv = ops_linear(embed[tokens.long()], wqkv)
        q, kk, vv = (x.unflatten(1, (-1, hd)) for x in qkv.split([n_q * hd, n_kv * hd, n_kv * hd], 1))
        q = ops.paged_kv_append(kk, vv, kc, vc, table, lens, cu_q=cu, rope=rope, q=q)
        o = ops.paged_attn(q, kc, vc, table, lens, scale, cu_q=cu, shared_pages=shared if shared_len else None,
                           shared_len=shared_len)
        return torch.softmax(ops_linear(o, wo), -1)

    def ops_linear(x, w):
        return (x.double() @ w.double().t()).float()

    def plain(tokens):
        """The plain model's probabilities after each token, in 64 bits."""
        x = embed.cpu().double()[tokens] @ wqkv.cpu().double().t()
        q, kk, vv = (y.unflatten(1, (-1, hd)) for y in x.split([n_q * hd, n_kv * hd, n_kv * hd], 1))
        pos = torch.arange(len(tokens))
        q, kk = rotated(q, pos, rope)[0], rotated(kk, pos, rope)[0].half().double()
        kk, vv = (y.repeat_interleave(n_q // n_kv, 1) for y in (kk, vv.half().double()))
        s = torch.einsum("ihd,jhd->hij", q, kk) * scale
        s = s.masked_fill(pos[None, None] > pos[None, :, None], -math.inf)
        o = torch.einsum("hij,jhd->ihd", torch.softmax(s, -1), vv).flatten(1)
        return torch.softmax(o @ wo.cpu().double().t(), -1)

    # the prefix alone, into its pages
    forward(i32(prefix, dev), i32([21], dev), None, shared[None], 0)
    # the third page of the prefix ends inside: its rows are copied to each sequence's own third page by nobody, for the
    # shared list serves positions 16 .. 20 and the table the rest
    seqs = [prefix + p for p in prompts]
    rows = [len(p) for p in prompts]
    cu = i32([0, rows[0], rows[0] + rows[1], sum(rows)], dev)
    probs = forward(i32([t for p in prompts for t in p], dev), i32([len(s) for s in seqs], dev), cu, table, 21)
    for b in range(n):
        p = plain(seqs[b])[21:]
        assert (probs[int(cu[b]):int(cu[b + 1])].cpu().double() - p).abs().max().item() <= 1e-3
        seqs[b].append(int(p[-1].argmax()))
    for _ in range(4):
        # drafts: a sharpened copy of the target's previous distribution, given at random
        q = torch.softmax(torch.randn(n, k, vocab, generator=g) * 2, -1)
        tok = torch.multinomial(q.flatten(0, 1), 1, generator=g).view(n, k).int()
        for b in range(n):  # some of them good ones
            want = plain(seqs[b])[-1]
            tok[b, 0] = int(want.argmax())
            q[b, 0] = torch.nn.functional.one_hot(want.argmax(), vocab).float()
        step = torch.tensor([[s[-1]] + t.tolist() for s, t in zip(seqs, tok)], dtype=torch.int32)
        lens = i32([len(s) + k for s in seqs], dev)
        target = forward(step.flatten().to(dev), lens, None, table, 21).view(n, k + 1, vocab)
        u = torch.rand(n, k + 1, generator=g).to(dev)
        out, count = ops.spec_verify(tok.to(dev), q.to(dev), target, u)
        for b in range(n):
            p = plain(seqs[b] + tok[b].tolist())[-(k + 1):]
            # the cache holds fp16 keys, equal to the plain model's but where a rounding falls the other way
            assert (target[b].cpu().double() - p).abs().max().item() <= 1e-3
        want = verified(tok, q, target, u)
        assert torch.equal(out.cpu(), want[0]) and torch.equal(count.cpu(), want[1])
        for b in range(n):
            seqs[b] += out[b, :int(count[b]) + 1].tolist()
        assert all(0 <= t < vocab for s in seqs for t in s)
    assert len({len(s) for s in seqs}) >= 1 and max(len(s) for s in seqs) + k <= 64
