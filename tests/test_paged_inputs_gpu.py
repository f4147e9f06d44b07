"""Batched serving: inputs that a caller may pass and that are laid out in unusual ways. References in 64 bits."""

import pytest
import torch

from q4llm import ops
from test_paged_gpu import DTYPES, IDS, Batch, check_rounded, half_step

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


@pytest.mark.parametrize("dt", DTYPES, ids=IDS)
@pytest.mark.parametrize("shared,cols", [(100, 1), (100, 6), (640, 1), (640, 39)])
@pytest.mark.parametrize("rows,ragged", [([1] * 6, False), ([5] * 6, False), ([1, 7, 140, 2, 3, 9], True)])
def test_a_page_table_narrower_than_the_prefix(dev, dt, shared, cols, rows, ragged):
    """Keys of the prefix come from shared_pages, whatever page_table holds; the keys behind it have no page here."""
    page, hd = 16, 64
    lens = [shared, shared - 3, shared + 9, 20, shared, shared + 400]
    b = Batch(dev, dt, hd, 2, page, lens, rows, shared, ragged, seed=shared + cols)
    b.page_table = torch.full((6, cols), 1 << 20, dtype=torch.int32, device=dev)  # no page of the pool
    b.check(b.q(6), hd ** -0.5, L=shared)  # (reference: no key from `shared` on)
    got = b.attn(b.q(6), hd ** -0.5, L=shared + 512)
    assert torch.isfinite(got).all()


@pytest.mark.parametrize("dt", DTYPES, ids=IDS)
@pytest.mark.parametrize("shared", [100, 640])
def test_a_page_table_wider_than_the_prefix_ends_before_the_keys(dev, dt, shared):
    """Positions from max_pages * page_size on have no page: the keys before them are all there are."""
    page, hd, cols = 16, 64, shared // 16 + 2
    lens = [shared + 200, shared + 3, shared + 40, shared]
    b = Batch(dev, dt, hd, 2, page, lens, [1] * 4, shared, seed=shared)
    b.page_table = b.page_table[:, :cols].contiguous()
    q = b.q(6)
    ref, err = b.reference(q, hd ** -0.5, L=cols * page)
    got = b.attn(q, hd ** -0.5, L=max(lens))
    check_rounded(got.unflatten(1, (6, hd)), ref, err, dt)


@pytest.mark.parametrize("dt", DTYPES, ids=IDS)
def test_queries_off_16_bytes_and_strides_of_single_rows(dev, dt):
    """q that starts between 16-byte words, and q whose one token or one head has a stride that is no multiple of 16 bytes: the same
    bits as an aligned copy of it gives."""
    hd = 64
    one = Batch(dev, dt, hd, 1, 16, [70], [1], seed=1)
    more = Batch(dev, dt, hd, 1, 16, [70, 33], [2, 2], seed=2)
    for b, n_q in ((one, 1), (one, 3), (more, 1), (more, 4)):
        q = b.q(n_q)
        want = b.check(q, hd ** -0.5)
        t = q.shape[0]
        flat = torch.zeros(q.numel() + 8, dtype=dt, device=dev)
        flat[1:1 + q.numel()] = q.flatten()
        shifted = flat[1:1 + q.numel()].view(t, n_q, hd)
        odd = torch.zeros(2 * q.numel() + 64, dtype=dt, device=dev)
        strides = (n_q * hd if t > 1 else 1, hd if n_q > 1 else 3, 1)
        strided = odd.as_strided(q.shape, strides).copy_(q)
        for x in (shifted, strided):
            assert torch.equal(b.attn(x, hd ** -0.5), want)


@pytest.mark.parametrize("dt", DTYPES, ids=IDS)
def test_no_sequence_and_no_token(dev, dt):
    hd = 64
    k = torch.zeros(3, 16, 2, hd, dtype=torch.bfloat16 if dt == torch.bfloat16 else torch.float16, device=dev)
    q = torch.zeros(0, 4, hd, dtype=dt, device=dev)
    for batch in (0, 2):
        table, lens = torch.zeros(batch, 4, dtype=torch.int32, device=dev), torch.zeros(batch, dtype=torch.int32, device=dev)
        assert ops.paged_attn(q, k, k.clone(), table, lens, 0.125).shape == (0, 4 * hd)
        assert ops.paged_kv_append(q[:, :2], q[:, :2], k, k.clone(), table, lens, q=q).shape == (0, 4, hd)
    assert ops.rope_rotate(q, lens[:0], ops_rope(dev)).shape == (0, 4, hd)


def ops_rope(dev):
    from q4llm.rope import Rope
    return Rope(torch.ones(16, device=dev))


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("rows,lens,shared", [([1, 1, 1], [9, 30, 17], 0), ([12, 5, 17], [12, 30, 17], 0), ([150, 90, 3], [150, 95, 40], 0),
                                              ([1, 2, 9], [530, 540, 525], 516)])
def test_16_bit_weights_are_as_exact_as_sums_in_32_bits(dev, dt, hd, rows, lens, shared):
    """The softmax weights are not rounded to the activations' type: the result is off by its own rounding and little else."""
    n_q, n_kv = 8, 2
    b = Batch(dev, dt, hd, n_kv, 16, lens, rows, shared, ragged=True, seed=hd + len(lens))
    q = b.q(n_q)
    got = b.attn(q, 0.5).unflatten(1, (n_q, hd)).cpu().double()
    ref, _ = b.reference(q, 0.5)
    qq, at = q.cpu().double(), 0
    for s, r in enumerate(rows):
        k, v = b.keys(s)
        for i in range(r):
            n = lens[s] - r + i + 1
            kk, vv = (x[:n].repeat_interleave(n_q // n_kv, 1) for x in (k, v))
            z = torch.einsum("hd,nhd->hn", qq[at], kk) * 0.5
            size = torch.einsum("hn,nhd->hd", torch.softmax(z, -1), vv.abs())
            # a score: hd products summed in fp32 and the exponent's rounding; a weight: two terms of its type, exp2; their sums: fp32,
            # of 16 products at a time, over the blocks and ranges of keys
            ds = 0.5 * torch.einsum("hd,nhd->hn", qq[at].abs(), kk.abs()).amax(-1, keepdim=True) * (hd / 8 + 4) * U
            e = 2 * ds + 2 * (2.0 ** -22 if dt == torch.float16 else 2.0 ** -17) + (n / 16 + 32) * U
            tol = e * size + half_step(dt) * (ref[at].abs() + e * size) + torch.finfo(dt).smallest_normal * torch.finfo(dt).eps
            worst = ((got[at] - ref[at]).abs() / tol).max().item()
            assert worst <= 1, (s, i, worst)
            at += 1


@pytest.mark.parametrize("ragged", [False, True])
def test_the_wrapper_takes_the_workspace_of_its_own_form(dev, ragged):
    """Nothing beside the result for 64 single tokens of at most 1000 keys without cu_q; and that query's bytes are enough."""
    n, n_q, n_kv, hd, L = 64, 24, 8, 128, 1000
    b = Batch(dev, torch.float16, hd, n_kv, 16, [1 + 2 * i for i in range(n)], [1] * n, 0, ragged)
    q = b.q(n_q)
    need = ops.paged_attn_workspace_bytes(n, n_q, n_kv, hd, n, L, 0, ragged)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    out = b.check(q, hd ** -0.5, L=L)
    assert torch.cuda.max_memory_allocated() - before <= max(need, 16) + out.numel() * 2 + 4096
    assert (need == 0) == (not ragged)
    ws = torch.full((max(need, 16),), 255, dtype=torch.uint8, device=dev)
    assert torch.equal(b.attn(q, hd ** -0.5, L=L, workspace=ws), out)
