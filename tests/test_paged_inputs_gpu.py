"""Batched serving: inputs that a caller may pass and that are laid out in unusual ways. References in 64 bits."""

import pytest
import torch

from test_paged_gpu import Batch, half_step

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


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
