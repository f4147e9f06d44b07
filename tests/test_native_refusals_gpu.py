"""The native call path of the batched operators takes a call whose every operand is as documented, and leaves each that has one
operand of another type, shape, layout or device to the Python wrapper. Operands that are too small are parts of larger ones."""

import pytest
import torch

from q4llm import ops

pytestmark = pytest.mark.gpu

HD, N_Q, N_KV, PAGE, PAGES, T = 64, 4, 2, 16, 6, 3


def i32(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def variants(x):
    """The operand x in another type, with a dim less, with a row less, with its last dim strided, and on the host."""
    other = torch.int64 if x.dtype == torch.int32 else torch.float64
    wide = torch.zeros(*x.shape[:-1], 2 * x.shape[-1], dtype=x.dtype, device=x.device)
    out = [x.to(other), x[0], x.cpu(), x.new_zeros(x.shape[0] + 1, *x.shape[1:])[:-2] if x.shape[0] > 1 else x.new_zeros(2, *x.shape[1:])]
    if x.shape[-1] > 1:
        out.append(wide[..., ::2])
    return out


def each_refused(fn, ok, operands, others):
    """fn(*ok) answers; with one of `operands` replaced by each of its variants, or ok[i] by a value of others[i], it does not."""
    for i in operands:
        for k, bad in enumerate(variants(ok[i])):
            assert fn(*ok[:i], bad, *ok[i + 1:]) is None, (i, k)
        for bad in (1, "x", object()):
            assert fn(*ok[:i], bad, *ok[i + 1:]) is None, (i, bad)
    for i, values in others.items():
        for bad in values:
            assert fn(*ok[:i], bad, *ok[i + 1:]) is None, (i, bad)
    assert fn(*ok[:-1]) is None and fn(*ok, None) is None and fn() is None
    assert fn(*ok) is not None
    torch.cuda.synchronize()


@pytest.fixture
def mod():
    from q4llm._lib import native_calls
    m = native_calls()
    assert m is not None
    return m


def caches(dev, dt=torch.float16):
    return [torch.zeros(PAGES, PAGE, N_KV, HD, dtype=dt, device=dev) for _ in range(2)]


def test_rope(dev, mod):
    x = torch.randn(T, N_Q, HD, device=dev)
    ok = [x, i32([0, 5, 9], dev), torch.ones(HD // 2, device=dev), False, 1.0, False, torch.empty_like(x)]
    assert mod.rope(*ok) is ok[-1] and mod.rope(*ok[:-1], None) is not None
    # x of another type or size is refused beside this `out`; frequencies for more dims than a head has
    each_refused(mod.rope, ok, [0, 1, 6], {2: [torch.ones(HD // 2 + 1, device=dev), torch.ones(HD // 2), torch.ones(HD // 2, device=dev).double(),
                                               torch.ones(HD, device=dev)[::2], torch.ones(1, HD // 2, device=dev), None, 3],
                                           3: [None, 1, "x"], 4: [None, 1, "x"], 5: [None, 0, "x"]})


@pytest.mark.parametrize("ragged", [False, True])
def test_append(dev, mod, ragged):
    k, v = (torch.randn(T, N_KV, HD, device=dev) for _ in range(2))
    q = torch.randn(T, N_Q, HD, device=dev)
    kc, vc = caches(dev)
    cu = i32([0, 1, 2, 3], dev) if ragged else None
    ok = [k, v, kc, vc, i32([[0], [1], [2]], dev), i32([1, 2, 3], dev), cu, torch.ones(HD // 2, device=dev), False, 1.0, q, torch.empty_like(q)]
    assert mod.append(*ok) is ok[-1] and mod.append(*ok[:10], None, None) is True
    each_refused(mod.append, ok, [0, 1, 3, 5, 10, 11] + ([6] if ragged else []),
                 {2: [kc.float(), kc.bfloat16(), kc[:, :, :1], kc[0], kc.transpose(1, 2), kc.cpu(), kc[:-1]],
                  4: [ok[4].long(), ok[4][0], ok[4].cpu(), i32([[0, 9]] * 3, dev)[:, ::2].expand(3, 1)[:2], ok[4][:0]],
                  7: [torch.ones(HD // 2 + 1, device=dev), torch.ones(HD // 2), torch.ones(HD // 2, device=dev).half(), 3],
                  8: [None, 1], 9: [None, 1], 10: [None]})  # (q_out without q)
    if not ragged:
        assert mod.append(*[x[:2] if i in (0, 1, 10, 11) else x for i, x in enumerate(ok)]) is None  # 2 tokens of 3 sequences


@pytest.mark.parametrize("ragged", [False, True])
def test_paged(dev, mod, ragged):
    q = torch.randn(T, N_Q, HD, device=dev)
    kc, vc = caches(dev)
    cu = i32([0, 1, 2, 3], dev) if ragged else None
    sp = i32([3, 4], dev)
    ws = torch.empty(1 << 20, dtype=torch.uint8, device=dev)
    out = torch.empty(T, N_Q * HD, device=dev)
    ok = [q, kc, vc, i32([[0, 1, 5], [1, 2, 5], [2, 0, 5]], dev), i32([33, 40, 47], dev), 0.125, cu, sp, 20, 48, ws, out]
    assert mod.paged(*ok) is out and mod.paged(*ok[:9], None, None, None) is not None
    flat = torch.zeros(q.numel() + 4, device=dev)
    each_refused(mod.paged, ok, [0, 2, 4, 11] + ([6] if ragged else []),
                 {0: [flat[1:-3].view(q.shape), torch.zeros(T, N_Q, HD + 1, device=dev)[..., :HD], q.bfloat16(), q[:, :3], q[..., :32]],
                  1: [kc.float(), kc.bfloat16(), kc[:, :, :1], kc[0], kc.transpose(1, 2), kc.cpu(), kc[:-1]],
                  3: [ok[3].long(), ok[3][0], ok[3].cpu(), i32([[0] * 6] * 3, dev)[:, ::2], ok[3][:2]],
                  5: [None, 1, "x", float("nan"), float("inf")], 7: [None, sp.long(), sp.cpu(), sp[:1], sp[None], i32([0] * 4, dev)[::2], 3],
                  8: [-1, 33, None, 1 << 40, 49], 9: [0, -1, "x", 1 << 40, 19, (1 << 30) + 1],
                  10: [ws.int(), ws.cpu(), ws[::2], 3]})
    big = ok[:9] + [4096, ws[:16], out]
    assert mod.paged(*big) is None  # a workspace that is too small


def test_verify(dev, mod):
    b, k, v = 2, 3, 50
    tok, u = torch.zeros(b, k, dtype=torch.int32, device=dev), torch.rand(b, k + 1, device=dev)
    draft, target = torch.rand(b, k, v, device=dev), torch.rand(b, k + 1, v, device=dev)
    ws = torch.empty(1 << 12, dtype=torch.uint8, device=dev)
    ok = [tok, draft, target, u, i32([3, 1], dev), ws]
    out, accepted = mod.verify(*ok)
    assert out.shape == (b, k + 1) and accepted.shape == (b,) and mod.verify(tok, None, target, u, None, None) is not None
    each_refused(mod.verify, ok, [0, 1, 2, 3, 4], {5: [ws.int(), ws.cpu(), ws[:16], ws[::2], 3]})


def test_the_python_wrapper_answers_what_the_native_path_leaves(dev, mod):
    """q off 16 bytes: left by the native path, copied by the wrapper; the same bits."""
    q = torch.randn(T, N_Q, HD, device=dev)
    kc, vc = caches(dev)
    vc.normal_()
    table, lens = i32([[0], [1], [2]], dev), i32([3, 9, 16], dev)
    flat = torch.zeros(q.numel() + 4, device=dev)
    odd = flat[1:-3].view(q.shape).copy_(q)
    assert mod.paged(odd, kc, vc, table, lens, 0.125, None, None, 0, None, None, None) is None
    assert torch.equal(ops.paged_attn(odd, kc, vc, table, lens, 0.125), ops.paged_attn(q, kc, vc, table, lens, 0.125))
