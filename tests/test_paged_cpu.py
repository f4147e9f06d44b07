"""Batched serving over a paged cache without a GPU: what the library and the tensor wrappers refuse before touching the
device, and the frequencies of scaled rotary positions."""

import ctypes as C
import math

import pytest
import torch

from q4llm import ops
from q4llm._lib import LIB
from q4llm.rope import Rope, inv_freq, rope_params

ERR = dict(NULL=-1, SHAPE=-2, ALIGN=-3, DTYPE=-4, WORKSPACE=-5, RANGE=-6, UNSUPPORTED=-7)
FAKE = 0x1000
F32, F16, BF16 = 0, 1, 2


def paged(**kw):
    base = dict(k_cache=FAKE, v_cache=FAKE, page_table=FAKE, seq_lens=FAKE, cu_q=None, num_pages=10, table_stride=4, dtype=F16,
                page_size=16, n_kv=2, head_dim=64, batch=3, max_pages=4)
    return ops._PagedC(**{**base, **kw})


def rope(**kw):
    return ops._RopeC(**{**dict(inv_freq=FAKE, rot_dim=64, layout=0, mscale=1.0), **kw})


ROTATE = dict(x=FAKE, xr=256, xh=64, y=FAKE, yr=256, yh=64, dt=F32, T=5, heads=4, hd=64, pos=FAKE, rope=rope(), inv=0, st=None)


@pytest.mark.parametrize("bad,code", [
    (dict(x=None), "NULL"), (dict(y=None), "NULL"), (dict(pos=None), "NULL"), (dict(rope=None), "NULL"),
    (dict(rope=rope(inv_freq=None)), "NULL"), (dict(dt=3), "DTYPE"), (dict(dt=-1), "DTYPE"), (dict(T=-1), "SHAPE"),
    (dict(T=1 << 31), "SHAPE"), (dict(heads=0), "SHAPE"), (dict(hd=63), "SHAPE"), (dict(hd=1026), "SHAPE"),
    (dict(T=1 << 29, heads=4), "SHAPE"), (dict(xr=-1), "SHAPE"), (dict(yh=-64), "SHAPE"), (dict(rope=rope(rot_dim=66)), "SHAPE"),
    (dict(rope=rope(rot_dim=3)), "SHAPE"), (dict(rope=rope(rot_dim=-2)), "SHAPE"), (dict(rope=rope(layout=2)), "RANGE"),
    (dict(x=FAKE + 2), "ALIGN"), (dict(dt=F16, y=FAKE + 1), "ALIGN"), (dict(pos=FAKE + 2), "ALIGN"),
    (dict(rope=rope(inv_freq=FAKE + 1)), "ALIGN")])
def test_rope_rotate_refuses(bad, code):
    a = {**ROTATE, **bad}
    args = [a["x"], a["xr"], a["xh"], a["y"], a["yr"], a["yh"], a["dt"], a["T"], a["heads"], a["hd"], a["pos"],
            None if a["rope"] is None else C.byref(a["rope"]), a["inv"], a["st"]]
    assert LIB.raw("rope_rotate")(*args) == ERR[code]


def test_nothing_to_do_is_no_error():
    assert LIB.raw("rope_rotate")(FAKE, 64, 64, FAKE, 64, 64, F32, 0, 1, 64, FAKE, C.byref(rope()), 0, None) == 0
    assert append(T=0) == 0 and attend(T=0) == 0


def append(kv=None, k=FAKE, v=FAKE, dt=F16, T=6, r=rope(), q=FAKE, qo=FAKE, n_q=4, strides=(256,) * 8):
    s = strides
    return LIB.raw("paged_kv_append")(C.byref(kv or paged()), k, s[0], s[1], v, s[2], s[3], dt, T,
                                      None if r is None else C.byref(r), q, s[4], s[5], qo, s[6], s[7], n_q, None)


@pytest.mark.parametrize("bad,code", [
    (dict(k=None), "NULL"), (dict(v=None), "NULL"), (dict(qo=None), "NULL"), (dict(kv=paged(k_cache=None)), "NULL"),
    (dict(kv=paged(page_table=None)), "NULL"), (dict(kv=paged(seq_lens=None)), "NULL"), (dict(dt=BF16), "DTYPE"),
    (dict(kv=paged(dtype=BF16)), "DTYPE"), (dict(kv=paged(dtype=BF16), dt=F32), "DTYPE"), (dict(kv=paged(dtype=F32), dt=F32), "DTYPE"),
    (dict(T=7), "SHAPE"), (dict(T=-3), "SHAPE"), (dict(kv=paged(batch=0)), "SHAPE"), (dict(kv=paged(page_size=0)), "SHAPE"),
    (dict(kv=paged(num_pages=0)), "SHAPE"), (dict(kv=paged(num_pages=1 << 28)), "SHAPE"), (dict(kv=paged(table_stride=3)), "SHAPE"),
    (dict(kv=paged(head_dim=63)), "SHAPE"), (dict(kv=paged(max_pages=0)), "SHAPE"), (dict(n_q=0), "SHAPE"),
    (dict(q=None, n_q=4), "SHAPE"), (dict(strides=(256, -1) + (256,) * 6), "SHAPE"), (dict(r=rope(rot_dim=128)), "SHAPE"),
    (dict(kv=paged(cu_q=FAKE + 2)), "ALIGN"), (dict(k=FAKE + 1), "ALIGN"), (dict(kv=paged(v_cache=FAKE + 1)), "ALIGN")])
def test_paged_kv_append_refuses(bad, code):
    assert append(**bad) == ERR[code]


def attend(kv=None, q=FAKE, row=256, head=64, out=FAKE, dt=F16, T=6, n_q=4, L=64, sp=FAKE, shared=16, scale=0.1, ws=FAKE,
           nbytes=1 << 40):
    return LIB.raw("paged_attn")(C.byref(kv or paged()), q, row, head, out, dt, T, n_q, L, sp, shared, scale, ws, nbytes, None)


@pytest.mark.parametrize("bad,code", [
    (dict(q=None), "NULL"), (dict(out=None), "NULL"), (dict(sp=None), "NULL"), (dict(kv=paged(v_cache=None)), "NULL"),
    (dict(dt=BF16), "DTYPE"), (dict(dt=7), "DTYPE"), (dict(n_q=5), "SHAPE"), (dict(n_q=0), "SHAPE"), (dict(L=0), "SHAPE"),
    (dict(shared=65), "SHAPE"), (dict(shared=-1), "SHAPE"), (dict(T=4), "SHAPE"), (dict(row=252), "SHAPE"), (dict(head=-64), "SHAPE"),
    (dict(kv=paged(head_dim=96)), "UNSUPPORTED"), (dict(n_q=130), "UNSUPPORTED"), (dict(scale=math.inf), "RANGE"),
    (dict(scale=math.nan), "RANGE"), (dict(kv=paged(num_pages=1), shared=33), "RANGE"), (dict(q=FAKE + 8), "ALIGN"),
    (dict(out=FAKE + 8), "ALIGN"), (dict(kv=paged(k_cache=FAKE + 8)), "ALIGN"), (dict(sp=FAKE + 1), "ALIGN"),
    (dict(L=(1 << 30) + 1), "RANGE")])
def test_paged_attn_refuses(bad, code):
    assert attend(**bad) == ERR[code]


@pytest.mark.parametrize("bad,code", [(dict(ws=FAKE + 8), "ALIGN"), (dict(ws=None), "WORKSPACE"), (dict(nbytes=64), "WORKSPACE")])
@pytest.mark.parametrize("shared", [0, 1024])
def test_paged_attn_refuses_a_workspace(bad, code, shared):
    """Where a row has several ranges of keys (one range writes the result itself and needs none)."""
    big = dict(kv=paged(num_pages=1000, max_pages=256, table_stride=256), L=4096, shared=shared)
    assert attend(**big, **bad) == ERR[code]
    b = C.c_size_t(0)
    assert LIB.raw("paged_attn_workspace_bytes")(6, 4, 2, 64, 3, 4096, shared, C.byref(b)) == 0 and b.value > 64
    assert attend(**big, nbytes=64) == ERR["WORKSPACE"]


@pytest.mark.parametrize("T,n_q,n_kv,code", [(1, 1 << 20, 1 << 20, "SHAPE"), (1, (1 << 20) - 1, (1 << 20) - 1, None),
                                             ((1 << 31) - 128, 1, 1, "SHAPE"), ((1 << 31) - 129, 1, 1, None), (1 << 26, 64, 1, "SHAPE")])
def test_paged_attn_limits_of_rows_and_heads(T, n_q, n_kv, code):
    b = C.c_size_t(0)
    assert LIB.raw("paged_attn_workspace_bytes")(T, n_q, n_kv, 128, 1, 256, 0, C.byref(b)) == (ERR[code] if code else 0)


def test_paged_attn_short_keys_need_no_workspace():
    """One range writes the result itself: up to 256 keys, up to 512 where the batch has 64 tiles of rows and heads."""
    need = LIB.raw("paged_attn_workspace_bytes")
    for batch, n_kv, L, some in ((1, 8, 256, False), (1, 8, 257, True), (7, 8, 512, True), (8, 8, 512, False), (8, 8, 513, True)):
        b = C.c_size_t(0)
        assert need(batch, 4 * n_kv, n_kv, 128, batch, L, 0, C.byref(b)) == 0 and (b.value > 0) == some, (batch, L)


def test_paged_attn_shared_keys_alone_need_a_workspace():
    """Where no key is a sequence's own (L == shared_len) and there are tiles enough for one range of the shared keys."""
    for batch in (2, 40, 640, 2000):
        b = C.c_size_t(0)
        assert LIB.raw("paged_attn_workspace_bytes")(batch, 32, 8, 128, batch, 512, 512, C.byref(b)) == 0
        assert b.value >= batch * 32 * (128 + 2) * 4, batch


def verify(tok=FAKE, draft=FAKE, target=FAKE, u=FAKE, nd=None, B=2, K=3, V=100, out=FAKE, acc=FAKE, ws=FAKE, nbytes=1 << 20,
           strides=(3, 300, 100, 400, 100, 4)):
    s = strides
    return LIB.raw("spec_verify")(tok, s[0], draft, s[1], s[2], target, s[3], s[4], u, s[5], nd, B, K, V, out, acc, ws, nbytes, None)


@pytest.mark.parametrize("bad,code", [
    (dict(tok=None), "NULL"), (dict(target=None), "NULL"), (dict(u=None), "NULL"), (dict(out=None), "NULL"),
    (dict(acc=None), "NULL"), (dict(ws=None), "NULL"), (dict(B=0), "SHAPE"), (dict(K=-1), "SHAPE"), (dict(V=0), "SHAPE"),
    (dict(V=(1 << 31) - 1), "SHAPE"), (dict(B=1 << 30, V=5000), "SHAPE"), (dict(strides=(3, -1, 100, 400, 100, 4)), "SHAPE"),
    (dict(nbytes=16), "WORKSPACE"), (dict(u=FAKE + 2), "ALIGN"), (dict(ws=FAKE + 8), "ALIGN"), (dict(nd=FAKE + 1), "ALIGN")])
def test_spec_verify_refuses(bad, code):
    assert verify(**bad) == ERR[code]


def test_workspace_queries():
    b = C.c_size_t(0)
    q = LIB.raw("paged_attn_workspace_bytes")
    assert q(4, 8, 2, 64, 4, 100, 0, C.byref(b)) == 0 and b.value >= 0
    assert q(4, 8, 2, 64, 4, 4000, 2000, C.byref(b)) == 0 and b.value > 0
    assert q(4, 8, 3, 64, 4, 100, 0, C.byref(b)) == ERR["SHAPE"] and q(4, 8, 2, 80, 4, 100, 0, C.byref(b)) == ERR["UNSUPPORTED"]
    assert q(4, 8, 2, 64, 4, 100, 0, None) == ERR["NULL"]
    v = LIB.raw("spec_verify_workspace_bytes")
    assert v(3, 2, 5000, C.byref(b)) == 0 and b.value > 0 and v(0, 2, 5000, C.byref(b)) == ERR["SHAPE"]


def caches(dt=torch.float16, n_kv=2, hd=64):
    return torch.zeros(5, 16, n_kv, hd, dtype=dt), torch.zeros(5, 16, n_kv, hd, dtype=dt)


TABLE, LENS = torch.zeros(3, 4, dtype=torch.int32), torch.ones(3, dtype=torch.int32)
ROPE = Rope(torch.ones(32))


def test_wrappers_refuse_on_the_host():
    """Wrong types, shapes, layouts and devices raise ValueError; valid CPU operands get as far as the device check."""
    x = torch.zeros(3, 2, 64)
    pos = torch.zeros(3, dtype=torch.int32)
    k, v = caches()
    ok = dict(k=x, v=x, k_cache=k, v_cache=v, page_table=TABLE, seq_lens=LENS, rope=ROPE, q=x)
    for bad in (dict(x=x.double()), dict(x=x[0]), dict(positions=pos.long()), dict(positions=pos[:2]),
                dict(rope=Rope(torch.ones(33))), dict(rope=Rope(torch.ones(32).double())), dict(x=x.transpose(1, 2)),
                dict(out=torch.zeros(3, 2, 32)), dict(out=torch.zeros(3, 2, 64).half())):
        with pytest.raises(ValueError):
            ops.rope_rotate(**{**dict(x=x, positions=pos, rope=ROPE), **bad})
    with pytest.raises(ValueError, match="ROCm device"):
        ops.rope_rotate(x, pos, ROPE)
    for bad in (dict(k=x.bfloat16()), dict(v=x.half()), dict(k_cache=k.float()), dict(v_cache=v[:3]), dict(k=x[:, :1]),
                dict(page_table=TABLE.long()), dict(page_table=TABLE[:, ::2]), dict(seq_lens=LENS[:2]), dict(seq_lens=LENS.float()),
                dict(cu_q=LENS), dict(k=x[:2], v=x[:2], q=x[:2]), dict(q=x.half()), dict(q_out=x.half()), dict(q=None, q_out=x),
                dict(rope=Rope(torch.ones(40))), dict(k_cache=k.transpose(1, 2))):
        with pytest.raises(ValueError):
            ops.paged_kv_append(**{**ok, **bad})
    with pytest.raises(ValueError, match="ROCm device"):
        ops.paged_kv_append(**ok)
    at = dict(q=x, k_cache=k, v_cache=v, page_table=TABLE, seq_lens=LENS, scale=0.1)
    for bad in (dict(q=x.bfloat16()), dict(q=x[:, :, :32]), dict(q=x.long()), dict(shared_len=5), dict(shared_len=-1),
                dict(shared_len=17, shared_pages=torch.zeros(1, dtype=torch.int32)), dict(shared_len=5, shared_pages=torch.zeros(1)),
                dict(out=torch.zeros(3, 64)), dict(workspace=torch.zeros(9)), dict(cu_q=torch.zeros(3, dtype=torch.int32))):
        with pytest.raises(ValueError):
            ops.paged_attn(**{**at, **bad})
    with pytest.raises(ValueError, match="ROCm device"):
        ops.paged_attn(**at)
    tok, p = torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, 4, 50)
    sv = dict(tokens=tok, draft_probs=p[:, :3], target_probs=p, uniforms=torch.zeros(2, 4))
    for bad in (dict(tokens=tok.long()), dict(tokens=tok[0]), dict(draft_probs=p), dict(target_probs=p[:, :3]), dict(target_probs=p.half()),
                dict(uniforms=torch.zeros(2, 3)), dict(n_draft=LENS), dict(target_probs=p.transpose(1, 2).contiguous().transpose(1, 2)),
                dict(workspace=torch.zeros(3))):
        with pytest.raises(ValueError):
            ops.spec_verify(**{**sv, **bad})
    with pytest.raises(ValueError, match="ROCm device"):
        ops.spec_verify(**sv)


CFG = dict(hidden_size=512, num_attention_heads=8, head_dim=64, max_position_embeddings=4096)


@pytest.mark.parametrize("scaling", [
    None, {"rope_type": "linear", "factor": 4.0}, {"rope_type": "dynamic", "factor": 2.0},
    {"rope_type": "yarn", "factor": 8.0, "original_max_position_embeddings": 4096},
    {"rope_type": "yarn", "factor": 16.0, "beta_fast": 16, "beta_slow": 2, "attention_factor": 1.3,
     "original_max_position_embeddings": 2048},
    {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
     "original_max_position_embeddings": 1024}])
@pytest.mark.parametrize("theta", [10000.0, 500000.0])
def test_rope_params_match_transformers(scaling, theta):
    """Run against transformers' functions where it is installed."""
    pytest.importorskip("transformers")
    from transformers import LlamaConfig
    from transformers.modeling_rope_utils import ROPE_INIT_FUNCTIONS
    cfg = {**CFG, "rope_theta": theta}
    if scaling:
        cfg["rope_scaling"] = scaling
    kind = scaling["rope_type"] if scaling else "default"
    seq = 10000 if kind == "dynamic" else None
    got = rope_params(cfg, seq_len=seq, interleaved=True)
    assert got.interleaved and got.inv_freq.dtype == torch.float32
    if kind == "default":
        assert torch.equal(got.inv_freq, inv_freq(cfg)) and got.mscale == 1.0
        return
    try:
        c = LlamaConfig(**{**cfg, "rope_parameters": {**(scaling or {}), "rope_theta": theta}})
        want, factor = ROPE_INIT_FUNCTIONS[kind](c, "cpu", seq_len=seq)
    except (KeyError, TypeError, AttributeError):
        c = LlamaConfig(**cfg)
        want, factor = ROPE_INIT_FUNCTIONS[kind](c, "cpu", seq_len=seq)
    # a few fp32 roundings in another order
    assert ((got.inv_freq - want).abs() <= 16 * 2.0 ** -24 * want.abs()).all()
    assert abs(got.mscale - factor) <= 1e-6


def test_rope_params_part_of_a_head_and_unknown_types():
    r = rope_params({**CFG, "partial_rotary_factor": 0.5})
    assert r.inv_freq.numel() == 16 and r.inv_freq[0] == 1.0
    with pytest.raises(NotImplementedError):
        rope_params({**CFG, "rope_scaling": {"rope_type": "other", "factor": 2.0}})
    with pytest.raises(NotImplementedError):
        inv_freq({**CFG, "rope_scaling": {"rope_type": "yarn", "factor": 2.0}})


@pytest.mark.parametrize("bad", [None, 1, "x", torch.zeros(2, 4, dtype=torch.int32), torch.zeros(0), object()])
def test_native_calls_leave_the_rest_to_python(bad):
    """Anything but plain device tensors of the documented types: None, nothing raised, nothing launched."""
    from q4llm._lib import native_calls
    mod = native_calls()
    x, pos, f, (k, v) = torch.zeros(3, 2, 64), torch.zeros(3, dtype=torch.int32), torch.ones(32), caches()
    ok = [x, pos, f, False, 1.0, False, None]
    for i in range(7):
        assert mod.rope(*ok[:i], bad, *ok[i + 1:]) is None
    ok = [x, x, k, v, TABLE, LENS, None, f, False, 1.0, x, None]
    for i in range(12):
        assert mod.append(*ok[:i], bad, *ok[i + 1:]) is None
    ok = [x, k, v, TABLE, LENS, 0.1, None, None, 0, None, None, None]
    for i in range(12):
        assert mod.paged(*ok[:i], bad, *ok[i + 1:]) is None
    ok = [pos.view(1, 3), None, torch.zeros(1, 4, 9), torch.zeros(1, 4), None, None]
    for i in range(6):
        assert mod.verify(*ok[:i], bad, *ok[i + 1:]) is None
    assert mod.rope() is None and mod.append(x) is None and mod.paged() is None and mod.verify() is None
