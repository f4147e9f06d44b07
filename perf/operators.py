"""Operators of batched serving over a paged KV cache: cases, inputs and plain forms.

The four operators are those that a server of several sequences calls in one step: rotary positions
(rope), the write of new keys and values into the pages (append), attention over the pages with a
prefix that the batch shares (attn), and the check of drafted tokens (verify). `run` computes them in
plain torch, or, where `own` is set, through this package's entry points.
"""

import math
import pathlib
import sys

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
CACHE = {"f32": torch.float16, "f16": torch.float16, "bf16": torch.bfloat16}  # activations -> cache


# ------------------------------------------------------------------------------------------------
# Cases
# ------------------------------------------------------------------------------------------------


def listed():
    return [
        # the q and k heads of a decode step of eight sequences, the 3B shape of this package (fp32 activations)
        dict(name="rope_step", op="rope", dtype="f32", tokens=8, heads=32, hd=128, rot=128, interleaved=False,
             mscale=1.0, far=131072),
        # a long prompt in one pass: part of each head rotated, in pairs, with a long-context factor on the tables
        dict(name="rope_prompt", op="rope", dtype="bf16", tokens=8192, heads=40, hd=128, rot=64, interleaved=True,
             mscale=1.2079, far=1 << 20),
        # decode step of 32 sequences: one token each, from the fused qkv row of the 3B shape
        dict(name="append_step", op="append", dtype="f32", batch=32, rows=1, ragged=False, n_q=24, n_kv=8, hd=128,
             page=16, past=4000, rot=128, interleaved=False),
        # prompts of sixteen sequences of different lengths, packed behind each other
        dict(name="append_prompt", op="append", dtype="bf16", batch=16, rows=1023, ragged=True, n_q=32, n_kv=8, hd=128,
             page=64, past=2000, rot=128, interleaved=False),
        # one sequence alone, nothing shared: the latency of a decode step
        dict(name="attn_one", op="attn", dtype="f32", batch=1, rows=1, ragged=False, n_q=24, n_kv=8, hd=128, page=16,
             shared=0, own_lo=700, own_hi=700),
        # chat behind one system prompt: every sequence has its own few hundred keys
        dict(name="attn_step", op="attn", dtype="f16", batch=32, rows=1, ragged=False, n_q=32, n_kv=8, hd=128, page=16,
             shared=2048, own_lo=40, own_hi=500),
        # many questions about one long document (fp32 queries, as this package's projections give them)
        dict(name="attn_long", op="attn", dtype="f32", batch=64, rows=1, ragged=False, n_q=24, n_kv=8, hd=128, page=32,
             shared=16384, own_lo=200, own_hi=1000),
        # the target's pass over four drafted tokens and the last accepted one
        dict(name="attn_check", op="attn", dtype="bf16", batch=48, rows=5, ragged=False, n_q=32, n_kv=8, hd=128, page=16,
             shared=4096, own_lo=100, own_hi=900),
        # long sequences of their own and nothing shared, one KV head per query head
        dict(name="attn_own", op="attn", dtype="f16", batch=8, rows=1, ragged=False, n_q=16, n_kv=16, hd=64, page=16,
             shared=0, own_lo=1000, own_hi=6000),
        # prompts of different lengths behind one prefix
        dict(name="attn_prompt", op="attn", dtype="bf16", batch=8, rows=511, ragged=True, n_q=32, n_kv=8, hd=128, page=64,
             shared=4096, own_lo=511, own_hi=511),
        # four drafted tokens of one sequence
        dict(name="verify_one", op="verify", batch=1, drafts=4, vocab=32000, given=True),
        # a batch with the vocabulary of the 3B shape
        dict(name="verify_batch", op="verify", batch=64, drafts=6, vocab=128256, given=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    most = {}
    for c in listed():
        w = work(c)
        most[c["op"]] = [max(a, b) for a, b in zip(most.get(c["op"], (0, 0)), (w["bytes"], w["flops"]))]
    op = rng.choice(["rope", "append", "attn", "attn", "verify"])
    while True:
        dtype = rng.choice(["f32", "f16", "bf16"])
        hd = rng.choice([64, 128])
        n_kv = rng.choice([1, 2, 4, 5, 8, 16])
        n_q = n_kv * rng.choice([1, 2, 3, 4, 6, 8])
        page = rng.choice([8, 16, 24, 32, 64, 128])
        if op == "rope":
            hd = rng.choice([32, 64, 80, 128, 256])
            c = dict(op=op, dtype=dtype, tokens=_log(rng, 1, 16384), heads=rng.randint(1, 48), hd=hd,
                     rot=rng.choice([hd, hd, hd // 2, hd // 4 * 2 - 2]), interleaved=rng.random() < 0.5,
                     mscale=rng.choice([1.0, round(rng.uniform(1.0, 1.5), 4)]), far=_log(rng, 100, 1 << 24))
        elif op == "append":
            c = dict(op=op, dtype=dtype, batch=_log(rng, 1, 128), rows=rng.choice([1, 1, _log(rng, 2, 1500)]),
                     ragged=rng.random() < 0.5, n_q=n_q, n_kv=n_kv, hd=hd, page=page, past=_log(rng, 1, 6000),
                     rot=rng.choice([hd, hd // 2]), interleaved=rng.random() < 0.5)
        elif op == "attn":
            rows = rng.choice([1, 1, 1, rng.randint(2, 9), _log(rng, 10, 600)])
            lo = _log(rng, rows, 2000)
            c = dict(op=op, dtype=dtype, batch=_log(rng, 1, 96), rows=rows, ragged=rng.random() < 0.5, n_q=n_q, n_kv=n_kv,
                     hd=hd, page=page, shared=rng.choice([0, _log(rng, 1, 20000), _log(rng, 1, 20000)]), own_lo=lo,
                     own_hi=_log(rng, lo, 8000))
        else:
            c = dict(op=op, batch=_log(rng, 1, 96), drafts=rng.randint(1, 10), vocab=_log(rng, 1000, 160000),
                     given=rng.random() < 0.75)
        w = work(c)
        if w["bytes"] <= most[op][0] and w["flops"] <= most[op][1] and _plain_bytes(c) < 12e9:
            return c


def _plain_bytes(c):
    """About what the plain form holds at once."""
    if c["op"] != "attn":
        return 0
    keys = c["shared"] + c["own_hi"]
    return c["batch"] * keys * 4 * (c["rows"] * c["n_q"] * 3 + 4 * c["n_kv"] * c["hd"])


def _spread(lo, hi, n):
    """n whole numbers evenly from hi down to lo (hi alone for n == 1)."""
    return [hi - (hi - lo) * i // max(n - 1, 1) for i in range(n)]


def _rows(c):
    """New tokens of each sequence."""
    return _spread(1, c["rows"], c["batch"]) if c["ragged"] else [c["rows"]] * c["batch"]


def _own(c):
    """Keys of each sequence behind the shared ones, its new tokens' included."""
    return [max(k, r) for k, r in zip(_spread(c["own_lo"], c["own_hi"], c["batch"]), _rows(c))]


def work(c):
    if c["op"] == "rope":
        n = c["tokens"] * c["heads"] * c["hd"]
        b = 2 * n * TYPES[c["dtype"]].itemsize + 4 * c["tokens"] + 2 * c["rot"]
        return dict(bytes=b, flops=3 * c["tokens"] * c["heads"] * c["rot"])
    if c["op"] == "append":
        t = sum(_rows(c))
        a, k = TYPES[c["dtype"]].itemsize, CACHE[c["dtype"]].itemsize
        b = t * c["hd"] * (2 * a * c["n_q"] + 2 * (a + k) * c["n_kv"])
        return dict(bytes=b, flops=3 * t * (c["n_q"] + c["n_kv"]) * c["rot"])
    if c["op"] == "attn":
        rows, keys = _rows(c), _own(c)
        row = c["n_kv"] * c["hd"] * CACHE[c["dtype"]].itemsize
        b = 2 * row * (c["shared"] + sum(keys)) + 2 * sum(rows) * c["n_q"] * c["hd"] * TYPES[c["dtype"]].itemsize
        seen = sum(r * (c["shared"] + k) - r * (r - 1) // 2 for r, k in zip(rows, keys))
        return dict(bytes=b, flops=4 * c["n_q"] * c["hd"] * seen)
    v = c["batch"] * c["vocab"]
    return dict(bytes=4 * v * (2 if c["given"] else 1), flops=4 * v)


# ------------------------------------------------------------------------------------------------
# Inputs
# ------------------------------------------------------------------------------------------------


def _inv_freq(rot):
    return (500000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot)).float()


def _cuts(rows):
    return torch.tensor(np.concatenate([[0], np.cumsum(rows)]), dtype=torch.int32, device="cuda")


def _paged(c, g, n, rng, shared, lens):
    """Caches, page table, lengths and shared page list of sequences of `lens` keys, the first `shared` of which
    are in pages that all of them hold."""
    page, dt = c["page"], CACHE[c["dtype"]]
    top = max(lens)
    most = -(-top // page)
    sp = -(-shared // page)
    need = [-(-k // page) - shared // page for k in lens]
    total = sp + sum(max(x, 0) for x in need) + 3
    order = rng.permutation(total).astype(np.int32)
    col, first = np.arange(most), shared // page
    at = sp + np.cumsum([0] + need[:-1])[:, None] - first  # a sequence's own pages follow those of the one before
    held = (col >= first) & (col < first + np.array(need)[:, None])
    table = np.where(held, order[np.where(held, at + col, 0)], np.where(col < first, order[np.minimum(col, sp)], 0))
    shape = (total, page, c["n_kv"], c["hd"])
    kc = torch.randn(shape, generator=g, device="cuda").to(dt)
    vc = torch.randn(shape, generator=g, device="cuda").to(dt)
    i32 = dict(dtype=torch.int32, device="cuda")
    return (kc, vc, torch.tensor(table, **i32), torch.tensor(lens, **i32), torch.tensor(order[:sp], **i32))


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    rng = np.random.RandomState(seed % (1 << 32))
    s = dict(case=c)
    if c["op"] == "rope":
        s["x"] = torch.randn(c["tokens"], c["heads"], c["hd"], generator=g, device="cuda").to(TYPES[c["dtype"]])
        s["pos"] = torch.randint(0, c["far"], (c["tokens"],), generator=g, device="cuda").int()
        s["inv_freq"] = _inv_freq(c["rot"])
    elif c["op"] in ("append", "attn"):
        n = c["batch"]
        order = rng.permutation(n)
        rows = [_rows(c)[i] for i in order]
        t = sum(rows)
        s["rows"], s["most"] = rows, max(rows)
        s["cu_q"] = _cuts(rows) if c["ragged"] else None
        if c["op"] == "append":
            past = _spread(0, c["past"], n)[::-1]  # keys that a sequence holds already
            kc, vc, table, lens, _ = _paged(c, g, n, rng, 0, [past[i] + _rows(c)[i] for i in order])
            # the rows of a fused q | k | v projection
            qkv = torch.randn(t, (c["n_q"] + 2 * c["n_kv"]) * c["hd"], generator=g, device="cuda").to(TYPES[c["dtype"]])
            q, k, v = (x.unflatten(1, (-1, c["hd"])) for x in
                       qkv.split([c["n_q"] * c["hd"], c["n_kv"] * c["hd"], c["n_kv"] * c["hd"]], 1))
            s.update(q=q, k=k, v=v, inv_freq=_inv_freq(c["rot"]))
        else:
            keys = [c["shared"] + _own(c)[i] for i in order]
            kc, vc, table, lens, sp = _paged(c, g, n, rng, c["shared"], keys)
            s["shared_pages"] = sp if c["shared"] else None
            s["q"] = torch.randn(t, c["n_q"], c["hd"], generator=g, device="cuda").to(TYPES[c["dtype"]])
            s["top"] = max(keys)
        s.update(kc=kc, vc=vc, table=table, lens=lens)
    else:
        b, k, v = c["batch"], c["drafts"], c["vocab"]
        z = torch.randn(b, k + 1, v, generator=g, device="cuda") * 2.5
        s["target"] = torch.softmax(z, -1)
        # a smaller model: its scores are near the target's
        z = z[:, :k] + 0.7 * torch.randn(b, k, v, generator=g, device="cuda")
        d = torch.softmax(z, -1)
        noise = torch.rand(b, k, v, generator=g, device="cuda")
        s["tokens"] = (d / -torch.log(noise.clamp(1e-12, 1 - 1e-7))).argmax(-1).int()  # a sample of each row
        s["draft"] = d if c["given"] else None
        s["uniforms"] = torch.rand(b, k + 1, generator=g, device="cuda")
        s["n_draft"] = torch.tensor(rng.randint(max(0, k - 2), k + 1, b), dtype=torch.int32, device="cuda")
    return s


# ------------------------------------------------------------------------------------------------
# One pass
# ------------------------------------------------------------------------------------------------


def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(s):
    package = str(pathlib.Path(__file__).resolve().parent.parent / "iree-adreno-genai-tuner_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    from q4llm import ops
    from q4llm.rope import Rope
    c = s["case"]
    if c["op"] == "rope":
        return ops.rope_rotate(s["x"], s["pos"], Rope(s["inv_freq"], c["interleaved"], c["mscale"]))
    if c["op"] == "append":
        q = ops.paged_kv_append(s["k"], s["v"], s["kc"], s["vc"], s["table"], s["lens"], cu_q=s["cu_q"],
                                rope=Rope(s["inv_freq"], c["interleaved"]), q=s["q"])
        return q, s["kc"], s["vc"]
    if c["op"] == "attn":
        return ops.paged_attn(s["q"], s["kc"], s["vc"], s["table"], s["lens"], c["hd"] ** -0.5, cu_q=s["cu_q"],
                              shared_pages=s["shared_pages"], shared_len=c["shared"])
    return ops.spec_verify(s["tokens"], s["draft"], s["target"], s["uniforms"], n_draft=s["n_draft"])


def _run_plain(s):
    op = s["case"]["op"]
    return {"rope": _plain_rope, "append": _plain_append, "attn": _plain_attn, "verify": _plain_verify}[op](s)


def _rotate(x, pos, inv_freq, interleaved, mscale):
    """x [T, heads, hd] at positions pos [T], in 32 bits with the angles in 64."""
    t = pos.double()[:, None] * inv_freq.double()
    cos = (torch.cos(t) * mscale).float()[:, None]
    sin = (torch.sin(t) * mscale).float()[:, None]
    x = x.float()
    h = inv_freq.numel()
    if interleaved:
        a, b = x[..., 0:2 * h:2], x[..., 1:2 * h:2]
        r = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = x[..., :h], x[..., h:2 * h]
        r = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([r, x[..., 2 * h:]], -1)


def _plain_rope(s):
    c = s["case"]
    return _rotate(s["x"], s["pos"], s["inv_freq"], c["interleaved"], c["mscale"]).to(s["x"].dtype)


def _tokens(s):
    """(sequence, position) of each new token."""
    n, lens = s["lens"].numel(), s["lens"].long()
    t = torch.arange(s["q"].shape[0], device="cuda")
    if s["cu_q"] is None:
        r = s["most"]
        b = t // r
        return b, lens[b] - r + t % r
    cu = s["cu_q"].long()
    b = (t[:, None] >= cu[None, 1:n]).sum(1)
    return b, lens[b] - (cu[b + 1] - cu[b]) + (t - cu[b])


def _plain_append(s):
    c = s["case"]
    b, pos = _tokens(s)
    page = s["kc"].shape[1]
    slot = s["table"].long()[b, pos // page] * page + pos % page
    k = _rotate(s["k"], pos, s["inv_freq"], c["interleaved"], 1.0)
    s["kc"].flatten(0, 1)[slot] = k.to(s["kc"].dtype)
    s["vc"].flatten(0, 1)[slot] = s["v"].to(s["vc"].dtype)
    q = _rotate(s["q"], pos, s["inv_freq"], c["interleaved"], 1.0).to(s["q"].dtype)
    return q, s["kc"], s["vc"]


def _plain_attn(s):
    c = s["case"]
    q, page, n, most = s["q"], c["page"], c["batch"], s["most"]
    n_kv, hd, g = c["n_kv"], c["hd"], c["n_q"] // c["n_kv"]
    j = torch.arange(s["top"], device="cuda")
    held = s["table"].long()[:, j // page]
    if c["shared"]:
        first = s["shared_pages"].long()[(j // page).clamp(max=s["shared_pages"].numel() - 1)]
        held = torch.where(j < c["shared"], first, held)
    slot = held * page + j % page  # [n, keys]
    k = s["kc"].flatten(0, 1)[slot].float().permute(0, 2, 3, 1).contiguous()  # [n, n_kv, hd, keys]
    v = s["vc"].flatten(0, 1)[slot].float().permute(0, 2, 1, 3).contiguous()  # [n, n_kv, keys, hd]
    lens = s["lens"].long()
    i = torch.arange(most, device="cuda")
    if s["cu_q"] is None:
        at, count = torch.arange(n, device="cuda") * most, torch.full((n,), most, device="cuda")
    else:
        cu = s["cu_q"].long()
        at, count = cu[:-1], cu[1:] - cu[:-1]
    row = (at[:, None] + i).clamp(max=q.shape[0] - 1)  # [n, most], those past a sequence's count unused
    pos = (lens - count)[:, None] + i
    x = q[row].float().unflatten(2, (n_kv, g)).permute(0, 2, 1, 3, 4).reshape(n, n_kv, most * g, hd).contiguous()
    p = (torch.matmul(x, k) * hd ** -0.5).unflatten(2, (most, g))
    seen = (j[None, None] <= pos[..., None]) & (i[None, :, None] < count[:, None, None])  # [n, most, keys]
    p = p.masked_fill(~seen[:, None, :, None], float("-inf"))
    p = torch.exp(p - p.amax(-1, keepdim=True).clamp(min=-3e38))
    p = (p / p.sum(-1, keepdim=True).clamp(min=1e-30)).flatten(2, 3)
    o = torch.matmul(p, v).unflatten(2, (most, g)).permute(0, 2, 1, 3, 4)  # [n, most, n_kv, g, hd]
    return o[i[None] < count[:, None]].reshape(q.shape[0], -1).to(q.dtype)


def _plain_verify(s):
    tokens, p, u = s["tokens"].long(), s["target"], s["uniforms"].double()
    b, k = tokens.shape
    i = torch.arange(k, device="cuda")
    px = p[:, :k].gather(2, tokens[..., None])[..., 0].double()
    qx = torch.ones_like(px) if s["draft"] is None else s["draft"].gather(2, tokens[..., None])[..., 0].double()
    good = (u[:, :k] * qx < px) & (i < s["n_draft"][:, None])
    count = good.long().cumprod(1).sum(1)
    rows = torch.arange(b, device="cuda")
    w = p[rows, count].double()
    refused = count < s["n_draft"]
    at = count.clamp(max=k - 1)
    if s["draft"] is None:
        left = w.scatter(1, tokens[rows, at][:, None], 0.0)
    else:
        left = (w - s["draft"][rows, at].double()).clamp(min=0)
    left = torch.where(refused[:, None], left, w)
    w = torch.where(left.sum(1, keepdim=True) > 0, left, w)
    c = w.cumsum(1)
    last = w.shape[1] - 1 - (w > 0).flip(1).int().argmax(1)
    new = torch.minimum((c <= u[:, k:] * c[:, -1:]).sum(1), last)
    j = torch.arange(k + 1, device="cuda")
    out = torch.cat([tokens, tokens[:, :1]], 1)
    out = torch.where(j < count[:, None], out, torch.where(j == count[:, None], new[:, None], -1))
    return out.int(), count.int()


# ------------------------------------------------------------------------------------------------
# The definition in 64 bits, sequence by sequence
# ------------------------------------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    c = case
    if c["op"] == "rope":
        return _exact_rotate(s["x"], s["pos"], s["inv_freq"], c["interleaved"], c["mscale"])
    if c["op"] == "append":
        kc, vc = s["kc"].double(), s["vc"].double()
        out, at = [], 0
        for b, r in enumerate(s["rows"]):
            end = int(s["lens"][b])
            pos = torch.arange(end - r, end, device="cuda")
            pages, off = s["table"][b].long()[pos // c["page"]], pos % c["page"]
            kc[pages, off] = _exact_rotate(s["k"][at:at + r], pos, s["inv_freq"], c["interleaved"], 1.0)
            vc[pages, off] = s["v"][at:at + r].double()
            out.append(_exact_rotate(s["q"][at:at + r], pos, s["inv_freq"], c["interleaved"], 1.0))
            at += r
        return torch.cat(out), kc, vc
    if c["op"] == "attn":
        g, out, at = c["n_q"] // c["n_kv"], [], 0
        sh, page = c["shared"], c["page"]
        for b, r in enumerate(s["rows"]):
            end = int(s["lens"][b])

            def keys(cache):
                parts = [cache[s["table"][b].long()].reshape(-1, c["n_kv"], c["hd"])[sh:end]]
                if sh:
                    parts.insert(0, cache[s["shared_pages"].long()].reshape(-1, c["n_kv"], c["hd"])[:sh])
                return torch.cat(parts).double()
            k, v = keys(s["kc"]), keys(s["vc"])
            o = torch.empty(r, c["n_q"], c["hd"], dtype=torch.float64, device="cuda")
            late = torch.arange(end, device="cuda")[None] > torch.arange(end - r, end, device="cuda")[:, None]
            for h in range(c["n_q"]):
                z = s["q"][at:at + r, h].double() @ k[:, h // g].t().contiguous() / math.sqrt(c["hd"])
                z[late] = -math.inf
                e = torch.exp(z - z.max(1, keepdim=True).values)
                o[:, h] = (e @ v[:, h // g].contiguous()) / e.sum(1, keepdim=True)
            out.append(o.reshape(r, -1))
            at += r
        return torch.cat(out)
    tokens, target = s["tokens"].tolist(), s["target"].cpu().numpy().astype(np.float64)
    draft = None if s["draft"] is None else s["draft"].cpu().numpy().astype(np.float64)
    u, n = s["uniforms"].cpu().numpy().astype(np.float64), s["n_draft"].tolist()
    out, counts = [], []
    for b in range(c["batch"]):
        a = 0
        while a < n[b] and u[b, a] * (1.0 if draft is None else draft[b, a, tokens[b][a]]) < target[b, a, tokens[b][a]]:
            a += 1
        w = target[b, a]
        if a < n[b]:
            q = np.eye(1, c["vocab"], tokens[b][a])[0] * 2 if draft is None else draft[b, a]
            left = np.maximum(w - q, 0)
            w = left if left.any() else w
        t = np.cumsum(w)
        new = min(int(np.searchsorted(t, u[b, -1] * t[-1], side="right")), int(np.flatnonzero(w)[-1]))
        out.append(tokens[b][:a] + [new] + [-1] * (c["drafts"] - a))
        counts.append(a)
    return torch.tensor(out, dtype=torch.int32), torch.tensor(counts, dtype=torch.int32)


def _exact_rotate(x, pos, inv_freq, interleaved, mscale):
    """The rotation as a product of complex numbers."""
    h = inv_freq.numel()
    z = torch.polar(torch.full((), mscale, dtype=torch.float64, device="cuda"),
                    pos.double()[:, None, None] * inv_freq.double())
    x = x.double()
    part = x[..., :2 * h]
    pairs = part.unflatten(-1, (h, 2)) if interleaved else part.unflatten(-1, (2, h)).transpose(-1, -2)
    y = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * z)
    y = y.flatten(-2) if interleaved else y.transpose(-1, -2).flatten(-2)
    return torch.cat([y, x[..., 2 * h:]], -1)
