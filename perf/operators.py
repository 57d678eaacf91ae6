"""Performance cases of the position and cache operators.

Each case is one call of an operator as a program makes it: the per-head query/key norm with the
position rotation between the QKV projection and attention (forward and backward, training layout),
the same written into a paged key/value cache (serving), and attention of new tokens over that cache.
``run`` computes a case with elementary torch operations in 32 bits, or, where ``own`` is set, with the
calls of ``beacon_b200.ops``.  ``exact`` computes the definition in 64 bits.
"""
import math

import numpy as np
import torch

own = False

_DT = {"bf16": torch.bfloat16, "f32": torch.float32}
_EPS = 1e-5
_THETA = 10000.0


# ---------------------------------------------------------------------------- cases

def listed():
    return [
        # The block of the benchmark: batch 4 x 2048, 32 heads of 128, between its QKV projection and attention.
        dict(name="rope_fwd_block", op="fwd", batch=4, seq=2048, heads=32, kv_heads=32, dim=128, rot=128,
             interleaved=False, dtype="bf16"),
        # The 4-head, 128-token, 32-bit parity configuration: the smallest call.
        dict(name="rope_fwd_f32_small", op="fwd", batch=1, seq=128, heads=4, kv_heads=4, dim=64, rot=64,
             interleaved=True, dtype="f32"),
        # Training backward at the attention benchmark's batch and length, grouped heads.
        dict(name="rope_bwd_train", op="bwd", batch=8, seq=4096, heads=32, kv_heads=8, dim=128, rot=128,
             interleaved=False, dtype="bf16"),
        # An odd length, half of each head rotated, 32-bit parity path.
        dict(name="rope_bwd_f32_odd", op="bwd", batch=3, seq=257, heads=6, kv_heads=2, dim=64, rot=32,
             interleaved=False, dtype="f32"),
        # One decode step of 64 sequences: their single new tokens go into the cache.
        dict(name="append_decode", op="append", seqs=64, q_min=1, q_max=1, kv_min=500, kv_max=4000, heads=32,
             kv_heads=8, dim=128, rot=128, interleaved=False, page=16, dtype="bf16"),
        # Prompts of uneven lengths entering an empty cache.
        dict(name="append_prompts", op="append", seqs=6, q_min=311, q_max=4096, kv_min=0, kv_max=0, heads=64,
             kv_heads=8, dim=128, rot=128, interleaved=False, page=64, dtype="bf16"),
        # One user's next token over a short context: latency.
        dict(name="decode_one", op="attention", seqs=1, q_min=1, q_max=1, kv_min=2047, kv_max=2047, heads=32,
             kv_heads=8, dim=128, page=16, dtype="bf16"),
        # A decode step of a busy server, contexts of very different lengths.
        dict(name="decode_batch", op="attention", seqs=64, q_min=1, q_max=1, kv_min=500, kv_max=8192, heads=32,
             kv_heads=8, dim=128, page=16, dtype="bf16"),
        # A few very long contexts, 64 query heads on 8 key/value heads.
        dict(name="decode_long", op="attention", seqs=4, q_min=1, q_max=1, kv_min=65537, kv_max=131071, heads=64,
             kv_heads=8, dim=128, page=64, dtype="bf16"),
        # A 2048-token chunk of a long prompt, the last of a 32768-token context.
        dict(name="chunk_long", op="attention", seqs=1, q_min=2048, q_max=2048, kv_min=30720, kv_max=30720, heads=64,
             kv_heads=8, dim=128, page=128, dtype="bf16"),
        # Prompt chunks and single tokens in one step.
        dict(name="chunk_mixed", op="attention", seqs=16, q_min=1, q_max=512, kv_min=100, kv_max=7500, heads=32,
             kv_heads=8, dim=128, page=16, dtype="bf16"),
        # The 32-bit parity path, a page size that divides no tile, ragged lengths.
        dict(name="attention_f32_ragged", op="attention", seqs=8, q_min=1, q_max=40, kv_min=33, kv_max=1500, heads=8,
             kv_heads=4, dim=64, page=24, dtype="f32"),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["fwd", "bwd", "append", "attention", "attention"])
    dtype = "f32" if rng.random() < 0.2 else "bf16"
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 6, 8])
    dim = rng.choice([64, 128])
    rot = rng.choice([dim, dim, dim // 2])
    inter = rng.random() < 0.5
    if op in ("fwd", "bwd"):
        batch = _log_int(rng, 1, 8)
        seq = _log_int(rng, 1, 4096)
        return dict(op=op, batch=batch, seq=seq, heads=heads, kv_heads=kv_heads, dim=dim, rot=rot, interleaved=inter,
                    dtype=dtype)
    page = rng.choice([8, 16, 24, 32, 64, 128, 256])
    kind = rng.choice(["decode", "decode", "chunk", "mixed"])
    if kind == "decode":
        seqs, q_min, q_max = _log_int(rng, 1, 96), 1, 1
        kv_max = _log_int(rng, 16, 524288 // seqs if op == "attention" else 4096)
    elif kind == "chunk":
        seqs = 1
        q_min = q_max = _log_int(rng, 2, 2048)
        kv_max = _log_int(rng, 1, 30720)
    else:
        seqs, q_min, q_max = rng.randint(2, 16), 1, _log_int(rng, 2, 512)
        kv_max = _log_int(rng, 16, 8192)
    if dtype == "f32":
        q_max = min(q_max, 64)
        q_min = min(q_min, q_max)
        kv_max = min(kv_max, 8192)
    if op == "append":
        kv_max = min(kv_max, 8192)
    kv_min = max(0, kv_max // rng.choice([1, 2, 16]))
    case = dict(op=op, seqs=seqs, q_min=q_min, q_max=q_max, kv_min=kv_min, kv_max=kv_max, heads=heads,
                kv_heads=kv_heads, dim=dim, page=page, dtype=dtype)
    if op == "append":
        case.update(rot=rot, interleaved=inter)
    return case


def _ladder(lo, hi, n, salt):
    """n whole numbers spread over [lo, hi] on a logarithmic scale, both ends among them, in a fixed mixed order."""
    if n == 1:
        return np.array([hi], dtype=np.int64)
    x = np.exp(np.linspace(math.log(max(lo, 1)), math.log(max(hi, 1)), n)).round().astype(np.int64)
    x = np.clip(x, lo, hi)
    x[0], x[-1] = lo, hi
    return x[np.random.RandomState(salt).permutation(n)]


def _lengths(case):
    """New tokens and total tokens (new ones included) of every sequence."""
    q = _ladder(case["q_min"], case["q_max"], case["seqs"], 7)
    before = _ladder(case["kv_min"], case["kv_max"], case["seqs"], 11)
    return q, q + before


# ---------------------------------------------------------------------------- inputs

def _randn(gen, *shape, scale=1.0, dtype=torch.float32):
    return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(dtype)


def _table(positions, rot):
    i = torch.arange(rot // 2, dtype=torch.float64, device="cuda")
    a = torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] * _THETA ** (-2.0 * i / rot)
    return torch.cat([a.cos(), a.sin()], dim=1).float()


def _paging(case, gen):
    q, kv = _lengths(case)
    page, n = case["page"], case["seqs"]
    width = int(-(-kv.max() // page))
    pool = int((-(-kv // page)).sum()) + 3  # a few pages that no sequence owns
    order = torch.randperm(pool, generator=gen, device="cuda").to(torch.int32)
    table = torch.zeros(n, width, dtype=torch.int32, device="cuda")
    at = 0
    for s in range(n):
        used = int(-(-kv[s] // page))
        table[s, :used] = order[at:at + used]
        at += used
    cu = np.concatenate([[0], np.cumsum(q)])
    return dict(page_table=table, pool=pool, max_q=int(q.max()), max_kv=int(kv.max()), tokens=int(q.sum()),
                cu_q=torch.tensor(cu, dtype=torch.int32, device="cuda"),
                kv_lens=torch.tensor(kv, dtype=torch.int32, device="cuda"))


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    st = dict(case)
    dt, H, K, D = _DT[case["dtype"]], case["heads"], case["kv_heads"], case["dim"]
    if case["op"] in ("append", "attention"):
        st.update(_paging(case, gen))
        shape = (st["pool"], K, case["page"], D)
        if case["op"] == "attention":
            st["q"] = _randn(gen, st["tokens"], H, D, scale=1.5, dtype=dt)
        st["k_cache"] = _randn(gen, *shape, dtype=dt)
        st["v_cache"] = _randn(gen, *shape, dtype=dt)
        tokens, positions = st["tokens"], st["max_kv"]
    else:
        tokens, positions = case["batch"] * case["seq"], case["seq"]
    if case["op"] != "attention":
        st["qkv"] = _randn(gen, tokens, (H + 2 * K) * D, scale=1.3, dtype=dt)
        st["q_gain"] = (1.0 + _randn(gen, D, scale=0.2)).to(dt)
        st["k_gain"] = (1.0 + _randn(gen, D, scale=0.2)).to(dt)
        st["table"] = _table(positions, case["rot"])
    if case["op"] == "bwd":
        B, S = case["batch"], case["seq"]
        st["dq"] = _randn(gen, B, H, S, D, dtype=dt)
        st["dk"] = _randn(gen, B, K, S, D, dtype=dt)
        st["dv"] = _randn(gen, B, K, S, D, dtype=dt)
    return st


# ---------------------------------------------------------------------------- plain form

def _pairs(x, rot, interleaved):
    """The two members of every rotated pair of x [..., D]."""
    if interleaved:
        return x[..., 0:rot:2], x[..., 1:rot:2]
    return x[..., :rot // 2], x[..., rot // 2:rot]


def _join(a, b, rest, interleaved):
    turned = torch.stack([a, b], dim=-1).flatten(-2) if interleaved else torch.cat([a, b], dim=-1)
    return torch.cat([turned, rest], dim=-1)


def _rotate(z, cos, sin, rot, interleaved):
    a, b = _pairs(z, rot, interleaved)
    return _join(a * cos - b * sin, b * cos + a * sin, z[..., rot:], interleaved)


def _norm_rope(x, gain, cos, sin, st):
    """x [T, heads, D] in 32 bits: per-head norm, gain, rotation."""
    z = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + _EPS) * gain.float()
    return _rotate(z, cos[:, None], sin[:, None], st["rot"], st["interleaved"])


def _split(st):
    H, K, D = st["heads"], st["kv_heads"], st["dim"]
    x = st["qkv"].float().view(-1, H + 2 * K, D)
    return x[:, :H], x[:, H:H + K], x[:, H + K:]


def _head_major(x, st):
    return x.view(st["batch"], st["seq"], -1, st["dim"]).transpose(1, 2).contiguous()


def _plain_fwd(st):
    dt, half = st["qkv"].dtype, st["rot"] // 2
    rows = st["table"].repeat(st["batch"], 1)
    cos, sin = rows[:, :half], rows[:, half:]
    q, k, v = _split(st)
    q, k = _norm_rope(q, st["q_gain"], cos, sin, st), _norm_rope(k, st["k_gain"], cos, sin, st)
    return dict(q=_head_major(q.to(dt), st), k=_head_major(k.to(dt), st), v=_head_major(v.to(dt).contiguous(), st))


def _plain_bwd_heads(dy, x, gain, cos, sin, st):
    """(dx, dgain) of one kind of heads; dy, x [T, heads, D] in 32 bits."""
    inv = torch.rsqrt(x.square().mean(-1, keepdim=True) + _EPS)
    dz = _rotate(dy, cos[:, None], -sin[:, None], st["rot"], st["interleaved"])
    xh = x * inv
    e = dz * gain.float()
    return inv * (e - xh * (e * xh).mean(-1, keepdim=True)), (dz * xh).sum((0, 1))


def _plain_bwd(st):
    dt, half, D = st["qkv"].dtype, st["rot"] // 2, st["dim"]
    rows = st["table"].repeat(st["batch"], 1)
    cos, sin = rows[:, :half], rows[:, half:]
    q, k, _ = _split(st)
    dq, dk, dv = (st[n].float().transpose(1, 2).flatten(0, 1) for n in ("dq", "dk", "dv"))
    gq, dgq = _plain_bwd_heads(dq, q, st["q_gain"], cos, sin, st)
    gk, dgk = _plain_bwd_heads(dk, k, st["k_gain"], cos, sin, st)
    return dict(dqkv=torch.cat([gq, gk, dv], dim=1).flatten(1).to(dt), dq_gain=dgq.to(dt), dk_gain=dgk.to(dt))


def _owners(st):
    """Sequence and place among its new tokens of every token."""
    t = torch.arange(st["tokens"], device="cuda", dtype=torch.int32)
    seq = torch.searchsorted(st["cu_q"], t, right=True) - 1
    return seq, (t - st["cu_q"][seq]).long()


def _plain_append(st):
    dt, half = st["qkv"].dtype, st["rot"] // 2
    seq, place = _owners(st)
    q_lens = (st["cu_q"][1:] - st["cu_q"][:-1])
    pos = (st["kv_lens"] - q_lens)[seq].long() + place
    rows = st["table"][pos]
    cos, sin = rows[:, :half], rows[:, half:]
    q, k, v = _split(st)
    page, slot = st["page_table"][seq, pos // st["page"]].long(), pos % st["page"]
    st["k_cache"][page, :, slot] = _norm_rope(k, st["k_gain"], cos, sin, st).to(dt)
    st["v_cache"][page, :, slot] = v.to(dt)
    return dict(q=_norm_rope(q, st["q_gain"], cos, sin, st).to(dt), k_cache=st["k_cache"], v_cache=st["v_cache"])


def _plain_attention(st):
    """Sequences padded to the longest chunk and the longest context."""
    H, K, D, N = st["heads"], st["kv_heads"], st["dim"], st["seqs"]
    g, maxq = H // K, st["max_q"]
    place = torch.arange(maxq, device="cuda")
    q_lens = (st["cu_q"][1:] - st["cu_q"][:-1]).long()
    kv = st["kv_lens"].long()
    rows = (st["cu_q"][:-1].long()[:, None] + place).clamp(max=st["tokens"] - 1)
    q = st["q"].float()[rows].view(N, maxq, K, g, D).permute(0, 2, 1, 3, 4).reshape(N, K, maxq * g, D)
    table = st["page_table"].long()
    k = st["k_cache"][table].float().transpose(1, 2).reshape(N, K, -1, D)
    v = st["v_cache"][table].float().transpose(1, 2).reshape(N, K, -1, D)
    s = (q @ k.transpose(-1, -2)).mul_(1.0 / math.sqrt(D))
    last = (kv - q_lens)[:, None] + place                      # the last key that each new token sees
    hidden = torch.arange(k.shape[2], device="cuda") > last[..., None]
    s.view(N, K, maxq, g, -1).masked_fill_(hidden[:, None, :, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    s.sub_(top).exp_()
    total = s.sum(-1, keepdim=True)
    o = (s @ v) / total
    lse = (top + total.log()).squeeze(-1)
    seq, place = _owners(st)
    o = o.view(N, K, maxq, g, D).permute(0, 2, 1, 3, 4).reshape(N, maxq, H, D)
    lse = lse.view(N, K, maxq, g).transpose(1, 2).reshape(N, maxq, H)
    return dict(out=o[seq, place].to(st["q"].dtype), lse=lse[seq, place])


# ---------------------------------------------------------------------------- the framework's calls

def _own(st):
    from beacon_b200 import ops
    if st["op"] == "fwd":
        q, k, v = ops.qk_norm_rope_fwd(st["qkv"], st["q_gain"], st["k_gain"], st["table"], st["batch"], st["seq"],
                                       st["heads"], st["kv_heads"], interleaved=st["interleaved"], eps=_EPS)
        return dict(q=q, k=k, v=v)
    if st["op"] == "bwd":
        dqkv, dgq, dgk = ops.qk_norm_rope_bwd(st["dq"], st["dk"], st["dv"], st["qkv"], st["q_gain"], st["k_gain"],
                                              st["table"], interleaved=st["interleaved"], eps=_EPS)
        return dict(dqkv=dqkv, dq_gain=dgq, dk_gain=dgk)
    if st["op"] == "append":
        q = ops.qk_norm_rope_append(st["qkv"], st["q_gain"], st["k_gain"], st["table"], st["k_cache"], st["v_cache"],
                                    st["page_table"], st["cu_q"], st["kv_lens"], st["heads"],
                                    interleaved=st["interleaved"], eps=_EPS)
        return dict(q=q, k_cache=st["k_cache"], v_cache=st["v_cache"])
    out, lse = ops.paged_attention(st["q"], st["k_cache"], st["v_cache"], st["page_table"], st["cu_q"], st["kv_lens"],
                                   max_q=st["max_q"])
    return dict(out=out, lse=lse)


def run(state):
    if own:
        return _own(state)
    return dict(fwd=_plain_fwd, bwd=_plain_bwd, append=_plain_append, attention=_plain_attention)[state["op"]](state)


# ---------------------------------------------------------------------------- the work that cannot be avoided

def work(case):
    H, K, D = case["heads"], case["kv_heads"], case["dim"]
    size = 4 if case["dtype"] == "f32" else 2
    if case["op"] in ("fwd", "bwd"):
        tokens = case["batch"] * case["seq"]
        elems = tokens * (H + 2 * K) * D
        extra = 4 * case["seq"] * case["rot"] + 2 * D * size
        if case["op"] == "fwd":
            return {"bytes": 2 * elems * size + extra, "flops": 10 * tokens * (H + K) * D}
        # the value columns of qkv are not needed backwards
        return {"bytes": (2 * elems + tokens * (H + K) * D) * size + extra + 2 * D * size,
                "flops": 20 * tokens * (H + K) * D}
    q, kv = _lengths(case)
    tokens = int(q.sum())
    if case["op"] == "append":
        elems = tokens * (H + 2 * K) * D
        return {"bytes": 2 * elems * size + 4 * tokens * case["rot"] + 2 * D * size,
                "flops": 10 * tokens * (H + K) * D}
    seen = sum(int(n) * int(t - n) + int(n) * (int(n) + 1) // 2 for n, t in zip(q, kv))
    return {"bytes": 2 * tokens * H * D * size + 4 * tokens * H + 2 * int(kv.sum()) * K * D * size,
            "flops": 4 * D * H * seen}


# ---------------------------------------------------------------------------- the definition in 64 bits

def _exact_turn(x, gain, pos, case, sign=1.0):
    """Rotation by sign * position angle of gain * x / rms as complex numbers; x [T, heads, D] in 64 bits."""
    rot = case["rot"]
    i = torch.arange(rot // 2, dtype=torch.float64, device="cuda")
    angle = (pos.double()[:, None] * _THETA ** (-2.0 * i / rot)) * sign
    # the table that the operators are given holds its values in 32 bits
    turn = torch.complex(angle.cos().float().double(), angle.sin().float().double())[:, None]
    y = x * gain
    if case["interleaved"]:
        c = torch.view_as_complex(y[..., :rot].reshape(*y.shape[:-1], rot // 2, 2).contiguous()) * turn
        head = torch.view_as_real(c).flatten(-2)
    else:
        c = torch.complex(y[..., :rot // 2].contiguous(), y[..., rot // 2:rot].contiguous()) * turn
        head = torch.cat([c.real, c.imag], -1)
    return torch.cat([head, y[..., rot:]], -1)


def _exact_unit(x):
    return x / torch.sqrt((x * x).sum(-1, keepdim=True) / x.shape[-1] + _EPS)


def _exact_attention(case, st):
    H, K, D, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    g = H // K
    q_lens, kv_lens = _lengths(case)
    out = torch.empty(st["tokens"], H, D, dtype=torch.float64, device="cuda")
    lse = torch.empty(st["tokens"], H, dtype=torch.float64, device="cuda")
    first = 0
    for s, (n, t) in enumerate(zip(q_lens.tolist(), kv_lens.tolist())):
        pages = st["page_table"][s, :-(-t // page)].long()
        at = torch.arange(t - n, t, device="cuda")
        for h in range(K):
            k = st["k_cache"][pages, h].reshape(-1, D)[:t].double()
            v = st["v_cache"][pages, h].reshape(-1, D)[:t].double()
            for c in range(0, n, 512):
                m = min(512, n - c)
                q = st["q"][first + c:first + c + m, h * g:(h + 1) * g].double()
                logits = torch.tensordot(q, k, dims=([2], [1])) / math.sqrt(D)
                seen = torch.arange(t, device="cuda") <= at[c:c + m, None]
                logits = torch.where(seen[:, None], logits, -math.inf)
                z = torch.logsumexp(logits, -1)
                lse[first + c:first + c + m, h * g:(h + 1) * g] = z
                out[first + c:first + c + m, h * g:(h + 1) * g] = torch.exp(logits - z[..., None]) @ v
        first += n
    return dict(out=out, lse=lse)


def exact(case, seed):
    st = prepare(case, seed)
    H, K, D = case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "attention":
        return _exact_attention(case, st)
    x = st["qkv"].double().view(-1, H + 2 * K, D)
    gq, gk = st["q_gain"].double(), st["k_gain"].double()
    if case["op"] == "append":
        q_lens, kv_lens = _lengths(case)
        seq = np.repeat(np.arange(case["seqs"]), q_lens)
        pos = np.concatenate([np.arange(t - n, t) for n, t in zip(q_lens, kv_lens)])
        pos_d = torch.tensor(pos, device="cuda")
        page = st["page_table"].long()[torch.tensor(seq, device="cuda"), pos_d // case["page"]]
        kc, vc = st["k_cache"].double(), st["v_cache"].double()
        kc[page, :, pos_d % case["page"]] = _exact_turn(_exact_unit(x[:, H:H + K]), gk, pos_d, case)
        vc[page, :, pos_d % case["page"]] = x[:, H + K:]
        return dict(q=_exact_turn(_exact_unit(x[:, :H]), gq, pos_d, case), k_cache=kc, v_cache=vc)
    B, S = case["batch"], case["seq"]
    pos = torch.arange(S, device="cuda").repeat(B)
    lay = lambda y: y.view(B, S, -1, D).transpose(1, 2).contiguous()  # noqa: E731
    if case["op"] == "fwd":
        return dict(q=lay(_exact_turn(_exact_unit(x[:, :H]), gq, pos, case)),
                    k=lay(_exact_turn(_exact_unit(x[:, H:H + K]), gk, pos, case)), v=lay(x[:, H + K:].contiguous()))
    one = torch.ones_like(gq)
    grads, gains = [], []
    for name, part, gain in (("dq", x[:, :H], gq), ("dk", x[:, H:H + K], gk)):
        dy = st[name].double().transpose(1, 2).flatten(0, 1)
        dz = _exact_turn(dy, one, pos, case, sign=-1.0)
        ms = (part * part).mean(-1, keepdim=True) + _EPS
        gains.append((dz * part / ms.sqrt()).sum((0, 1)))
        e = dz * gain
        grads.append(e / ms.sqrt() - part * (e * part).sum(-1, keepdim=True) / (D * ms ** 1.5))
    grads.append(st["dv"].double().transpose(1, 2).flatten(0, 1))
    return dict(dqkv=torch.cat(grads, 1).flatten(1), dq_gain=gains[0], dk_gain=gains[1])
