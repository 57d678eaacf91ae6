"""Attention over a paged key/value cache, and the append that fills it, through the C ABI against
64-bit NumPy (paged_ref).

Tolerances (norm-wise relative error).  f32: exact fp32 products, 1e-5.  bf16: the inputs are exact bf16
values; the probabilities are rounded to bf16 for the second product (at most 2^-9 each, their sum is
kept in fp32) and the output once more, so the error is below 2^-9 sum p|v| / |sum p v| + 2^-9; the
rounding errors average over the keys as the values do, which leaves a few times 2^-9: 2^-7.
lse is fp32 throughout: 1e-5 absolute for values of order ten."""
import numpy as np
import pytest

import paged_ref as R
from helpers import F32_TOL, as_bf16, normal, rel_err, to_dev, to_np

pytestmark = pytest.mark.gpu

BF16_ATTN, BF16_ONCE, LSE_TOL = 2.0 ** -7, 2.0 ** -8, 1e-5


def _dt(name):
    import torch
    return (torch.bfloat16, as_bf16, BF16_ATTN) if name == "bf16" else (torch.float32, lambda a: a, F32_TOL)


class Case:
    """Sequences over a shuffled pool; slots at or beyond a sequence's length hold NaN, and page table
    entries beyond its last page are out of range."""

    def __init__(self, q_lens, kv_lens, H, K, D, page, dt, seed=1, spare=2, table_pad=1):
        import torch
        self.tdt, self.r, self.tol = _dt(dt)
        self.q_lens, self.kv_lens, self.H, self.K, self.D, self.page = q_lens, kv_lens, H, K, D, page
        need = [-(-n // page) for n in kv_lens]
        pool = sum(need) + spare
        order = np.random.RandomState(seed).permutation(pool)
        self.table = np.full((len(kv_lens), max(need + [0]) + table_pad), -7, dtype=np.int32)
        self.k = np.full((pool, K, page, D), np.nan, dtype=np.float32)
        self.v = np.full((pool, K, page, D), np.nan, dtype=np.float32)
        at = 0
        for s, n in enumerate(kv_lens):
            pages = order[at:at + need[s]]
            at += need[s]
            self.table[s, :need[s]] = pages
            kk, vv = (self.r(normal((n, K, D), seed + 10 * s + i, std=1.2)) for i in (3, 4))
            for j in range(n):
                self.k[pages[j // page], :, j % page] = kk[j]
                self.v[pages[j // page], :, j % page] = vv[j]
        self.T = int(sum(q_lens))
        self.q = self.r(normal((self.T, H, D), seed + 5, std=1.2))
        self.cu = torch.tensor(np.concatenate([[0], np.cumsum(q_lens)]).astype(np.int32), device="cuda")
        self.kv = torch.tensor(np.array(kv_lens, dtype=np.int32), device="cuda")
        self.pt = torch.from_numpy(self.table).cuda()
        self.dq, self.dk, self.dv = (to_dev(a, self.tdt) for a in (self.q, self.k, self.v))

    def run(self, **kw):
        from beacon_b200 import ops
        return ops.paged_attention(self.dq, self.dk, self.dv, self.pt, self.cu, self.kv, **kw)

    def check(self, out, lse, causal=True):
        ref, rl = R.paged_attention(self.q, self.k, self.v, self.table, self.q_lens, self.kv_lens, causal)
        got, gl = to_np(out).astype(np.float64), to_np(lse).astype(np.float64)
        assert np.isfinite(got).all()
        empty = np.isneginf(rl)
        assert np.array_equal(np.isneginf(gl), empty) and np.all(got[empty] == 0)
        if (~empty).any():
            assert rel_err(got, ref) <= self.tol
            assert np.abs(gl[~empty] - rl[~empty]).max() <= LSE_TOL
            # no single row hides behind the others
            rows = np.linalg.norm(got - ref, axis=-1) / np.maximum(np.linalg.norm(ref, axis=-1), 1e-30)
            assert rows[~empty].max() <= 4 * self.tol


LENGTHS = {
    "one_token": ([1], [1]),
    "decode": ([1, 1, 1, 1, 1], [1, 127, 128, 129, 700]),
    "prompt_alone": ([300], [300]),
    "chunks": ([5, 64, 1, 130], [5, 100, 257, 513]),
    "empty_sequences": ([0, 3, 0, 2, 0], [0, 9, 40, 2, 0]),
    "rows_that_see_nothing": ([6, 4], [2, 0]),  # more new tokens than cached ones: the first see no key
    "many": ([1] * 70, [(37 * i) % 90 + 1 for i in range(70)]),
}
HEADS = [(4, 4, 64), (8, 2, 128), (6, 2, 64), (8, 1, 128), (3, 1, 32), (2, 2, 16), (5, 1, 128)]


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("H,K,D", HEADS)
@pytest.mark.parametrize("lengths", LENGTHS)
def test_lengths_and_heads(lengths, H, K, D, dt):
    from beacon_b200 import ops
    c = Case(*LENGTHS[lengths], H, K, D, 16, dt, seed=H + D)
    out, lse = c.run()
    assert ops.device_status(0)[0] == 0
    c.check(out, lse)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("page", [1, 5, 8, 24, 32, 64, 100, 128, 256, 384])
@pytest.mark.parametrize("q_lens,kv_lens", [([1, 1, 1], [300, 64, 385]), ([70, 3], [301, 129])])
def test_page_sizes(page, q_lens, kv_lens, dt):
    from beacon_b200 import ops
    c = Case(q_lens, kv_lens, 4, 2, 128, page, dt, seed=page)
    out, lse = c.run(max_q=max(q_lens))
    assert ops.device_status(0)[0] == 0
    c.check(out, lse)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("H,K,D", [(4, 2, 128), (16, 1, 64), (40, 2, 64)])
def test_every_key_for_every_token(H, K, D, dt):
    c = Case([3, 140, 0, 1, 2], [200, 150, 30, 1, 0], H, K, D, 32, dt)
    out, lse = c.run(causal=False)
    c.check(out, lse, causal=False)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("H,K,D,max_q", [(8, 8, 128, 1), (8, 1, 64, 1), (130, 1, 64, 1), (32, 2, 128, 3)])
def test_wide_groups_and_either_kernel_for_any_length(H, K, D, max_q, dt):
    """max_q is a hint: a wrong one changes the kernel, not the result."""
    c = Case([1, 9, 2], [260, 40, 129], H, K, D, 16, dt, seed=H)
    for hint in (max_q, 0, 4096):
        out, lse = c.run(max_q=hint)
        c.check(out, lse)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_long_context_split_over_the_device_repeats_bit_for_bit(dt):
    import torch
    c = Case([1, 2], [9000, 33], 4, 1, 64, 64, dt, seed=5)
    first = c.run(max_q=2)
    c.check(*first)
    for _ in range(3):
        again = c.run(max_q=2)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("D", [64, 128])
def test_full_and_short_items_split_in_two_repeat_bit_for_bit(D, causal):
    """Items of 256 rows and of at most 128 take different times per key tile; most of these fall into two
    runs, either of which may end last."""
    import torch
    c = Case([130, 60, 3, 200, 64, 20, 128, 65], [1900, 1100, 1501, 1280, 1663, 1, 1409, 1153], 16, 8, D, 16, "bf16",
             seed=D)
    first = c.run(max_q=200, causal=causal)
    c.check(*first, causal=causal)
    for _ in range(5):
        again = c.run(max_q=200, causal=causal)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_strided_pool_strided_queries_and_unowned_rows(dt):
    """Keys and values interleaved in one pool of another layout ([pages, page, 2, heads, D]), queries as a
    slice of wider rows, token rows beyond the last sequence left alone."""
    import torch
    from beacon_b200 import ops
    c = Case([1, 30, 2], [77, 50, 200], 4, 2, 64, 16, dt, seed=8)
    pool = torch.empty(c.k.shape[0], c.page, 2, c.K, c.D, dtype=c.tdt, device="cuda")
    kc, vc = pool[:, :, 0].transpose(1, 2), pool[:, :, 1].transpose(1, 2)
    kc.copy_(c.dk)
    vc.copy_(c.dv)
    wide = torch.full((c.T + 3, c.H * c.D + 40), float("nan"), dtype=c.tdt, device="cuda")
    q = wide[:, 16:16 + c.H * c.D].unflatten(1, (c.H, c.D))
    q[:c.T] = c.dq
    out = torch.full((c.T + 3, c.H, c.D), 7.0, dtype=c.tdt, device="cuda")
    lse = torch.full((c.T + 3, c.H), 7.0, device="cuda")
    ops.paged_attention(q, kc, vc, c.pt, c.cu, c.kv, out=out, lse=lse)
    assert ops.device_status(0)[0] == 0
    c.check(out[:c.T], lse[:c.T])
    assert (out[c.T:] == 7).all() and (lse[c.T:] == 7).all()
    plain = c.run()
    assert torch.equal(out[:c.T], plain[0]) and torch.equal(lse[:c.T], plain[1])


def test_offsets_beyond_32_bits():
    """A pool of more than 2^32 bytes and 2^31 elements per cache, the pages in use at its end."""
    import torch
    from beacon_b200 import ops
    K, D, page = 8, 128, 64
    pages = (1 << 31) // (K * D * page) + 4
    c = Case([1, 5], [130, 64], 16, K, D, page, "bf16", spare=0)
    n = c.k.shape[0]
    kc, vc = (torch.empty(pages, K, page, D, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    kc[pages - n:] = c.dk
    vc[pages - n:] = c.dv
    pt = torch.where(c.pt >= 0, c.pt + (pages - n), c.pt)
    for hint in (1, 5, 200):
        out, lse = ops.paged_attention(c.dq, kc, vc, pt, c.cu, c.kv, max_q=hint)
        c.check(out, lse)
    table = to_dev(R.table64(130, D).astype(np.float32), torch.float32)
    x = to_dev(as_bf16(normal((c.T, 32 * D), 4)), torch.bfloat16)
    small_k, small_v = c.dk.clone(), c.dv.clone()
    ops.qk_norm_rope_append(x, None, None, table, kc, vc, pt, c.cu, c.kv, 16)
    ops.qk_norm_rope_append(x, None, None, table, small_k, small_v, c.pt, c.cu, c.kv, 16)
    assert torch.equal(kc[pages - n:].nan_to_num(5.0), small_k.nan_to_num(5.0))
    assert torch.equal(vc[pages - n:].nan_to_num(5.0), small_v.nan_to_num(5.0))
    assert ops.device_status(0)[0] == 0


@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_bad_pages_and_lengths_are_not_followed(dt):
    """A page index outside the cache reads as zeros, lengths past the tensors are cut; both are recorded."""
    import torch
    from beacon_b200 import errors, ops
    c = Case([1, 2], [40, 20], 4, 2, 64, 16, dt, seed=3)
    bad = c.pt.clone()
    bad[0, 1] = c.k.shape[0] + 100
    out, lse = ops.paged_attention(c.dq, c.dk, c.dv, bad, c.cu, c.kv)
    with pytest.raises(errors.Cuda, match="code 3"):
        ops.device_status(0)
    zero = c.k.shape[0]
    k0, v0 = (np.concatenate([a, np.zeros_like(a[:1])]) for a in (c.k, c.v))
    t0 = c.table.copy()
    t0[0, 1] = zero
    ref, _ = R.paged_attention(c.q, k0, v0, t0, c.q_lens, c.kv_lens)
    assert rel_err(to_np(out), ref) <= c.tol
    long_kv = c.kv.clone()
    long_kv[1] = 1 << 20
    out, _ = ops.paged_attention(c.dq, c.dk, c.dv, c.pt.clamp(min=0), c.cu, long_kv)
    with pytest.raises(errors.Cuda, match="code 3"):
        ops.device_status(0)
    assert rel_err(to_np(out[:1]), ref[:1]) > 0  # sequence 0 was computed; nothing faulted
    past = c.cu.clone()
    past[2] = 1 << 20
    out, lse = torch.zeros_like(c.dq), torch.zeros(c.T, c.H, device="cuda")
    ops.paged_attention(c.dq, c.dk, c.dv, c.pt, c.cu * 0 + past, c.kv, out=out, lse=lse)
    with pytest.raises(errors.Cuda, match="code 3"):
        ops.device_status(0)


# ------------------------------------------------------------------------------ append

@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("H,K,D,rot,page", [(8, 2, 128, 128, 16), (6, 2, 64, 32, 5), (4, 4, 64, 64, 64),
                                            (3, 1, 40, 40, 16), (5, 1, 32, 0, 8)])
def test_append(H, K, D, rot, page, interleaved, dt):
    """Queries and the written slots against 64 bits; every other slot keeps its bits."""
    import torch
    from beacon_b200 import ops
    q_lens, kv_lens = [1, 0, 40, 3, 1], [130, 12, 40, 67, 1]
    c = Case(q_lens, kv_lens, H, K, D, page, dt, seed=D + page)
    tol = BF16_ONCE if dt == "bf16" else F32_TOL
    x = c.r(normal((c.T + 2, (H + 2 * K) * D), 31, std=1.3))
    gq, gk = c.r(1 + 0.2 * normal((D,), 32)), c.r(1 + 0.2 * normal((D,), 33))
    table = R.table64(200, rot).astype(np.float32) if rot else None
    t64 = None if table is None else table.astype(np.float64)
    kc, vc = c.dk.clone(), c.dv.clone()
    q = torch.full((c.T + 2, H, D), 9.0, dtype=c.tdt, device="cuda")
    ops.qk_norm_rope_append(to_dev(x, c.tdt), to_dev(gq, c.tdt), to_dev(gk, c.tdt),
                            None if table is None else to_dev(table, torch.float32), kc, vc, c.pt, c.cu, c.kv, H,
                            interleaved=interleaved, q=q)
    assert ops.device_status(0)[0] == 0
    assert (q[c.T:] == 9).all()  # rows that no sequence owns
    x3 = x[:c.T].reshape(c.T, H + 2 * K, D)
    pos = np.concatenate([np.arange(t - n, t) for n, t in zip(q_lens, kv_lens)]).astype(np.int64)
    seq = np.repeat(np.arange(len(q_lens)), q_lens)
    assert rel_err(to_np(q[:c.T]), R.norm_rope(x3[:, :H], gq, t64, pos, interleaved)) <= tol
    pages, slots = c.table[seq, pos // page], pos % page
    got_k, got_v = to_np(kc), to_np(vc)
    assert rel_err(got_k[pages, :, slots], R.norm_rope(x3[:, H:H + K], gk, t64, pos, interleaved)) <= tol
    assert np.array_equal(got_v[pages, :, slots], x3[:, H + K:])
    keep = np.ones(c.k.shape[:1] + (page,), dtype=bool)
    keep[pages, slots] = False
    keep = np.broadcast_to(keep[:, None, :, None], c.k.shape)
    assert np.array_equal(got_k[keep], c.k[keep], equal_nan=True) and np.array_equal(got_v[keep], c.v[keep],
                                                                                      equal_nan=True)


def test_append_with_given_positions_and_places_it_cannot_write():
    import torch
    from beacon_b200 import errors, ops
    c = Case([2, 3], [20, 2], 4, 2, 64, 16, "bf16")  # sequence 1: its first new token has no place
    x = c.r(normal((c.T, 8 * 64), 31))
    table = R.table64(500, 64).astype(np.float32)
    pos = np.array([400, 401, 3, 17, 499], dtype=np.int32)
    kc, vc = c.dk.clone(), c.dv.clone()
    q = ops.qk_norm_rope_append(to_dev(x, c.tdt), None, None, to_dev(table, torch.float32), kc, vc, c.pt, c.cu, c.kv,
                                4, positions=torch.from_numpy(pos).cuda())
    with pytest.raises(errors.Cuda, match="code 3"):
        ops.device_status(0)
    x3 = x.reshape(c.T, 8, 64)
    ref = R.norm_rope(x3[:, :6], None, table.astype(np.float64), pos, False)
    ref[2] = 0.0
    assert rel_err(to_np(q), ref[:, :4]) <= BF16_ONCE
    got = to_np(kc)
    for t, (s, j) in zip((0, 1, 3, 4), ((0, 18), (0, 19), (1, 0), (1, 1))):
        assert rel_err(got[c.table[s, j // 16], :, j % 16], ref[t, 4:]) <= BF16_ONCE
    bad = c.pt.clone()
    bad[0, 1] = -1  # the page of tokens 16 .. 19 of sequence 0
    k2, v2 = c.dk.clone(), c.dv.clone()
    ops.qk_norm_rope_append(to_dev(x, c.tdt), None, None, to_dev(table, torch.float32), k2, v2, bad, c.cu, c.kv, 4)
    with pytest.raises(errors.Cuda, match="code 3"):
        ops.device_status(0)
    p = c.table[0, 1]
    assert np.array_equal(to_np(k2)[p], c.k[p], equal_nan=True)


# ------------------------------------------------------------------------------ together

def test_prompt_in_chunks_equals_the_training_forward():
    """Appending and attending chunk by chunk gives what the training path gives for the whole prompt
    (qk_norm_rope_fwd, then causal attention)."""
    import torch
    from beacon_b200 import ops
    S, H, K, D, page = 333, 8, 2, 128, 16
    x = to_dev(as_bf16(normal((S, (H + 2 * K) * D), 3)), torch.bfloat16)
    g = to_dev(as_bf16(1 + 0.2 * normal((D,), 4)), torch.bfloat16)
    table = ops.rope_table(S, D)
    q, k, v = ops.qk_norm_rope_fwd(x, g, g, table, 1, S, H, K)
    ref, _ = ops.attention_fwd(q, k, v)  # its lse carries that kernel's exponential error, up to 2e-5
    n = -(-S // page)
    kc, vc = (torch.full((n, K, page, D), float("nan"), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    pt = torch.randperm(n, device="cuda").to(torch.int32).view(1, n)
    outs, at = [], 0
    for c in (100, 1, 1, 130, 90, 11):
        cu = torch.tensor([0, c], dtype=torch.int32, device="cuda")
        kv = torch.tensor([at + c], dtype=torch.int32, device="cuda")
        qc = ops.qk_norm_rope_append(x[at:at + c], g, g, table, kc, vc, pt, cu, kv, H)
        outs.append(ops.paged_attention(qc, kc, vc, pt, cu, kv, max_q=c))
        at += c
    assert at == S and ops.device_status(0)[0] == 0
    out, lse = torch.cat([o for o, _ in outs]), torch.cat([l for _, l in outs])
    assert rel_err(to_np(out), to_np(ref[0].transpose(0, 1))) <= BF16_ATTN
    tokens = lambda a: to_np(a[0].transpose(0, 1))  # noqa: E731
    ref64, lse64 = R.paged_attention(tokens(q), tokens(k)[None].transpose(0, 2, 1, 3),
                                     tokens(v)[None].transpose(0, 2, 1, 3), np.zeros((1, 1), np.int32), [S], [S])
    assert rel_err(to_np(out), ref64) <= BF16_ATTN
    assert np.abs(to_np(lse) - lse64).max() <= LSE_TOL


def test_block_over_chunks_and_single_tokens():
    """The pre-norm block on two sequences' prompts in ragged chunks, then on single tokens, against the
    whole sequences in 64 bits (the framework's bf16 tolerance)."""
    import torch
    from beacon_b200 import ops
    from helpers import BF16_TOL
    dm, H, K, D, F, page, lens = 256, 4, 2, 64, 384, 16, (75, 40)
    r = as_bf16
    w = dict(attn_norm=r(1 + 0.1 * normal((dm,), 1)), w_qkv=r(normal((dm, (H + 2 * K) * D), 2, std=0.05)),
             w_o=r(normal((H * D, dm), 3, std=0.05)), ffn_norm=r(1 + 0.1 * normal((dm,), 4)),
             w_gate=r(normal((dm, F), 5, std=0.05)), w_up=r(normal((dm, F), 6, std=0.05)),
             w_down=r(normal((F, dm), 7, std=0.05)))
    gq, gk = r(1 + 0.2 * normal((D,), 8)), r(1 + 0.2 * normal((D,), 9))
    xs = [r(normal((n, dm), 10 + i)) for i, n in enumerate(lens)]
    t64 = R.table64(max(lens), D).astype(np.float32).astype(np.float64)

    def rms(a, g):
        return a / np.sqrt((a * a).mean(-1, keepdims=True) + 1e-5) * g

    refs = []
    for x in xs:
        n, x = len(x), x.astype(np.float64)
        qkv = (rms(x, w["attn_norm"]) @ w["w_qkv"]).reshape(n, H + 2 * K, D)
        q, k = (R.norm_rope(a, g, t64, np.arange(n), False) for a, g in ((qkv[:, :H], gq), (qkv[:, H:H + K], gk)))
        ao, _ = R.paged_attention(q, k[None].transpose(0, 2, 1, 3), qkv[None, :, H + K:].transpose(0, 2, 1, 3),
                                  np.zeros((1, 1), np.int32), [n], [n])
        h = x + ao.reshape(n, -1) @ w["w_o"]
        z = rms(h, w["ffn_norm"])
        gate = z @ w["w_gate"]
        refs.append(h + (gate / (1 + np.exp(-gate)) * (z @ w["w_up"])) @ w["w_down"])
    dev = [to_dev(w[n], torch.bfloat16) for n in ("attn_norm", "w_qkv", "w_o", "ffn_norm", "w_gate", "w_up", "w_down")]
    tab, dgq, dgk = ops.rope_table(max(lens), D), to_dev(gq, torch.bfloat16), to_dev(gk, torch.bfloat16)
    kc, vc = (torch.full((10, K, page, D), float("nan"), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    pt = torch.tensor([[3, 9, 0, 5, 1], [2, 7, 4, -1, -1]], dtype=torch.int32, device="cuda")
    need = ops.llama_block_paged_workspace_bytes(80, dm, H, K, D, F)
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    at, got = [0, 0], [[], []]
    for step in ((40, 0), (0, 33), (30, 5), (1, 1), (1, 1), (3, 0)):
        x = np.concatenate([xs[i][at[i]:at[i] + n] for i, n in enumerate(step)])
        at = [a + n for a, n in zip(at, step)]
        cu = torch.tensor([0, step[0], sum(step)], dtype=torch.int32, device="cuda")
        kv = torch.tensor(at, dtype=torch.int32, device="cuda")
        out = ops.llama_block_paged_fwd(to_dev(x, torch.bfloat16), *dev, kc, vc, pt, cu, kv, H, table=tab, q_gain=dgq,
                                        k_gain=dgk, max_q=max(step), workspace=ws if step[0] % 2 else None)
        out = to_np(out)
        got[0].append(out[:step[0]])
        got[1].append(out[step[0]:])
    assert at == list(lens) and ops.device_status(0)[0] == 0
    for i in range(2):
        mine = np.concatenate(got[i])
        assert rel_err(mine, refs[i]) <= BF16_TOL
        assert rel_err(mine - xs[i], refs[i] - xs[i]) <= BF16_TOL


def test_captured_step_follows_the_tables_on_the_device():
    """One captured append + attention, replayed while kv_lens and the inputs change on the device, on a
    side stream with a workspace of its own."""
    import torch
    from beacon_b200 import ops
    c = Case([1, 1, 1], [50, 7, 129], 8, 2, 128, 16, "bf16", table_pad=2)
    c.pt.clamp_(min=0)
    g = torch.ones(128, dtype=torch.bfloat16, device="cuda")
    table = ops.rope_table(200, 128)
    x = torch.zeros(3, 12 * 128, dtype=torch.bfloat16, device="cuda")
    kc, vc = c.dk.nan_to_num(0.5), c.dv.nan_to_num(0.5)
    q, out, lse = torch.empty_like(c.dq), torch.empty_like(c.dq), torch.empty(3, 8, device="cuda")
    ws = torch.empty(ops.paged_attention_workspace_bytes(128), dtype=torch.uint8, device="cuda")
    kv = c.kv.clone()

    def step():
        ops.qk_norm_rope_append(x, g, g, table, kc, vc, c.pt, c.cu, kv, 8, q=q)
        ops.paged_attention(q, kc, vc, c.pt, c.cu, kv, max_q=1, out=out, lse=lse, workspace=ws)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            step()
        for i in range(3):
            x.copy_(to_dev(as_bf16(normal(tuple(x.shape), 40 + i)), torch.bfloat16))
            kv.copy_(c.kv + i)
            graph.replay()
            side.synchronize()
            got, got_lse = out.clone(), lse.clone()
            ref, ref_lse = R.paged_attention(to_np(q), to_np(kc), to_np(vc), c.pt.cpu().numpy(), [1, 1, 1],
                                             [n + i for n in c.kv_lens])
            assert rel_err(to_np(got), ref) <= BF16_ATTN
            assert np.abs(to_np(got_lse) - ref_lse).max() <= LSE_TOL
    del graph
    assert ops.device_status(0)[0] == 0
