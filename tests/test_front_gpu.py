"""The two call paths of the rotation and paged-cache operators, beacon_front's and ops' own, give the same
results and take the same operands."""
import pytest

from test_paged_gpu import Case

pytestmark = pytest.mark.gpu


def _both(monkeypatch, fn):
    from beacon_b200 import _lib
    a = fn()
    monkeypatch.setattr(_lib, "_front", _lib._NoFront())
    b = fn()
    monkeypatch.undo()
    return a, b


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("q_lens,kv_lens", [([1, 1, 1], [50, 700, 3000]), ([40, 1, 130], [40, 90, 1500]), ([1], [1])])
@pytest.mark.parametrize("interleaved", [False, True])
def test_same_bits_from_both_paths(q_lens, kv_lens, interleaved, dt, monkeypatch):
    import torch
    from beacon_b200 import _lib, ops
    assert not isinstance(_lib.front(), _lib._NoFront)
    H, K, D = 8, 2, 128
    c = Case(q_lens, kv_lens, H, K, D, 16, dt)
    gen = torch.Generator("cuda").manual_seed(1)
    rnd = lambda *s: torch.randn(*s, generator=gen, device="cuda").to(c.tdt)  # noqa: E731
    table = ops.rope_table(max(kv_lens), D)
    x, gq, gk = rnd(c.T, (H + 2 * K) * D + 16)[:, :(H + 2 * K) * D], rnd(D), rnd(D)
    pos = torch.arange(c.T, dtype=torch.int32, device="cuda") % max(kv_lens)
    dy = [rnd(1, n, c.T, D) for n in (H, K, K)]
    one = max(kv_lens) >= c.T

    def call():
        kc, vc = c.dk.nan_to_num(2.0), c.dv.nan_to_num(2.0)
        got = list(ops.qk_norm_rope_fwd(x, gq, gk, table, 1, c.T, H, K, positions=pos, interleaved=interleaved))
        got += ops.qk_norm_rope_fwd(x, None, gk, table if one else None, c.T, 1, H, K, interleaved=interleaved)
        got += ops.qk_norm_rope_bwd(*dy, x, gq, gk, table, positions=pos, interleaved=interleaved)
        got += ops.qk_norm_rope_bwd(*dy, x, gq, None, None)[:2]
        q = ops.qk_norm_rope_append(x, gq, gk, table, kc, vc, c.pt, c.cu, c.kv, H, interleaved=interleaved)
        got += [q, kc, vc]
        for causal in (True, False):
            got += ops.paged_attention(q, kc, vc, c.pt, c.cu, c.kv, max_q=max(q_lens), causal=causal)
        return got

    a, b = _both(monkeypatch, call)
    assert len(a) == len(b)
    assert all(p.shape == q.shape and p.dtype == q.dtype and torch.equal(p, q) for p, q in zip(a, b))
    assert ops.device_status(0)[0] == 0


def test_same_refusals_from_both_paths(monkeypatch):
    import torch
    from beacon_b200 import errors, ops
    c = Case([1, 2], [20, 30], 4, 2, 64, 16, "bf16")
    x = torch.zeros(c.T, 8 * 64, dtype=torch.bfloat16, device="cuda")
    g, t = torch.ones(64, dtype=torch.bfloat16, device="cuda"), ops.rope_table(40, 64)
    calls = [
        lambda: ops.qk_norm_rope_fwd(x, g, g.float(), t, 1, c.T, 4, 2),
        lambda: ops.qk_norm_rope_fwd(x, g, g, t.half(), 1, c.T, 4, 2),
        lambda: ops.qk_norm_rope_fwd(x, g[:32], g, t, 1, c.T, 4, 2),
        lambda: ops.qk_norm_rope_fwd(x.half(), None, None, t, 1, c.T, 4, 2),
        lambda: ops.qk_norm_rope_fwd(x, g, g, t, 1, c.T, 3, 2),
        lambda: ops.qk_norm_rope_fwd(x, g, g, t, 1, c.T, 4, 2, positions=c.kv),
        lambda: ops.qk_norm_rope_append(x, g, g, t, c.dk, c.dv.float(), c.pt, c.cu, c.kv, 4),
        lambda: ops.qk_norm_rope_append(x, g, g, t, c.dk, c.dv, c.pt, c.cu[:2], c.kv, 4),
        lambda: ops.qk_norm_rope_append(x, g, g, t, c.dk, c.dv, c.pt.long(), c.cu, c.kv, 4),
        lambda: ops.paged_attention(c.dq.float(), c.dk, c.dv, c.pt, c.cu, c.kv),
        lambda: ops.paged_attention(c.dq[:, :, :32], c.dk, c.dv, c.pt, c.cu, c.kv),
        lambda: ops.paged_attention(c.dq, c.dk, c.dv.transpose(1, 2), c.pt, c.cu, c.kv),
        lambda: ops.paged_attention(c.dq, c.dk, c.dv, c.pt, c.cu, c.kv.cpu()),
        lambda: ops.paged_attention(c.dq, c.dk, c.dv, c.pt, c.cu, c.kv, workspace=torch.empty(1 << 26, dtype=torch.uint8)),
    ]

    def names():
        got = []
        for call in calls:
            with pytest.raises(errors.LaunchError) as e:
                call()
            got.append((type(e.value), str(e.value)))
        return got

    a, b = _both(monkeypatch, names)
    assert a == b
    assert ops.device_status(0)[0] == 0
