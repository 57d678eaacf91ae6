"""The per-head query/key norm with the position rotation, forward and backward, through the C ABI
against 64-bit NumPy (paged_ref).

Tolerances (norm-wise relative error): a bf16 result is rounded once from fp32, at most 2^-9 of each
value, so 2^-8 holds with the fp32 arithmetic's error on top; a bf16 backward rounds dx once too.  The
f32 results are sums of at most a few thousand products, 1e-5 as on the framework's f32 path."""
import numpy as np
import pytest

import paged_ref as R
from helpers import F32_TOL, as_bf16, normal, rel_err, to_dev, to_np

pytestmark = pytest.mark.gpu

BF16_ONCE = 2.0 ** -8


def _dt(name):
    import torch
    return (torch.bfloat16, as_bf16, BF16_ONCE) if name == "bf16" else (torch.float32, lambda a: a, F32_TOL)


def _inputs(B, S, H, K, D, dt, seed):
    tdt, r, tol = _dt(dt)
    x = r(normal((B * S, (H + 2 * K) * D), seed, std=1.3))
    gq, gk = r(1.0 + 0.2 * normal((D,), seed + 1)), r(1.0 + 0.2 * normal((D,), seed + 2))
    return tdt, r, tol, x, gq, gk


def _head_major(y, B, S):
    return y.reshape(B, S, y.shape[1], y.shape[2]).transpose(0, 2, 1, 3)


# one token; odd lengths; every vectorised head_dim, and head dims and rotated widths that only the
# element-by-element kernel takes (2, 40, 80, 96, 250; rot 8, 30); groups of 1, 3, 8; no rotation
SHAPES = [
    (1, 1, 1, 1, 64, 64), (2, 129, 4, 4, 128, 128), (3, 67, 6, 2, 64, 32), (1, 33, 8, 1, 128, 64),
    (2, 20, 3, 1, 16, 16), (1, 50, 4, 2, 32, 16), (1, 9, 2, 2, 256, 256), (1, 7, 3, 1, 40, 40),
    (2, 5, 5, 5, 80, 30), (1, 31, 2, 1, 96, 96), (1, 3, 2, 2, 250, 250), (1, 4, 1, 1, 2, 2),
    (1, 17, 4, 2, 64, 8), (2, 19, 4, 2, 128, 0), (1, 700, 12, 4, 128, 128),
]


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("B,S,H,K,D,rot", SHAPES)
def test_forward(B, S, H, K, D, rot, interleaved, dt):
    import torch
    from beacon_b200 import ops
    tdt, r, tol, x, gq, gk = _inputs(B, S, H, K, D, dt, 3 * D + S)
    table = R.table64(S, rot).astype(np.float32) if rot else None
    q, k, v = ops.qk_norm_rope_fwd(to_dev(x, tdt), to_dev(gq, tdt), to_dev(gk, tdt),
                                   None if table is None else to_dev(table, torch.float32), B, S, H, K,
                                   interleaved=interleaved)
    assert ops.device_status(0)[0] == 0
    x3, pos = x.reshape(B * S, H + 2 * K, D), np.tile(np.arange(S), B)
    t64 = None if table is None else table.astype(np.float64)
    assert rel_err(to_np(q), _head_major(R.norm_rope(x3[:, :H], gq, t64, pos, interleaved), B, S)) <= tol
    assert rel_err(to_np(k), _head_major(R.norm_rope(x3[:, H:H + K], gk, t64, pos, interleaved), B, S)) <= tol
    assert np.array_equal(to_np(v), _head_major(x3[:, H + K:], B, S))


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("B,S,H,K,D,rot", SHAPES)
def test_backward(B, S, H, K, D, rot, interleaved, dt):
    import torch
    from beacon_b200 import ops
    tdt, r, tol, x, gq, gk = _inputs(B, S, H, K, D, dt, 5 * D + S)
    table = R.table64(S, rot).astype(np.float32) if rot else None
    dq, dk, dv = (r(normal((B, n, S, D), 70 + i)) for i, n in enumerate((H, K, K)))
    args = [to_dev(a, tdt) for a in (dq, dk, dv, x, gq, gk)]
    tab = None if table is None else to_dev(table, torch.float32)
    dx, dgq, dgk = ops.qk_norm_rope_bwd(*args, tab, interleaved=interleaved)
    again = ops.qk_norm_rope_bwd(*args, tab, interleaved=interleaved)
    assert ops.device_status(0)[0] == 0
    assert all(torch.equal(a, b) for a, b in zip((dx, dgq, dgk), again))  # sums in a fixed order
    x3, pos = x.reshape(B * S, H + 2 * K, D), np.tile(np.arange(S), B)
    t64 = None if table is None else table.astype(np.float64)
    rows = lambda a: a.transpose(0, 2, 1, 3).reshape(B * S, a.shape[1], D)  # noqa: E731
    rq, rgq = R.norm_rope_bwd(rows(dq), x3[:, :H], gq, t64, pos, interleaved)
    rk, rgk = R.norm_rope_bwd(rows(dk), x3[:, H:H + K], gk, t64, pos, interleaved)
    got = to_np(dx).reshape(x3.shape)
    assert rel_err(got[:, :H], rq) <= tol and rel_err(got[:, H:H + K], rk) <= tol
    assert np.array_equal(got[:, H + K:], rows(dv))
    assert rel_err(to_np(dgq), rgq) <= tol and rel_err(to_np(dgk), rgk) <= tol


@pytest.mark.parametrize("interleaved", [False, True])
def test_backward_against_differences(interleaved):
    """<dy, f(x + h u) - f(x - h u)> / 2h = <dx, u> in every input, f in 64 bits: the difference's own
    error is h^2 of order 1e-8 at h = 1e-4, the gradient's 1e-5 of its size."""
    import torch
    from beacon_b200 import ops
    B, S, H, K, D, rot = 1, 13, 4, 2, 64, 32
    tdt, r, tol, x, gq, gk = _inputs(B, S, H, K, D, "f32", 9)
    table = R.table64(S, rot).astype(np.float32)
    dq, dk, dv = (normal((B, n, S, D), 80 + i) for i, n in enumerate((H, K, K)))
    dx, dgq, dgk = (to_np(t).astype(np.float64) for t in ops.qk_norm_rope_bwd(
        *(to_dev(a, tdt) for a in (dq, dk, dv, x, gq, gk)), to_dev(table, torch.float32), interleaved=interleaved))

    def loss(xv, a, b):
        x3, pos = xv.reshape(S, H + 2 * K, D), np.arange(S)
        t64 = table.astype(np.float64)
        q = R.norm_rope(x3[:, :H], a, t64, pos, interleaved).transpose(1, 0, 2)
        k = R.norm_rope(x3[:, H:H + K], b, t64, pos, interleaved).transpose(1, 0, 2)
        return (q * dq[0]).sum() + (k * dk[0]).sum() + (x3[:, H + K:].transpose(1, 0, 2) * dv[0]).sum()

    h, base = 1e-4, [a.astype(np.float64) for a in (x, gq, gk)]
    for i, grad in enumerate((dx, dgq, dgk)):
        for seed in (1, 2, 3):
            u = normal(base[i].shape, 200 + 10 * i + seed).astype(np.float64)
            up, dn = list(base), list(base)
            up[i], dn[i] = base[i] + h * u, base[i] - h * u
            diff = (loss(*up) - loss(*dn)) / (2 * h)
            scale = np.linalg.norm(grad) * np.linalg.norm(u)
            assert abs(diff - (grad * u).sum()) <= 1e-5 * scale


def test_one_gain_or_none_positions_strides_and_missing_values():
    import torch
    from beacon_b200 import ops
    B, S, H, K, D = 2, 11, 4, 2, 128
    tdt, r, tol, x, gq, gk = _inputs(B, S, H, K, D, "bf16", 17)
    table = R.table64(100, D).astype(np.float32)
    pos = (normal((B * S,), 3) * 20).astype(np.int32) % 100
    wide = torch.full((B * S, x.shape[1] + 24), float("nan"), dtype=tdt, device="cuda")
    wide[:, 8:8 + x.shape[1]] = to_dev(x, tdt)  # rows 48 bytes apart beyond their width, 16-byte aligned
    odd = torch.full((B * S, x.shape[1] + 3), float("nan"), dtype=tdt, device="cuda")
    odd[:, 1:1 + x.shape[1]] = to_dev(x, tdt)   # rows that no 16-byte load can take
    x3 = x.reshape(B * S, H + 2 * K, D)
    dpos = torch.from_numpy(pos).cuda()
    dq, dk, dv = (r(normal((B, n, S, D), 60 + i)) for i, n in enumerate((H, K, K)))
    rows = lambda a: a.transpose(0, 2, 1, 3).reshape(B * S, a.shape[1], D)  # noqa: E731
    for a, b in ((gq, None), (None, gk), (None, None), (gq, gk)):
        da, db = (None if g is None else to_dev(g, tdt) for g in (a, b))
        ref_q = _head_major(R.norm_rope(x3[:, :H], a, table.astype(np.float64), pos, False), B, S)
        ref_k = _head_major(R.norm_rope(x3[:, H:H + K], b, table.astype(np.float64), pos, False), B, S)
        rq, rgq = R.norm_rope_bwd(rows(dq), x3[:, :H], a, table.astype(np.float64), pos, False)
        rk, rgk = R.norm_rope_bwd(rows(dk), x3[:, H:H + K], b, table.astype(np.float64), pos, False)
        for src in (wide[:, 8:8 + x.shape[1]], odd[:, 1:1 + x.shape[1]]):
            q, k, v = ops.qk_norm_rope_fwd(src, da, db, to_dev(table, torch.float32), B, S, H, K, positions=dpos)
            assert rel_err(to_np(q), ref_q) <= tol and rel_err(to_np(k), ref_k) <= tol
            dx, dgq, dgk = ops.qk_norm_rope_bwd(to_dev(dq, tdt), to_dev(dk, tdt), to_dev(dv, tdt), src, da, db,
                                                to_dev(table, torch.float32), positions=dpos)
            got = to_np(dx).reshape(x3.shape)
            assert rel_err(got[:, :H], rq) <= tol and rel_err(got[:, H:H + K], rk) <= tol
            for mine, ref in ((dgq, rgq), (dgk, rgk)):
                assert (mine is None) == (ref is None)
                assert mine is None or rel_err(to_np(mine), ref) <= tol
    assert ops.device_status(0)[0] == 0


def test_zero_rows_large_values_and_a_position_outside_the_table():
    import torch
    from beacon_b200 import errors, ops
    S, H, K, D = 6, 2, 1, 64
    tdt, r, tol, x, gq, gk = _inputs(1, S, H, K, D, "bf16", 23)
    x[0] = 0.0       # a head of zeros: r = sqrt(eps), y = 0
    x[1] *= 1e15     # squares near 1e30, sums still inside fp32
    x = r(x)         # what the device receives
    table = R.table64(S - 1, D).astype(np.float32)
    x3 = x.reshape(S, H + 2 * K, D)
    dev = [to_dev(x, tdt), to_dev(gq, tdt), to_dev(gk, tdt), to_dev(table, torch.float32)]
    q, k, v = ops.qk_norm_rope_fwd(*dev, 1, S, H, K)
    with pytest.raises(errors.Cuda, match="code 3"):  # token 5 has no row in a table of 5
        ops.device_status(0)
    ref = _head_major(R.norm_rope(x3[:5, :H], gq, table.astype(np.float64), np.arange(5), False), 1, 5)
    assert rel_err(to_np(q)[:, :, :5], ref) <= tol
    assert np.all(to_np(q)[:, :, 5] == 0) and np.all(to_np(k)[:, :, 5] == 0)
    assert np.array_equal(to_np(v), _head_major(x3[:, H + K:], 1, S))
    dy = [to_dev(r(normal((1, n, S, D), 90 + n)), tdt) for n in (H, K, K)]
    dx, _, _ = ops.qk_norm_rope_bwd(*dy, *dev)
    with pytest.raises(errors.Cuda, match="code 3"):
        ops.device_status(0)
    got = to_np(dx).reshape(x3.shape)
    assert np.all(got[5, :H + K] == 0) and np.isfinite(got).all()


def test_empty_batch_zeroes_the_gain_gradients_and_table_matches():
    import torch
    from beacon_b200 import ops
    g = torch.ones(64, dtype=torch.float32, device="cuda")
    e = lambda n: torch.empty(0, n, 5, 64, device="cuda")  # noqa: E731
    dx, dgq, dgk = ops.qk_norm_rope_bwd(e(4), e(2), e(2), torch.empty(0, 8 * 64, device="cuda"), g, g, None)
    assert dx.numel() == 0 and not dgq.any() and not dgk.any()
    got = to_np(ops.rope_table(70000, 32, theta=5e5))
    # each entry is the 64-bit value rounded once to fp32: off by at most 2^-25 below 1
    assert np.abs(got - R.table64(70000, 32, 5e5)).max() <= 2.0 ** -24
