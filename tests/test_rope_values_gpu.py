"""The rotation's backward where a token has no position: its gradients are zeros and the gains get nothing from
it, whatever the token's rows hold."""
import numpy as np
import pytest

import paged_ref as R
from helpers import normal, rel_err, to_dev, to_np
from test_rope_gpu import _inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("gains", [True, False])
@pytest.mark.parametrize("D,rot", [(64, 64), (128, 64), (256, 256), (40, 40)])
def test_nan_at_a_token_without_a_position(D, rot, gains, interleaved, dt):
    import torch
    from beacon_b200 import errors, ops
    B, S, H, K = 1, 37, 6, 3
    tdt, r, tol, x, gq, gk = _inputs(B, S, H, K, D, dt, 11 + D)
    table = R.table64(S, rot).astype(np.float32)
    pos = np.arange(S, dtype=np.int32)
    lost = [4, 36]
    pos[lost] = [-1, S]
    dq, dk, dv = (r(normal((B, n, S, D), 50 + i)) for i, n in enumerate((H, K, K)))
    x3 = x.reshape(S, H + 2 * K, D)
    keep = np.setdiff1d(np.arange(S), lost)
    rows = lambda a: a.transpose(0, 2, 1, 3).reshape(S, a.shape[1], D)  # noqa: E731
    t64 = table.astype(np.float64)
    rq, rgq = R.norm_rope_bwd(rows(dq)[keep], x3[keep, :H], gq if gains else None, t64, keep, interleaved)
    rk, rgk = R.norm_rope_bwd(rows(dk)[keep], x3[keep, H:H + K], gk if gains else None, t64, keep, interleaved)
    want_dv = rows(dv).copy()
    for a in (dq, dk):
        a[:, :, lost] = np.nan
    x3[lost, :H + K] = np.nan
    g = [to_dev(a, tdt) if gains else None for a in (gq, gk)]
    ops.device_status(0)
    dx, dgq, dgk = ops.qk_norm_rope_bwd(*(to_dev(a, tdt) for a in (dq, dk, dv)), to_dev(x, tdt), *g,
                                        to_dev(table, torch.float32), positions=torch.from_numpy(pos).cuda(),
                                        interleaved=interleaved)
    with pytest.raises(errors.Cuda, match="code 3"):
        ops.device_status(0)
    got = to_np(dx).reshape(x3.shape)
    assert np.all(got[lost, :H + K] == 0)
    assert rel_err(got[keep, :H], rq) <= tol and rel_err(got[keep, H:H + K], rk) <= tol
    assert np.array_equal(got[:, H + K:], want_dv)
    if gains:
        assert rel_err(to_np(dgq), rgq) <= tol and rel_err(to_np(dgk), rgk) <= tol
