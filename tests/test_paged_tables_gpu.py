"""Tables of a paged cache that do not describe a batch."""
import numpy as np
import pytest

from helpers import as_bf16, normal, to_dev, to_np
from test_paged_gpu import Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt,hint", [("bf16", 1), ("bf16", 4096), ("f32", 0)])
@pytest.mark.parametrize("cu", [[0, 4, 2, 6], [6, 0, 3, 6], [0, 6, 0, 6], [0, 6, 6, 5], [0, -(1 << 31), 3, 6]])
def test_offsets_that_decrease_are_not_followed(cu, dt, hint):
    """Sequences would overlap: nothing is computed, the fault is recorded, and the next call is right."""
    import torch
    from beacon_b200 import errors, ops
    c = Case([1, 3, 2], [300, 40, 129], 4, 2, 64, 16, dt)
    want = c.run(max_q=hint)
    assert ops.device_status(0)[0] == 0
    bad = torch.tensor(cu, dtype=torch.int32, device="cuda")
    out, lse = torch.full_like(want[0], 7.0), torch.full_like(want[1], 7.0)
    ops.paged_attention(c.dq, c.dk, c.dv, c.pt, bad, c.kv, max_q=hint, out=out, lse=lse)
    with pytest.raises(errors.Cuda, match="code 3"):
        ops.device_status(0)
    assert (out == 7).all() and (lse == 7).all()
    again = c.run(max_q=hint)
    assert torch.equal(again[0], want[0]) and torch.equal(again[1], want[1])
    assert ops.device_status(0)[0] == 0


def test_many_sequences_one_of_them_decreasing():
    """Beyond the 32 sequences that a warp looks at in one step."""
    import torch
    from beacon_b200 import errors, ops
    n = 100
    c = Case([1] * n, [(13 * i) % 60 + 1 for i in range(n)], 4, 2, 64, 16, "bf16")
    bad = c.cu.clone()
    bad[90] = 3
    out = torch.full_like(c.dq, 7.0)
    ops.paged_attention(c.dq, c.dk, c.dv, c.pt, bad, c.kv, max_q=1, out=out)
    with pytest.raises(errors.Cuda, match="code 3"):
        ops.device_status(0)
    assert (out == 7).all()


@pytest.mark.parametrize("D", [64, 40])
def test_append_writes_only_tokens_of_a_place(D):
    """With offsets that decrease, a token that lies outside its sequence's range goes nowhere."""
    import torch
    from beacon_b200 import errors, ops
    c = Case([2, 2, 2], [40, 20, 33], 2, 1, D, 16, "bf16")
    x = to_dev(as_bf16(normal((6, 4 * D), 3)), torch.bfloat16)
    bad = torch.tensor([0, 2, 1, 6], dtype=torch.int32, device="cuda")
    kc, vc = c.dk.clone(), c.dv.clone()
    ops.device_status(0)
    q = torch.full((6, 2, D), 7.0, dtype=torch.bfloat16, device="cuda")
    ops.qk_norm_rope_append(x, None, None, None, kc, vc, c.pt.clamp(min=0), bad, c.kv, 2, q=q)
    # every token has one owner at most: a token's value row stands in one slot at most
    got = to_np(vc).reshape(-1, D)
    rows = to_np(x)[:, 3 * D:]
    for t in range(6):
        assert (got == rows[t]).all(1).sum() <= 1
    # and nothing was written beyond a sequence's own tokens
    for s, n in enumerate(c.kv_lens):
        for j in range(n, c.page * -(-n // c.page)):
            assert np.isnan(to_np(vc)[c.table[s, j // 16], 0, j % 16]).all()
    try:
        ops.device_status(0)
    except errors.Cuda as e:
        assert "code 3" in str(e)
