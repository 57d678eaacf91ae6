"""NaN and infinity that attention over a paged cache sees: they stay in the rows that see them, and never
turn into numbers.  A row that sees a score of NaN or +inf, or scores of -inf only, has out = NaN and
lse = NaN, +inf, -inf; every other row keeps the bits that it has without them."""
import numpy as np
import pytest

import paged_ref as R
from test_paged_gpu import LSE_TOL, Case

pytestmark = pytest.mark.gpu

# (dtype, head_dim, largest number of new tokens that the kernel choice is told): the decode kernel, the
# tensor-core kernel, the exact kernel with either kind of copies
KERNELS = [("bf16", 64, 1), ("bf16", 128, 1), ("bf16", 64, 4096), ("bf16", 128, 4096), ("bf16", 32, 0), ("f32", 64, 0),
           ("f32", 128, 0)]
# items of one piece, of short and full rows; items split over two pieces; over many
LENGTHS = {
    "whole": ([1, 3, 40], [100, 130, 200]),
    "two pieces": ([130, 60, 200, 64, 128, 65], [1900, 1100, 1280, 1663, 1409, 1153]),
    "many pieces": ([2, 1], [9000, 7000]),
}


def _case(lengths, dt, D, seed=2):
    H, K = (16, 8) if lengths == "two pieces" else (8, 2)
    return Case(*LENGTHS[lengths], H, K, D, 16, dt, seed=seed)


def _rows_that_see(c, s, key):
    """Whether each token of the batch sees key `key` of sequence s."""
    first = sum(c.q_lens[:s])
    at = np.arange(c.T) - first + c.kv_lens[s] - c.q_lens[s]
    mine = (np.arange(c.T) >= first) & (np.arange(c.T) < first + c.q_lens[s])
    return mine & (at >= key)


def _same_elsewhere(got, want, hit):
    """hit [T, H]: rows that must be NaN in out; the others keep their bits."""
    import torch
    hit = torch.from_numpy(hit).cuda()
    assert got[0][hit].isnan().all()
    assert torch.equal(got[0][~hit], want[0][~hit]) and torch.equal(got[1][~hit], want[1][~hit])
    return got[1][hit]


@pytest.mark.parametrize("lengths", LENGTHS)
@pytest.mark.parametrize("dt,D,hint", KERNELS)
@pytest.mark.parametrize("whole_row", [True, False])
def test_nan_in_a_query(dt, D, hint, lengths, whole_row):
    from beacon_b200 import ops
    c = _case(lengths, dt, D)
    want = c.run(max_q=hint)
    hit = np.zeros((c.T, c.H), dtype=bool)
    for t, h in ((0, 1), (c.T - 1, c.H - 1), (c.T // 2, 0)):
        c.dq[t, h, slice(None) if whole_row else D - 1] = float("nan")
        hit[t, h] = True
    lse = _same_elsewhere(c.run(max_q=hint), want, hit)
    assert lse.isnan().all()
    assert ops.device_status(0)[0] == 0


@pytest.mark.parametrize("lengths", LENGTHS)
@pytest.mark.parametrize("dt,D,hint", KERNELS)
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_a_key_that_makes_a_score_nan_or_infinite(dt, D, hint, lengths, value):
    """The first, the last and some key between, of every KV head in turn."""
    c = _case(lengths, dt, D)
    c.dq[:, :, 0] = 1.0  # an infinite key element gives an infinite score
    want = c.run(max_q=hint)
    clean = c.dk.clone()
    for s in range(len(c.q_lens)):
        for i, key in enumerate((0, 77 % c.kv_lens[s], c.kv_lens[s] // 2, c.kv_lens[s] - 1)):
            kvh = i % c.K
            c.dk.copy_(clean)
            c.dk[c.table[s, key // 16], kvh, key % 16, 0] = value
            hit = np.zeros((c.T, c.H), dtype=bool)
            hit[_rows_that_see(c, s, key), kvh * c.H // c.K:(kvh + 1) * c.H // c.K] = True
            lse = _same_elsewhere(c.run(max_q=hint), want, hit)
            assert (lse.isnan() if value != value else lse == value).all()


@pytest.mark.parametrize("dt,D,hint", KERNELS)
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_every_column_of_a_key_tile(dt, D, hint, value):
    """Sequence j has its key 128 + j poisoned: each column of a 128-key tile, whichever unit its exponential
    takes."""
    n = 128
    c = Case([1] * n, [300] * n, 4, 1, D, 16, dt, seed=4)
    c.dq[:, :, 0] = 1.0
    for j in range(n):
        key = 128 + j
        c.dk[c.table[j, key // 16], 0, key % 16, 0] = value
    out, lse = c.run(max_q=hint)
    assert out.isnan().all()
    assert (lse.isnan() if value != value else lse == value).all()


@pytest.mark.parametrize("lengths", LENGTHS)
@pytest.mark.parametrize("dt,D,hint", KERNELS)
def test_scores_of_minus_infinity(dt, D, hint, lengths):
    """Some keys at -inf have no weight; only keys at -inf: NaN, lse -inf, and not the empty row's zeros."""
    import torch
    c = _case(lengths, dt, D)
    c.q[:, :, 0] = 1.0
    for s, n in enumerate(c.kv_lens):
        for j in range(0, n, 3):
            c.k[c.table[s, j // 16], :, j % 16, 0] = -np.inf
    c.k[c.table[0, 0], :, 0, 0] = -np.inf
    c.dq.copy_(torch.from_numpy(c.q))
    c.dk.copy_(torch.from_numpy(c.k))
    if lengths == "whole":  # a row of the first sequence's only token has none left
        c.dk[torch.from_numpy(c.table[0, :7]).long().cuda(), :, :, 0] = -float("inf")
        out, lse = c.run(max_q=hint)
        assert out[0].isnan().all() and (lse[0] == -float("inf")).all()
        c.dk.copy_(torch.from_numpy(c.k))
    out, lse = c.run(max_q=hint)
    if lengths != "two pieces":
        c.check(out, lse)
    else:  # the plain form's loops are slow here: some tokens
        assert out.isfinite().all() and lse.isfinite().all()
        for t in (0, 129, 130, 189, c.T - 1):
            s = int(np.searchsorted(np.cumsum(c.q_lens), t, side="right"))
            seen = c.kv_lens[s] - c.q_lens[s] + t - sum(c.q_lens[:s]) + 1
            ref, rl = R.paged_attention(c.q[t:t + 1], c.k, c.v, c.table[s:s + 1], [1], [seen])
            assert np.linalg.norm(out[t].float().cpu().numpy() - ref[0]) <= 4 * c.tol * np.linalg.norm(ref[0])
            assert np.abs(lse[t].cpu().numpy() - rl[0]).max() <= LSE_TOL


@pytest.mark.parametrize("dt,D,hint", KERNELS)
@pytest.mark.parametrize("key", [0, 4500])
def test_minus_infinity_only_in_split_work(dt, D, hint, key):
    """Every key of a long sequence at -inf: NaN and -inf; one key of it finite: that key's value."""
    import torch
    c = Case([2], [9000], 4, 1, D, 16, dt, seed=6)
    c.dq[:, :, 0] = 1.0
    pages = torch.from_numpy(c.table[0, :-1]).long().cuda()
    finite = c.dk[pages[key // 16], 0, key % 16].clone()
    c.dk[pages, :, :, 0] = -float("inf")
    out, lse = c.run(max_q=hint)
    assert out.isnan().all() and (lse == -float("inf")).all()
    c.dk[pages[key // 16], 0, key % 16] = finite
    out, lse = c.run(max_q=hint)
    assert torch.equal(out, c.dv[pages[key // 16], 0, key % 16].expand_as(out).contiguous())
    assert lse.isfinite().all()
