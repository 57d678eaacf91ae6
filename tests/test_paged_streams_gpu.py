"""Calls over a paged cache that overlap, that are captured and replayed, and whose workspace holds anything:
the results are those of the same call alone, bit for bit (split work is joined in a fixed order)."""
import pytest

from test_paged_gpu import Case

pytestmark = pytest.mark.gpu

# 4 sequences over 148 SMs: every item of the decode kernel and most of the tensor-core kernel's are split
DECODE = dict(q_lens=[1, 1, 2, 1], kv_lens=[3000, 2500, 1800, 4000], H=8, K=2, D=128, page=16, dt="bf16")
CHUNKS = dict(q_lens=[70, 130, 40], kv_lens=[1900, 2100, 1500], H=16, K=4, D=128, page=16, dt="bf16")


def _workspace(fill):
    import torch
    from beacon_b200 import ops
    n = ops.paged_attention_workspace_bytes(128)
    if fill == "random":
        return torch.randint(0, 256, (n,), dtype=torch.uint8, device="cuda",
                             generator=torch.Generator("cuda").manual_seed(5))
    return torch.full((n,), fill, dtype=torch.uint8, device="cuda")


@pytest.mark.parametrize("which", [DECODE, CHUNKS])
@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_workspace_contents_do_not_matter(which, dt):
    """Counters of finished pieces among them: a call does not rely on what the workspace held."""
    import torch
    from beacon_b200 import ops
    c = Case(**{**which, "dt": dt})
    first = c.run(max_q=max(c.q_lens))
    c.check(*first)
    for fill in (0, 1, 2, 255, "random"):
        ws = _workspace(fill)
        for _ in range(2):
            out, lse = c.run(max_q=max(c.q_lens), workspace=ws)
            assert torch.equal(out, first[0]) and torch.equal(lse, first[1])
    assert ops.device_status(0)[0] == 0


@pytest.mark.parametrize("beside", ["decode", "chunks", "replay"])
def test_replays_beside_other_calls_of_another_stream(beside):
    """A captured decode step replayed on one stream while calls with a workspace of their own run on
    another, through more launches than any set of counters could hold."""
    import torch
    from beacon_b200 import ops
    a, b = Case(**DECODE, seed=3), Case(**(CHUNKS if beside == "chunks" else DECODE), seed=4)
    want_a, want_b = a.run(max_q=2), b.run(max_q=max(b.q_lens))
    ws_a, ws_b = _workspace("random"), _workspace("random")
    bufs_a, bufs_b = [[torch.empty_like(t) for t in w] for w in (want_a, want_b)]
    sa, sb = torch.cuda.Stream(), torch.cuda.Stream()

    def capture(case, ws, bufs, stream, hint):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            case.run(max_q=hint, out=bufs[0], lse=bufs[1], workspace=ws)
        return graph

    ga = capture(a, ws_a, bufs_a, sa, 2)
    for _ in range(63):  # eager calls between two captures: a rotation of 64 would come back to the same place
        b.run(max_q=max(b.q_lens), out=bufs_b[0], lse=bufs_b[1], workspace=ws_b)
    gb = capture(b, ws_b, bufs_b, sb, max(b.q_lens)) if beside == "replay" else None
    torch.cuda.synchronize()
    bad = torch.zeros(2, dtype=torch.int64, device="cuda")
    one = torch.ones((), dtype=torch.int64, device="cuda")
    torch.cuda.synchronize()
    for _ in range(200):
        with torch.cuda.stream(sa):
            ga.replay()
            bad[0] += torch.where((bufs_a[0] == want_a[0]).all() & (bufs_a[1] == want_a[1]).all(), 0 * one, one)
        with torch.cuda.stream(sb):
            if gb is not None:
                gb.replay()
            else:
                b.run(max_q=max(b.q_lens), out=bufs_b[0], lse=bufs_b[1], workspace=ws_b)
            bad[1] += torch.where((bufs_b[0] == want_b[0]).all() & (bufs_b[1] == want_b[1]).all(), 0 * one, one)
    torch.cuda.synchronize()
    assert bad.tolist() == [0, 0]
    del ga, gb
    assert ops.device_status(0)[0] == 0
