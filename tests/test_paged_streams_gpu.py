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


def _graph(fn):
    import torch
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = fn()
    return graph, out


@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_captured_default_calls_outlive_larger_ones(dt):
    """Attention and the rotation's backward captured without a workspace given, then eager calls that need far
    more scratch, from the library and from the allocator: replays give the same bits."""
    import torch
    from beacon_b200 import ops
    c = Case(**{**DECODE, "dt": dt})
    want = c.run(max_q=2)
    c.check(*want)
    B, S, H, K, D = 1, 40, 4, 2, 128
    gen = torch.Generator("cuda").manual_seed(3)
    rnd = lambda *s: torch.randn(*s, generator=gen, device="cuda").to(c.tdt)  # noqa: E731
    bwd = (rnd(B, H, S, D), rnd(B, K, S, D), rnd(B, K, S, D), rnd(B * S, (H + 2 * K) * D), rnd(D), rnd(D),
           ops.rope_table(S, D))
    want_bwd = ops.qk_norm_rope_bwd(*bwd)
    g1, out = _graph(lambda: c.run(max_q=2))
    g2, grads = _graph(lambda: ops.qk_norm_rope_bwd(*bwd))
    x = torch.randn(4096, 1024, device="cuda").bfloat16()  # SwiGLU backward: the library's own buffer grows
    w = [torch.randn(*s, device="cuda").bfloat16() for s in ((1024, 4096), (1024, 4096), (4096, 1024))]
    ops.swiglu_bwd(x, x, *w)
    long = Case([200, 90], [900, 700], 16, 4, 128, 16, "bf16")
    long.run(max_q=200)
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    junk = torch.full((1 << 26,), float("nan"), device="cuda")
    for _ in range(2):
        for t in (*out, *grads):
            t.fill_(9.0)
        g1.replay()
        g2.replay()
        assert all(torch.equal(a, b) for a, b in zip((*out, *grads), (*want, *want_bwd)))
    assert junk.isnan().all()
    del g1, g2
    assert ops.device_status(0)[0] == 0


def _block(T=3):
    import torch
    dm, H, K, D, F = 256, 4, 2, 64, 384
    gen = torch.Generator("cuda").manual_seed(7)
    rnd = lambda *s: (torch.randn(*s, generator=gen, device="cuda") * 0.05).bfloat16()  # noqa: E731
    w = [1 + rnd(dm), rnd(dm, (H + 2 * K) * D), rnd(H * D, dm), 1 + rnd(dm), rnd(dm, F), rnd(dm, F), rnd(F, dm)]
    kc, vc = (rnd(6, K, 16, D) for _ in range(2))
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    return [rnd(T, dm) * 20, *w, kc, vc, i32([[2, 5, 0]]), i32([0, T]), i32([33 + T]), H]


def test_captured_block_without_a_workspace():
    import torch
    from beacon_b200 import ops
    args = _block()
    want = ops.llama_block_paged_fwd(*args)
    graph, out = _graph(lambda: ops.llama_block_paged_fwd(*args))
    x = torch.randn(4096, 1024, device="cuda").bfloat16()
    w = [torch.randn(*s, device="cuda").bfloat16() for s in ((1024, 4096), (1024, 4096), (4096, 1024))]
    ops.swiglu_bwd(x, x, *w)
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    out.zero_()
    graph.replay()
    assert torch.equal(out, want)
    del graph


def test_capture_refuses_the_librarys_buffer():
    """Through the C ABI: NULL on a capturing stream is refused, and the capture goes on."""
    import torch
    from beacon_b200 import _lib
    L = _lib.lib()
    c = Case([1], [40], 4, 2, 64, 16, "bf16")
    out, lse = torch.empty_like(c.dq), torch.empty(1, 4, device="cuda")
    x = torch.zeros(1, 8 * 64, dtype=torch.bfloat16, device="cuda")
    dy = [torch.zeros(1, n, 1, 64, dtype=torch.bfloat16, device="cuda") for n in (4, 2, 2)]
    g, dg = (torch.zeros(64, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    dx = torch.empty_like(x)
    pages, K, page, D = c.dk.shape
    block = _block()
    p = lambda t: t.data_ptr()  # noqa: E731

    def calls(stream):
        paging = (c.pt.shape[1], c.pt.stride(0), pages, page, *c.dk.stride()[:3])
        attn = L.beacon_paged_attention_fwd(p(out), p(lse), p(c.dq), 256, p(c.dk), p(c.dv), p(c.cu), p(c.kv), p(c.pt), 1, 1,
                                            1, *paging, 4, 2, 64, 1, _lib.BF16, None, 0, stream)
        bwd = L.beacon_qk_norm_rope_bwd(p(dx), 512, p(dg), p(dg), p(dy[0]), p(dy[1]), p(dy[2]), p(x), 512, p(g), p(g), None,
                                        0, None, 1, 1, 4, 2, 64, 0, 0, 1e-5, _lib.BF16, None, 0, stream)
        bx, n1, wqkv, wo, n2, wg, wu, wd, kc, vc, pt, cu, kv, H = block
        fwd = L.beacon_llama_block_paged_fwd(
            p(bx.clone()), p(bx), p(n1), p(wqkv), None, None, p(wo), p(n2), p(wg), p(wu), p(wd), None, 0, 0, 0, p(kc), p(vc),
            p(cu), p(kv), p(pt), 3, 1, 0, 3, 3, 6, 16, *kc.stride()[:3], 256, H, 2, 64, 384, 1e-5, _lib.BF16, None, 0, stream)
        return attn, bwd, fwd

    assert calls(torch.cuda.current_stream().cuda_stream) == (_lib.OK,) * 3
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    y = torch.zeros(8, device="cuda")
    with torch.cuda.graph(graph, stream=side):
        got = calls(side.cuda_stream)
        y.add_(1)
    assert got == (_lib.ERR_INVALID_LAUNCH_CONFIG,) * 3 and "workspace of its own" in _lib.last_error()
    graph.replay()
    torch.cuda.synchronize()
    assert (y == 1).all()
    del graph


def test_default_calls_on_two_streams_do_not_share_scratch():
    import torch
    from beacon_b200 import ops
    a, b = Case(**DECODE, seed=3), Case(**CHUNKS, seed=4)
    want = a.run(max_q=2), b.run(max_q=130)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(60):
        for i, (c, hint) in enumerate(((a, 2), (b, 130))):
            with torch.cuda.stream(streams[i]):
                out, lse = c.run(max_q=hint)
                got[i].append(((out == want[i][0]).all() & (lse == want[i][1]).all()).view(1))
    torch.cuda.synchronize()
    assert torch.cat(got[0]).all() and torch.cat(got[1]).all()
    assert ops.device_status(0)[0] == 0
