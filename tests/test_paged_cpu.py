"""Refusals of the rotation and paged-cache entry points: answered on the host, before any device call."""
import ctypes

import pytest

from beacon_b200 import _lib

_BUF = ctypes.create_string_buffer(1 << 16)
H = (ctypes.addressof(_BUF) + 255) & ~255  # never dereferenced

FWD = dict(q=H, k=H, v=H, qkv=H, ld=512, qg=H, kg=H, table=H, rows=16, pos=None, batch=1, seq=16, heads=4, kv=2, D=64,
           rot=64, inter=0, eps=1e-5, dtype=_lib.BF16, stream=None)
BWD = dict(dqkv=H, ldo=512, dqg=H, dkg=H, dq=H, dk=H, dv=H, qkv=H, ld=512, qg=H, kg=H, table=H, rows=16, pos=None,
           batch=1, seq=16, heads=4, kv=2, D=64, rot=64, inter=0, eps=1e-5, dtype=_lib.BF16, ws=None, wsb=0,
           stream=None)
PAGES = dict(max_pages=4, table_stride=4, num_pages=9, page=16, page_stride=2 * 16 * 64, head_stride=16 * 64,
             token_stride=64)
APPEND = dict(q=H, kc=H, vc=H, qkv=H, ld=512, qg=H, kg=H, table=H, rows=16, pos=None, cu=H, kv_lens=H, pt=H, tokens=3,
              seqs=2, **PAGES, heads=4, kv=2, D=64, rot=64, inter=0, eps=1e-5, dtype=_lib.BF16, stream=None)
ATTN = dict(out=H, lse=H, q=H, qs=256, kc=H, vc=H, cu=H, kv_lens=H, pt=H, tokens=3, seqs=2, max_q=0, **PAGES, heads=4,
            kv=2, D=64, causal=1, dtype=_lib.BF16, ws=None, wsb=0, stream=None)
BLOCK = dict(out=H, x=H, attn_norm=H, w_qkv=H, qg=H, kg=H, w_o=H, ffn_norm=H, w_gate=H, w_up=H, w_down=H, table=H,
             rows=16, rot=64, inter=0, kc=H, vc=H, cu=H, kv_lens=H, pt=H, tokens=3, seqs=2, max_q=0, **PAGES, dm=128,
             heads=4, kv=2, D=64, F=256, eps=1e-5, dtype=_lib.BF16, ws=None, wsb=0, stream=None)
ENTRY = dict(block=("beacon_llama_block_paged_fwd", BLOCK), fwd=("beacon_qk_norm_rope_fwd", FWD), bwd=("beacon_qk_norm_rope_bwd", BWD),
             append=("beacon_qk_norm_rope_append", APPEND), attn=("beacon_paged_attention_fwd", ATTN))

INV, SHAPE, UNIMPL = _lib.ERR_INVALID_LAUNCH_CONFIG, _lib.ERR_SHAPE_MISMATCH, _lib.ERR_UNIMPLEMENTED


def call(which, **change):
    name, args = ENTRY[which]
    assert not set(change) - set(args)
    return getattr(_lib.lib(), name)(*{**args, **change}.values())


NULLS = dict(fwd=("q", "k", "qkv", "table"), bwd=("dqkv", "dq", "dk", "qkv", "table"),
             append=("q", "kc", "vc", "qkv", "table", "cu", "kv_lens", "pt"),
             attn=("out", "q", "kc", "vc", "cu", "kv_lens", "pt"),
             block=("out", "x", "attn_norm", "w_qkv", "w_o", "ffn_norm", "w_gate", "w_up", "w_down", "table", "kc", "vc",
                    "cu", "kv_lens", "pt"))


@pytest.mark.parametrize("which,arg", [(w, a) for w, args in NULLS.items() for a in args])
def test_null_pointers(which, arg):
    assert call(which, **{arg: None}) == INV
    assert "null pointer" in _lib.last_error()


@pytest.mark.parametrize("which,change,status", [
    ("fwd", dict(dtype=_lib.F16), UNIMPL), ("fwd", dict(D=258, rot=0), UNIMPL), ("fwd", dict(D=0), UNIMPL),
    ("fwd", dict(heads=3), SHAPE), ("fwd", dict(rot=63), SHAPE), ("fwd", dict(rot=66), SHAPE),
    ("fwd", dict(rot=-2), SHAPE), ("fwd", dict(ld=511), SHAPE), ("fwd", dict(seq=-1), INV), ("fwd", dict(batch=-1), INV),
    ("fwd", dict(kv=0), INV), ("fwd", dict(batch=1 << 50, seq=1 << 20), INV),
    ("bwd", dict(dtype=7), UNIMPL), ("bwd", dict(ldo=500), SHAPE), ("bwd", dict(qg=None), INV),
    ("bwd", dict(kg=None), INV), ("bwd", dict(heads=5), SHAPE),
    ("append", dict(tokens=-1), INV), ("append", dict(page=0), INV), ("append", dict(table_stride=3), SHAPE),
    ("append", dict(token_stride=63), SHAPE), ("append", dict(head_stride=32), SHAPE),
    ("append", dict(page_stride=8), SHAPE), ("append", dict(dtype=_lib.FP8E4M3), UNIMPL),
    ("append", dict(num_pages=1 << 31), INV), ("append", dict(max_pages=1 << 30, table_stride=1 << 30), INV),
    ("attn", dict(dtype=_lib.F16), UNIMPL), ("attn", dict(D=48, head_stride=768), UNIMPL), ("attn", dict(heads=5), SHAPE),
    ("attn", dict(qs=255), SHAPE), ("attn", dict(seqs=-1), INV), ("attn", dict(tokens=-1), INV),
    ("attn", dict(max_q=-1), INV), ("attn", dict(page=-16), INV), ("attn", dict(page_stride=-5), SHAPE),
    ("attn", dict(kv=0), INV), ("attn", dict(tokens=1 << 31), INV),
    ("block", dict(dtype=_lib.F32), UNIMPL), ("block", dict(D=32, rot=32), UNIMPL), ("block", dict(heads=5), SHAPE),
    ("block", dict(dm=100), INV), ("block", dict(x=H + 2), INV), ("block", dict(page=0), INV),
    ("block", dict(table_stride=1), SHAPE), ("block", dict(rot=33), SHAPE), ("block", dict(tokens=-1), INV),
])
def test_refusals(which, change, status):
    assert call(which, **change) == status, _lib.last_error()
    assert _lib.last_error()


def test_nothing_to_do_needs_no_device():
    for which, change in (("fwd", dict(batch=0)), ("fwd", dict(seq=0)), ("append", dict(tokens=0)),
                          ("append", dict(seqs=0)), ("block", dict(tokens=0)), ("attn", dict(tokens=0)), ("attn", dict(seqs=0))):
        assert call(which, **change) == _lib.OK, _lib.last_error()


def test_table_and_workspace_sizes():
    L = _lib.lib()
    assert L.beacon_rope_table(None, 4, 64, 1e4, None) == INV
    for positions, rot, theta in ((-1, 64, 1e4), (4, 3, 1e4), (4, 64, 0.0), (4, 512, 1e4), (4, 64, float("nan"))):
        assert L.beacon_rope_table(H, positions, rot, theta, None) == INV
    assert L.beacon_rope_table(None, 0, 64, 1e4, None) == _lib.OK
    assert L.beacon_paged_attention_workspace_size(128, _lib.BF16) > 0
    assert L.beacon_paged_attention_workspace_size(0, _lib.BF16) == 0
    assert L.beacon_llama_block_paged_workspace_size(64, 4096, 32, 8, 128, 14336, _lib.BF16) > 64 * 14336 * 2
    assert L.beacon_llama_block_paged_workspace_size(64, 4096, 32, 8, 96, 14336, _lib.BF16) == 0
    assert L.beacon_qk_norm_rope_bwd_workspace_size(128) >= 148 * 2 * 128 * 4
    assert L.beacon_qk_norm_rope_bwd_workspace_size(0) == 0


def test_front_end_refuses_cpu_and_misshapen_tensors():
    import torch
    from beacon_b200 import errors, ops
    bf = torch.bfloat16
    x, g = torch.zeros(4, 8 * 64, dtype=bf), torch.ones(64, dtype=bf)
    c = torch.zeros(3, 2, 16, 64, dtype=bf)
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    with pytest.raises(errors.InvalidLaunchConfig):
        ops.qk_norm_rope_fwd(x, g, g, None, 1, 4, 4, 2)
    with pytest.raises(errors.InvalidLaunchConfig):
        ops.qk_norm_rope_fwd(x, g, g, None, 1, 5, 4, 2)
    with pytest.raises(errors.InvalidLaunchConfig):
        ops.qk_norm_rope_bwd(torch.zeros(1, 4, 4, 64), torch.zeros(1, 2, 4, 64), torch.zeros(1, 2, 5, 64), x, g, g, None)
    with pytest.raises(errors.InvalidLaunchConfig):
        ops.qk_norm_rope_append(x, g, g, None, c, c, i32(1, 2), i32(2), i32(1), 4)
    with pytest.raises(errors.InvalidLaunchConfig):
        ops.paged_attention(torch.zeros(4, 4, 64, dtype=bf), c, c[:, :, :8], i32(1, 2), i32(2), i32(1))
