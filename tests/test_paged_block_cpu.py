"""What the block over a paged cache refuses, it refuses before anything is launched: its attention's
conditions, answered without a device, and operands of ops that the kernels would index wrongly."""
import pytest

from beacon_b200 import _lib
from test_paged_cpu import H, INV, call


@pytest.mark.parametrize("which", ["block", "attn"])
@pytest.mark.parametrize("off", [1, 4, 8, 16])
def test_workspace_that_partial_rows_cannot_be_stored_in(which, off):
    assert call(which, ws=H + off, wsb=1 << 40) == INV
    assert "32-byte aligned" in _lib.last_error()


@pytest.mark.parametrize("change", [dict(max_q=-1), dict(tokens=1 << 20, heads=1 << 12, kv=1 << 12),
                                    dict(tokens=100000, seqs=100000, max_pages=1 << 24, table_stride=1 << 24)])
def test_block_refuses_what_its_attention_refuses(change):
    assert call("block", **change) == INV, _lib.last_error()
    assert "llama_block_paged_fwd" in _lib.last_error()


def _operands():
    import torch
    dm, heads, K, D, F, T = 128, 4, 2, 64, 256, 3
    z = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)  # noqa: E731
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    return dict(x=z(T, dm), attn_norm=z(dm), w_qkv=z(dm, (heads + 2 * K) * D), w_o=z(heads * D, dm), ffn_norm=z(dm),
                w_gate=z(dm, F), w_up=z(dm, F), w_down=z(F, dm), k_cache=z(5, K, 16, D), v_cache=z(5, K, 16, D),
                page_table=i32(1, 2), cu_q=i32(2), kv_lens=i32(1), heads=heads)


@pytest.mark.parametrize("name,shape", [
    ("attn_norm", (64,)), ("ffn_norm", (127,)), ("w_qkv", (128, 256)), ("w_qkv", (64, 512)),
    ("w_o", (128, 128)), ("w_gate", (64, 256)), ("w_up", (128, 255)), ("w_up", (256, 128)), ("w_down", (256, 64)),
    ("w_down", (128, 256)), ("out", (3, 64)), ("out", (2, 128)), ("q_gain", (32,)), ("k_gain", (128,)),
])
def test_block_operands_of_the_wrong_shape(name, shape):
    import torch
    from beacon_b200 import errors, ops
    args = _operands()
    args[name] = torch.zeros(*shape, dtype=torch.bfloat16)
    with pytest.raises(errors.InvalidLaunchConfig, match=name if name != "w_gate" else "is not"):
        ops.llama_block_paged_fwd(**args)


def test_block_operands_of_the_wrong_rank_or_place():
    import torch
    from beacon_b200 import errors, ops
    for name, shape in (("x", (3, 1, 128)), ("k_cache", (5, 16, 64)), ("w_gate", (128,))):
        args = _operands()
        args[name] = torch.zeros(*shape, dtype=torch.bfloat16)
        with pytest.raises(errors.InvalidLaunchConfig):
            ops.llama_block_paged_fwd(**args)
    with pytest.raises(errors.InvalidLaunchConfig, match="CUDA"):
        ops.llama_block_paged_fwd(**_operands())
