"""Argument checks of the routing and block-scaled fp8 entry points, and the C
ABI's refusals that return before any launch.  No GPU."""
import ctypes as C

import pytest
import torch

from spider_web_moe_b200 import _lib as L
from spider_web_moe_b200.fp8_blocks import (Fp8BlockExperts, Fp8BlockTensor, fp8_block_linear, fp8_block_matmul,
                                            quantize_fp8_blocks)
from spider_web_moe_b200.routing import route_experts


def fp8(r, c, block_rows=1, lead=()):
    q = torch.zeros(*lead, r, -(-c // 16) * 16, dtype=torch.float8_e4m3fn)[..., :c]
    return Fp8BlockTensor(q, torch.ones(*lead, -(-r // block_rows), -(-c // 128)), block_rows)


@pytest.mark.parametrize("kw,err", [
    (dict(top_k=0), ValueError), (dict(top_k=9), ValueError), (dict(top_k=2, score="tanh"), ValueError),
    (dict(top_k=2, group_score="mean"), ValueError), (dict(top_k=2, num_groups=3), ValueError),
    (dict(top_k=3, num_groups=4, topk_groups=1), ValueError), (dict(top_k=2, num_groups=4, topk_groups=5), ValueError),
    (dict(top_k=2, bias=torch.zeros(7)), ValueError), (dict(top_k=2), RuntimeError),  # the last one: CPU tensors
])
def test_route_experts_refusals(kw, err):
    with pytest.raises(err):
        route_experts(torch.zeros(4, 8), **kw)


def test_route_experts_refuses_types_and_sizes():
    with pytest.raises(TypeError):
        route_experts(torch.zeros(4, 8, dtype=torch.float16), 2)
    with pytest.raises(ValueError):
        route_experts(torch.zeros(4, 1025), 2)
    with pytest.raises(ValueError):
        route_experts(torch.zeros(4, 64), 33)


def test_fp8_tensor_refusals():
    with pytest.raises(ValueError):  # row pitch not a multiple of 16 bytes
        Fp8BlockTensor(torch.zeros(4, 40, dtype=torch.float8_e4m3fn), torch.ones(4, 1), 1)
    with pytest.raises(ValueError):  # scales of another block shape
        Fp8BlockTensor(torch.zeros(256, 256, dtype=torch.float8_e4m3fn), torch.ones(256, 2), 128)
    with pytest.raises(ValueError):
        Fp8BlockTensor(torch.zeros(4, 32, dtype=torch.float8_e4m3fn), torch.ones(4, 1), 64)
    with pytest.raises(TypeError):
        Fp8BlockTensor(torch.zeros(4, 32, dtype=torch.float8_e5m2), torch.ones(4, 1), 1)
    with pytest.raises(TypeError):
        Fp8BlockTensor(torch.zeros(4, 32, dtype=torch.float8_e4m3fn), torch.ones(4, 1).half(), 1)
    with pytest.raises(ValueError):
        fp8(4, 32).transpose()


def test_quantize_and_product_refusals():
    with pytest.raises(TypeError):
        quantize_fp8_blocks(torch.zeros(4, 4, dtype=torch.float16))
    with pytest.raises(ValueError):
        quantize_fp8_blocks(torch.zeros(4))
    with pytest.raises(ValueError):
        quantize_fp8_blocks(torch.zeros(4, 4), 64)
    with pytest.raises(RuntimeError):
        quantize_fp8_blocks(torch.zeros(4, 4))
    with pytest.raises(ValueError):
        fp8_block_matmul(fp8(4, 32), fp8(4, 48))
    with pytest.raises(ValueError):
        fp8_block_matmul(fp8(4, 32, 128), fp8(4, 32, 128))
    with pytest.raises(TypeError):
        fp8_block_matmul(fp8(4, 32), fp8(4, 32, 128), torch.float16)
    with pytest.raises(ValueError):
        fp8_block_matmul(fp8(4, 32), fp8(4, 32, 128), out=torch.zeros(4, 5))
    with pytest.raises(RuntimeError):
        fp8_block_matmul(fp8(4, 32), fp8(4, 32, 128))
    with pytest.raises(ValueError):
        fp8_block_linear(torch.zeros(4, 32), torch.zeros(8, 33))
    with pytest.raises(ValueError):
        fp8_block_linear(torch.zeros(4, 32), fp8(8, 32, 1))
    with pytest.raises(TypeError):
        fp8_block_linear(torch.zeros(4, 32), torch.zeros(8, 32, dtype=torch.float16))
    with pytest.raises(RuntimeError):
        fp8_block_linear(torch.zeros(4, 32), torch.zeros(8, 32))


def test_expert_packing_refusals():
    up, down = fp8(40, 64, 128, (3,)), fp8(64, 40, 128, (3,))
    with pytest.raises(ValueError):
        Fp8BlockExperts(up, None, up, None)  # w_down must be [E, H, U]
    with pytest.raises(ValueError):
        Fp8BlockExperts(up, None, down, None, None, torch.zeros(3, 40))
    with pytest.raises(ValueError):
        Fp8BlockExperts(up, None, down, None, down)
    with pytest.raises(ValueError):
        Fp8BlockExperts(fp8(40, 64, 1, (3,)), None, down, None)
    with pytest.raises(RuntimeError):
        Fp8BlockExperts(up, None, down, None)


def test_c_abi_refuses_before_any_launch():
    lib = L.load()
    p = 4096  # a non-null, 16-byte aligned address that is never dereferenced
    r = lambda **k: lib.sb_route_experts(  # noqa: E731
        k.get("logits", p), k.get("dtype", 0), k.get("ld", 8), 4, 8, k.get("k", 2), k.get("score", 0), None,
        k.get("groups", 1), k.get("tg", 1), k.get("gt", 2), 1, 1.0, p, p, None)
    for bad in (dict(logits=None), dict(dtype=2), dict(ld=7), dict(k=9), dict(k=0), dict(score=2), dict(groups=3),
                dict(groups=4, tg=5), dict(groups=4, tg=1, k=3), dict(gt=3)):
        assert r(**bad) == L.SB_ERR_ARG, bad
    assert lib.sb_route_experts_backward(None, 0, 8, 4, 8, 2, 0, None, 1, 1.0, p, p, p, 8, None) == L.SB_ERR_ARG
    assert lib.sb_route_experts_backward(p, 0, 8, 4, 8, 2, 0, None, 1, 1.0, p, p, p, 7, None) == L.SB_ERR_ARG

    def q(**k):
        a = dict(x=p, dtype=0, block_rows=1, batch=1, rows=4, cols=8, x_row=8, x_col=1, q=p, ldq=16, scale=p)
        a.update(k)
        return lib.sb_fp8_quantize_blocks(C.byref(L.Fp8QuantizeArgs(**a)), None)
    for bad in (dict(x=None), dict(dtype=3), dict(block_rows=2), dict(ldq=17), dict(ldq=0), dict(q=p + 8),
                dict(scale=None), dict(rows=-1), dict(row_index=p, block_rows=128), dict(row_index=p, batch=2)):
        assert q(**bad) == L.SB_ERR_ARG, bad
    assert q(rows=0, x=None) == L.SB_OK
    assert lib.sb_fp8_quantize_blocks(None, None) == L.SB_ERR_ARG

    def m(**k):
        a = dict(epilogue=L.SB_EPI_LINEAR, out_dtype=0, num_groups=1, max_rows=4, n=8, k=32, a=p, lda=32, a_scale=p,
                 b=p, ldb=32, b_scale=p, b_block_rows=128, out=p, ldo=8)
        a.update(k)
        return lib.sb_fp8_matmul(C.byref(L.Fp8MatmulArgs(**a)), None)
    for bad in (dict(a=None), dict(a=p + 4), dict(lda=40), dict(ldb=16), dict(b_block_rows=64), dict(n=0), dict(k=0),
                dict(ldo=7), dict(num_groups=2), dict(num_groups=1025, offsets=p), dict(epilogue=L.SB_EPI_SWIGLU_IL),
                dict(epilogue=L.SB_EPI_GELU, ldo=16, out_scale=None), dict(epilogue=L.SB_EPI_GELU, ldo=8, out_scale=p),
                dict(epilogue=L.SB_EPI_SWIGLU, ldo=16, out_scale=p), dict(out_dtype=2), dict(max_rows=-1),
                dict(num_groups=2, offsets=p, b_group_rows=7), dict(epilogue=L.SB_EPI_GELU, ldo=16, out_scale=p,
                                                                    b_block_rows=1)):
        assert m(**bad) == L.SB_ERR_ARG, bad
    assert m(max_rows=0, a=None) == L.SB_OK

    e = L.Fp8Experts(num_experts=4, hidden=64, ffn=32, activation=L.SB_ACT_GELU, ld_in=64, ld_ffn=32)
    need = lib.sb_fp8_expert_delta_workspace_bytes(C.byref(e), 5, 2)
    assert need > 0
    assert lib.sb_fp8_expert_delta_workspace_bytes(C.byref(e), 5, 65) == 0
    e.ld_in = 60
    assert lib.sb_fp8_expert_delta_workspace_bytes(C.byref(e), 5, 2) == 0
    e.ld_in = 64
    call = lambda ws, n: lib.sb_fp8_expert_delta(C.byref(e), p, 0, 64, p, p, 5, 2, p, 0, None, ws, n, None)  # noqa: E731
    assert call(p, need) == L.SB_ERR_ARG  # no weights
    for f in ("w_up", "s_up", "w_down", "s_down"):
        setattr(e, f, p)
    assert call(p, need - 256) == L.SB_ERR_WORKSPACE
    assert call(None, need) == L.SB_ERR_WORKSPACE

    assert lib.sb_fp8_linear_workspace_bytes(4, 8, 0, 0) == 0
    need = lib.sb_fp8_linear_workspace_bytes(4, 8, 32, 0)
    assert need > lib.sb_fp8_linear_workspace_bytes(4, 8, 32, 1) > 0
    lin = lambda x=p, dt=0, ld=32, wd=0, ldw=32, w=p, ws=p, n=need: lib.sb_fp8_linear(  # noqa: E731
        x, dt, ld, 4, 8, 32, w, wd, ldw, None, 0, 0, p, None, ws, n, None)
    assert lin(x=None) == lin(dt=2) == lin(ld=31) == lin(wd=3) == lin(ldw=31) == lin(w=None) == L.SB_ERR_ARG
    assert lin(ws=None) == lin(n=64) == L.SB_ERR_WORKSPACE
    need = lib.sb_fp8_linear_backward_workspace_bytes(4, 8, 32)
    back = lambda x=p, w=p, dy=p, dr=8, n=need: lib.sb_fp8_linear_backward(  # noqa: E731
        x, 0, 32, 4, 8, 32, w, 0, 32, dy, dr, 1, p, p, None, p, n, None)
    assert back(x=None) == back(w=None) == back(dy=None) == back(dr=-1) == L.SB_ERR_ARG
    assert back(n=64) == L.SB_ERR_WORKSPACE


def test_layer_refuses_other_block_sizes():
    from spider_web_moe_b200 import ModelConfig, SpiderMoELayer

    kw = dict(hidden_size=64, num_heads=4, num_experts=4, top_k=2, edges_per_expert=2, num_loops=2, expert_ffn_size=128)
    with pytest.raises(ValueError):
        SpiderMoELayer(ModelConfig(**kw)).quantize_experts_fp8(block_size=64)
    with pytest.raises(ValueError):
        SpiderMoELayer(ModelConfig(**kw, offload_experts=True)).quantize_experts_fp8(block_size=128)
