"""The combines of at least 512 tokens at every multiple of 128 columns (a warp per
token has code for some of them only), and the calls that end in them."""
import pytest
import torch

from spider_web_moe_b200 import ModelConfig, SpiderMoELayer
from spider_web_moe_b200 import _lib as L
from spider_web_moe_b200.fp8_blocks import check_status, fp8_expert_delta
from spider_web_moe_b200.routing import route_experts

from test_gpu_fp8_blocks import make_experts, rand

pytestmark = pytest.mark.gpu

WIDTHS = [128 * i for i in range(1, 18)] + [132, 1020, 2560, 4096]


def stream():
    return torch.cuda.current_stream().cuda_stream


@pytest.mark.parametrize("cols", WIDTHS)
@pytest.mark.parametrize("n", [511, 513])
def test_rows_and_layernorm(n, cols, cuda_device):
    """Against 64 bits.  A sum of 3 rows: 2 roundings of partial sums below S = sum
    |y|.  LayerNorm: u within 6 * 2^-24 of its parts, the mean and variance within
    (cols / 128 + 12) 2^-24 (additions along a lane's or thread's chunks, then by
    halves); outputs up to about 5, so 2^-14 absolute leaves room for all of it."""
    slots = 3
    y = rand(n * slots, cols, seed=cols).to(cuda_device)
    g = torch.Generator().manual_seed(n)
    inv = torch.randperm(n * slots, generator=g).view(n, slots).int()
    inv[torch.rand(n, slots, generator=g) < 0.2] = -1
    d = inv.to(cuda_device)
    rows = torch.where(d[..., None] >= 0, y[d.clamp_min(0).long()], 0.0).double()
    want, s = rows.sum(1), rows.abs().sum(1)
    out = torch.empty(n, cols, device=cuda_device)
    lib = L.load()
    L.check(lib.sb_combine_rows(y.data_ptr(), cols, 1, 0, d.data_ptr(), slots, n, cols, out.data_ptr(), None, 0, None,
                                L.SB_BF16, stream()), "sb_combine_rows")
    assert ((out.double() - want).abs() <= 2 * 2.0 ** -24 * s).all()
    low = torch.empty(n, cols, device=cuda_device, dtype=torch.bfloat16)
    L.check(lib.sb_combine_rows(y.data_ptr(), cols, 1, 0, d.data_ptr(), slots, n, cols, None, None, 0, low.data_ptr(),
                                L.SB_BF16, stream()), "sb_combine_rows")
    assert torch.equal(low, out.bfloat16())
    h, x0 = rand(n, cols, seed=1).to(cuda_device), rand(n, cols, seed=2).to(cuda_device)
    lw, lb = rand(cols, seed=3).to(cuda_device), rand(cols, seed=4).to(cuda_device)
    got = torch.empty(n, cols, device=cuda_device)
    L.check(lib.sb_combine_ln(y.data_ptr(), cols, 1, 0, d.data_ptr(), slots, None, h.data_ptr(), x0.data_ptr(), L.SB_F32,
                              n, cols, lw.data_ptr(), lb.data_ptr(), 0.5, 0.25, 1e-5, got.data_ptr(), None, stream()),
            "sb_combine_ln")
    u = h.double() + 0.5 * want + 0.25 * x0.double()
    c = u - u.mean(1, keepdim=True)
    ln = c / (c.square().mean(1, keepdim=True) + 1e-5).sqrt() * lw.double() + lb.double()
    assert (got.double() - ln).abs().max() < 2.0 ** -14


@pytest.mark.parametrize("hidden", [384, 640, 766, 1152, 1536, 1661])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_expert_delta_of_many_tokens(hidden, dtype, cuda_device):
    """In one call and in two of fewer than 512 tokens: within an activation's
    rounding of each other, row by row (another schedule may sum in another order)."""
    ex, _ = make_experts(4, hidden, 160, True, hidden, cuda_device)
    x = rand(700, hidden, seed=5, dtype=dtype).to(cuda_device)
    idx, w = route_experts(rand(700, 4, seed=6).to(cuda_device), 2)
    got = fp8_expert_delta(x, idx, w, ex).double()
    want = torch.cat([fp8_expert_delta(x[a:b], idx[a:b], w[a:b], ex) for a, b in ((0, 350), (350, 700))]).double()
    check_status(cuda_device)
    assert ((got - want).norm(dim=1) / want.norm(dim=1)).max() < 2.0 ** -5


@pytest.mark.parametrize("hidden", [384, 768])
@torch.no_grad()
def test_layer_of_many_tokens(hidden, cuda_device):
    """The block in its own formats and in block-scaled fp8, 600 tokens at once and
    in two halves (bf16: two steps of the output)."""
    cfg = ModelConfig(hidden_size=hidden, num_heads=4, num_experts=8, top_k=2, edges_per_expert=2, num_loops=2,
                      expert_ffn_size=256)
    torch.manual_seed(1)
    layer = SpiderMoELayer(cfg).to(cuda_device, torch.bfloat16).eval()
    h, x0 = rand(1, 600, hidden, seed=7).to(cuda_device, torch.bfloat16), rand(1, 600, hidden, seed=8).to(cuda_device, torch.bfloat16)
    for pack in (lambda: None, layer.quantize_experts_fp8, lambda: layer.quantize_experts_fp8(block_size=128)):
        pack()
        got = layer(h, x0, 0).double()
        want = torch.cat([layer(h[:, a:a + 300].contiguous(), x0[:, a:a + 300].contiguous(), 0) for a in (0, 300)], 1).double()
        assert ((got - want).norm(dim=-1) / want.norm(dim=-1)).max() < 2.0 ** -7
