"""Block-scaled fp8 on the GPU: quantisation bit for bit against plain torch
steps; products, the linear layer's gradients and the experts' FFNs against fp64.

Tolerance of a product, with S = sum_k |a_k b_k|: e4m3 products are exact in
fp32; the tensor core adds the 32 of an instruction aligned to the largest of
them with at least 13 fraction bits, so a block of 128 is off by less than 2^-12
of its S; scaling and the running sum over KB blocks add (KB + 4) 2^-24 S, and a
bf16 result its half step, 2^-8 of the value.
"""
import pytest
import torch

from spider_web_moe_b200 import _lib as L
from spider_web_moe_b200 import fp8_blocks as F
from spider_web_moe_b200.fp8_blocks import (Fp8BlockExperts, Fp8BlockTensor, check_status, fp8_block_linear,
                                            fp8_block_matmul, fp8_expert_delta, quantize_fp8_blocks)
from spider_web_moe_b200.routing import route_experts

pytestmark = pytest.mark.gpu


def plain_quantize(x, br):
    """The definition, on the CPU: (bytes, scale)."""
    *lead, r, c = x.shape
    rb, cb = -(-r // br), -(-c // 128)
    xp = torch.nn.functional.pad(x.float(), (0, cb * 128 - c, 0, rb * br - r)).view(*lead, rb, br, cb, 128)
    a = xp.abs().amax(dim=(-3, -1), keepdim=True).clamp_min(2.0 ** -100)
    # not 448.0 / a, which is a reciprocal and a product
    q = (xp * (torch.full_like(a, 448.0) / a)).clamp(-448, 448).to(torch.float8_e4m3fn).view(*lead, rb * br, cb * 128)[..., :r, :c]
    return q.contiguous().view(torch.uint8), (a / 448.0).view(*lead, rb, cb)


def rand(*shape, seed=0, dtype=torch.float32, spread=False):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(*shape, generator=g)
    if spread:  # magnitudes over many octaves: blocks with very different scales
        x = x * torch.exp2(torch.randint(-20, 20, shape, generator=g).float())
    return x.to(dtype)


def bound(a, b, dtype, want):
    kb = -(-a.shape[1] // 128)
    s = a.abs() @ b.abs().t()
    return (2.0 ** -12 + (kb + 4) * 2.0 ** -24) * s + (2.0 ** -8 if dtype == torch.bfloat16 else 0) * want.abs()


def check(got, a, b, what=""):
    want = a @ b.t()
    err = (got.double().cpu() - want).abs()
    tol = bound(a, b, got.dtype, want)
    assert (err <= tol).all(), f"{what}: off by {float((err / tol.clamp_min(1e-300)).max())} tolerances"


QSHAPES = [(1, 1), (1, 128), (5, 127), (130, 129), (17, 1000), (300, 520), (128, 256), (33, 2048), (1000, 40)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("br", [1, 128])
@pytest.mark.parametrize("shape", QSHAPES)
def test_quantize_bits(shape, br, dtype, cuda_device):
    x = rand(*shape, seed=shape[0] + shape[1], dtype=dtype, spread=True)
    for view in (lambda t: t, lambda t: t.t()):
        xv = view(x)
        q = quantize_fp8_blocks(view(x.to(cuda_device)), br)
        wq, ws = plain_quantize(xv, br)
        assert torch.equal(q.scale.cpu(), ws)
        assert torch.equal(q.q.cpu().contiguous().view(torch.uint8), wq)


def test_quantize_strides_stacks_and_values(cuda_device):
    x = rand(3, 70, 200, seed=3, dtype=torch.bfloat16)
    d = x.to(cuda_device)
    views = [lambda t: t, lambda t: t.transpose(1, 2), lambda t: t[:, 1::2, 5:], lambda t: t[:, :, ::3],
             lambda t: t[1:, 3:, :133], lambda t: t.permute(1, 0, 2), lambda t: t[0, :1].expand(9, 200),
             lambda t: t.permute(2, 1, 0)]
    for i, v in enumerate(views):
        for br in (1, 128):
            q = quantize_fp8_blocks(v(d), br)
            wq, ws = plain_quantize(v(x), br)
            assert torch.equal(q.scale.cpu(), ws), (i, br)
            assert torch.equal(q.q.cpu().contiguous().view(torch.uint8), wq), (i, br)
    # zeros, the smallest and largest values, inf and NaN
    x = torch.zeros(6, 300)
    x[1, 5] = 1e-42
    x[2, 130] = 3.3e38
    x[3, 7], x[3, 8] = float("inf"), 1.0
    x[4, 299] = float("nan")
    x[5, :] = 2.0 ** -101
    for br in (1, 128):
        q = quantize_fp8_blocks(x.to(cuda_device), br)
        wq, ws = plain_quantize(x, br)
        finite = torch.isfinite(ws)
        assert torch.equal(torch.isfinite(q.scale.cpu()), finite)
        assert torch.equal(q.scale.cpu()[finite], ws[finite])
        rows = torch.tensor([0, 1, 2, 5]) if br == 1 else torch.tensor([], dtype=torch.long)
        assert torch.equal(q.q.cpu().contiguous().view(torch.uint8)[rows], wq[rows])
        deq = q.dequantize().cpu()
        assert torch.isnan(deq[3, 7]) and torch.isnan(deq[4, 299])
    assert quantize_fp8_blocks(torch.zeros(0, 64, device=cuda_device)).shape == (0, 64)


MM = [(1, 16, 1), (1, 2048, 384), (3, 128, 256), (32, 130, 129), (33, 256, 512), (128, 1024, 128), (129, 64, 257),
      (200, 1000, 300), (257, 2048, 640), (64, 4096, 1000), (512, 16, 2048), (300, 33, 70), (2, 1360, 2056)]


@pytest.mark.parametrize("m,k,n", MM)
@pytest.mark.parametrize("br", [128, 1])
def test_product(m, k, n, br, cuda_device):
    a = quantize_fp8_blocks(rand(m, k, seed=m).to(cuda_device))
    b = quantize_fp8_blocks(rand(n, k, seed=n + 1).to(cuda_device), br)
    ad, bd = a.dequantize().double().cpu(), b.dequantize().double().cpu()
    for dtype in (torch.float32, torch.bfloat16):
        got = fp8_block_matmul(a, b, dtype)
        assert got.dtype == dtype and got.shape == (m, n)
        check(got, ad, bd, f"{dtype}")
        assert torch.equal(got, fp8_block_matmul(a, b, dtype))  # no order of additions is left open
    check_status(cuda_device)


# more 128 x 64 items than SMs: tiles of 128 rows (up to 128 rows) and of CTA pairs
TILES = [(100, 160, 9700), (33 + 64, 2048, 9601), (257, 200, 4000), (700, 130, 2056), (513, 1040, 3900), (1029, 16, 1300)]


@pytest.mark.parametrize("m,k,n", TILES)
@pytest.mark.parametrize("br", [128, 1])
def test_product_row_tiles(m, k, n, br, cuda_device):
    a = quantize_fp8_blocks(rand(m, k, seed=m).to(cuda_device))
    b = quantize_fp8_blocks(rand(n, k, seed=n + 1).to(cuda_device), br)
    ad, bd = a.dequantize().double().cpu(), b.dequantize().double().cpu()
    for dtype in (torch.float32, torch.bfloat16):
        got = fp8_block_matmul(a, b, dtype)
        check(got, ad, bd, f"{dtype}")
        for off in (11, 16):  # an output that bulk stores cannot address, and one that they can
            big = torch.full((m + 9, n + 40), 7.0, device=cuda_device, dtype=dtype)
            fp8_block_matmul(a, b, out=big[5:m + 5, off:n + off])
            assert torch.equal(big[5:m + 5, off:n + off], got)
            big[5:m + 5, off:n + off] = 7
            assert (big == 7).all()
    check_status(cuda_device)


def test_product_long_k_and_one_row(cuda_device):
    """128 blocks of k split over a cluster, and one block in a problem that could be split."""
    for m, k, n in ((1, 16384, 256), (1, 128, 128), (3, 40000, 130), (16, 17000, 1)):
        a = quantize_fp8_blocks(rand(m, k, seed=m).to(cuda_device))
        b = quantize_fp8_blocks(rand(n, k, seed=n + 1).to(cuda_device), 128)
        check(fp8_block_matmul(a, b, torch.float32), a.dequantize().double().cpu(), b.dequantize().double().cpu())


def test_product_rows_do_not_mix(cuda_device):
    """A NaN row and rows of very different size leave the others as they were."""
    x = rand(140, 256, seed=8)
    x[7] = float("nan")
    x[100] *= 1e30
    b = quantize_fp8_blocks(rand(200, 256, seed=9).to(cuda_device), 128)
    got = fp8_block_matmul(quantize_fp8_blocks(x.to(cuda_device)), b, torch.float32)
    clean = x.clone()
    clean[7] = 0
    want = fp8_block_matmul(quantize_fp8_blocks(clean.to(cuda_device)), b, torch.float32)
    assert torch.isnan(got[7]).all()
    keep = torch.arange(140) != 7
    assert torch.equal(got[keep], want[keep])


def test_product_strides(cuda_device):
    a = quantize_fp8_blocks(rand(70, 300, seed=1).to(cuda_device))
    b = quantize_fp8_blocks(rand(300, 300, seed=2).to(cuda_device), 128)
    want = fp8_block_matmul(a, b, torch.float32)
    # scales and values with other pitches, a transposed copy, an output inside a larger tensor
    q2 = torch.zeros(70, 512, dtype=torch.uint8, device=cuda_device)
    q2[:, :300] = a.q.contiguous().view(torch.uint8)
    a2 = Fp8BlockTensor(q2.view(torch.float8_e4m3fn)[:, :300], a.scale.contiguous(), 1)
    b2 = b.transpose().transpose()
    big = torch.full((80, 333), 7.0, device=cuda_device)
    fp8_block_matmul(a2, b2, out=big[5:75, 11:311])
    assert torch.equal(big[5:75, 11:311], want)
    mask = torch.ones_like(big, dtype=torch.bool)
    mask[5:75, 11:311] = False
    assert (big[mask] == 7).all()
    assert torch.equal(b.transpose().dequantize(), b.dequantize().t())


def grouped(epi, e, u, h, counts, seed, device):
    """sb_fp8_matmul by groups through the C ABI; returns everything a check needs."""
    counts = torch.tensor(counts)
    total, cap = int(counts.sum()), int(counts.sum()) + 5
    off = torch.cat([torch.zeros(1, dtype=torch.long), counts.cumsum(0)]).int().to(device)
    x = quantize_fp8_blocks(rand(cap, h, seed=seed).to(device))
    up = quantize_fp8_blocks((rand(e, u, h, seed=seed + 1) * h ** -0.5).to(device), 128)
    gate = quantize_fp8_blocks((rand(e, u, h, seed=seed + 2) * h ** -0.5).to(device), 128)
    bias = (rand(e, u, seed=seed + 3) * 0.1).to(device)
    bgate = (rand(e, u, seed=seed + 4) * 0.1).to(device)
    rs = rand(cap, seed=seed + 5).abs().to(device)
    linear = epi == L.SB_EPI_LINEAR
    pitch = u if linear else -(-u // 16) * 16
    out = torch.full((cap, pitch), 3.0, device=device) if linear else torch.full((cap, pitch), 99, dtype=torch.uint8,
                                                                                 device=device)
    osc = torch.full((-(-u // 128), cap), -1.0, device=device)
    import ctypes as C

    a = L.Fp8MatmulArgs(epilogue=epi, out_dtype=L.SB_F32, num_groups=e, max_rows=cap, n=u, k=h, a=x.q.data_ptr(),
                        lda=x.pitch, a_scale=x.scale.data_ptr(), a_scale_row=x.scale.stride(0),
                        a_scale_block=x.scale.stride(1), b=up.q.data_ptr(), b_gate=gate.q.data_ptr(), ldb=up.pitch,
                        b_group_rows=u, b_scale=up.scale.data_ptr(), b_gate_scale=gate.scale.data_ptr(),
                        b_scale_row=up.scale.stride(1), b_scale_block=up.scale.stride(2),
                        b_scale_group=up.scale.stride(0), b_block_rows=128, bias=bias.data_ptr(),
                        bias_gate=bgate.data_ptr(), bias_group=u, row_scale=rs.data_ptr() if linear else None,
                        offsets=off.data_ptr(), out=out.data_ptr(), ldo=pitch, out_scale=osc.data_ptr(),
                        out_scale_row=1, out_scale_block=cap, status=F._status_ptr(device))
    L.check(L.load().sb_fp8_matmul(C.byref(a), torch.cuda.current_stream().cuda_stream), "sb_fp8_matmul")
    torch.cuda.synchronize()
    check_status(device)
    d = lambda t: t.dequantize().double().cpu()  # noqa: E731
    return dict(total=total, off=off.cpu().tolist(), x=d(x), up=d(up), gate=d(gate), bias=bias.double().cpu(),
                bgate=bgate.double().cpu(), rs=rs.double().cpu(), out=out, scale=osc)


GROUPS = [(1, 128, 128, [3]), (3, 129, 70, [0, 1, 200]), (5, 256, 384, [130, 0, 32, 33, 64]),
          (40, 64, 256, [i % 4 for i in range(40)]), (4, 200, 300, [70, 0, 33, 17]),
          (6, 300, 256, [129, 300, 128, 0, 256, 31]), (4, 300, 512, [0, 0, 0, 0]), (2, 1000, 1040, [257, 128])]


@pytest.mark.parametrize("e,u,h,counts", GROUPS)
@pytest.mark.parametrize("epi", [L.SB_EPI_LINEAR, L.SB_EPI_GELU, L.SB_EPI_SWIGLU])
def test_grouped_product(epi, e, u, h, counts, cuda_device):
    """Every group against fp64.  Quantised outputs are compared with the exact
    activation: each is its nearest e4m3 multiple of the block's scale, so off by
    half a step (2^-4 of the value, or 2^-10 of the scale near zero) of a value
    that is itself off by the product's error.  The activations' slopes are below
    1.13 (GELU) and 1.1 (SiLU).  Rows behind the last group are left as they were."""
    g = grouped(epi, e, u, h, counts, 100 * e + u, cuda_device)
    used = g["total"]
    if epi == L.SB_EPI_LINEAR:
        assert (g["out"][used:] == 3).all()
    else:
        assert (g["out"][used:] == 99).all() and (g["scale"][:, used:] == -1).all()
    for i in range(e):
        lo, hi = g["off"][i], g["off"][i + 1]
        if lo == hi:
            continue
        x = g["x"][lo:hi]
        s_up, s_gate = x.abs() @ g["up"][i].abs().t(), x.abs() @ g["gate"][i].abs().t()
        rel = 2.0 ** -12 + (h / 128 + 8) * 2.0 ** -24
        up = x @ g["up"][i].t() + g["bias"][i]
        if epi == L.SB_EPI_LINEAR:
            rs = g["rs"][lo:hi, None]
            err = (g["out"][lo:hi].double().cpu() - up * rs).abs()
            assert (err <= (rel * s_up + 2.0 ** -22 * up.abs()) * rs).all()
            continue
        gate = x @ g["gate"][i].t() + g["bgate"][i]
        if epi == L.SB_EPI_SWIGLU:
            y = torch.nn.functional.silu(gate) * up
            slack = 1.1 * rel * s_gate * up.abs() + rel * s_up * gate.abs() + 1.1 * rel * rel * s_gate * s_up
        else:
            y = torch.nn.functional.gelu(up)
            slack = 1.13 * rel * s_up
        slack = slack + 2.0 ** -20 * y.abs() + 2.0 ** -22
        sc = g["scale"][:, lo:hi].t().cpu()
        want_amax = torch.nn.functional.pad(y, (0, -u % 128)).view(hi - lo, -1, 128).abs().amax(-1)
        smax = torch.nn.functional.pad(slack, (0, -u % 128)).view(hi - lo, -1, 128).amax(-1)
        assert ((sc.double() * 448 - want_amax).abs() <= smax + 2.0 ** -22 * want_amax).all()
        se = sc.double().repeat_interleave(128, 1)[:, :u]
        got = g["out"][lo:hi, :u].contiguous().view(torch.float8_e4m3fn).double().cpu() * se
        err = (got - y).abs()
        assert (err <= 2.0 ** -4 * (y.abs() + slack) + 2.0 ** -10 * se + slack).all()


@pytest.mark.parametrize("m,k,n", [(1, 64, 48), (40, 300, 130), (257, 512, 384), (7, 1000, 2056), (130, 129, 1),
                                   (300, 264, 136), (129, 72, 8)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_linear_and_gradients(m, k, n, dtype, cuda_device):
    x, w, dy = rand(m, k, seed=1, dtype=dtype), rand(n, k, seed=2, dtype=dtype), rand(m, n, seed=3, dtype=dtype)
    xd, wd = x.to(cuda_device).requires_grad_(), w.to(cuda_device).requires_grad_()
    y = fp8_block_linear(xd, wd)
    y.backward(dy.to(cuda_device))
    deq = lambda t, br: (lambda q, s: q.view(torch.float8_e4m3fn).double()  # noqa: E731
                         * s.double().repeat_interleave(br, 0)[: t.shape[0]].repeat_interleave(128, 1)[:, : t.shape[1]])(
        *plain_quantize(t, br))
    check(y.detach(), deq(x, 1), deq(w, 128), "y")
    check(xd.grad, deq(dy, 1), deq(w, 128).t(), "dx")
    check(wd.grad, deq(dy.t(), 1), deq(x.t(), 1), "dw")
    assert y.dtype == dtype and xd.grad.dtype == dtype and wd.grad.dtype == dtype
    # against the unquantised gradients: two roundings to e4m3 of at most 2^-4 each
    # (values near zero: 2^-10 of the block's scale, below 2^-18 of its amax)
    for got, a, b in ((xd.grad, dy.double(), w.double().t()), (wd.grad, dy.double().t(), x.double().t())):
        err = (got.double().cpu() - a @ b.t()).abs()
        amax = a.abs().amax() * b.abs().amax() * a.shape[1]
        assert (err <= (2.0 ** -3 + 2.0 ** -7) * (a.abs() @ b.abs().t()) + 2.0 ** -16 * amax).all()
    # a packed weight: the same values, and the input's gradient
    packed = quantize_fp8_blocks(w.to(cuda_device), 128)
    x2 = x.to(cuda_device).requires_grad_()
    y2 = fp8_block_linear(x2, packed)
    y2.backward(dy.to(cuda_device))
    assert torch.equal(y2, y) and torch.equal(x2.grad, xd.grad)
    assert torch.equal(fp8_block_linear(x.to(cuda_device), packed), y)


def test_linear_differences(cuda_device):
    """A difference of the layer along an axis is its gradient times the step,
    within the rounding of x and of the outputs: with x and x + step both exactly
    representable (multiples of the scale's step), y is linear in x and the
    difference is that of the exact product."""
    w = rand(96, 128, seed=4).to(cuda_device)
    x = torch.zeros(2, 128, device=cuda_device)
    x[:, 0] = 448.0                       # scale 1: small integers are exact
    x[:, 1:] = torch.arange(127, device=cuda_device) % 9 - 4.0
    dy = torch.ones(2, 96, device=cuda_device)
    leaf = x.clone().requires_grad_()
    fp8_block_linear(leaf, w).backward(dy)
    for i in (1, 64, 127):
        hi = x.clone()
        hi[:, i] += 1.0
        diff = (fp8_block_linear(hi, w) - fp8_block_linear(x, w)).double().sum(1)
        s = (x.abs() + 1).double() @ quantize_fp8_blocks(w, 128).dequantize().double().abs().t()
        assert ((diff - leaf.grad[:, i].double()).abs() <= 2.0 ** -11 * s.sum(1)).all()


def test_linear_shapes(cuda_device):
    w = rand(48, 64, seed=5, dtype=torch.bfloat16).to(cuda_device)
    x = rand(2, 3, 64, seed=6, dtype=torch.bfloat16).to(cuda_device)
    y = fp8_block_linear(x, w)
    assert y.shape == (2, 3, 48)
    assert torch.equal(y[1, 2], fp8_block_linear(x[1, 2], w))
    assert fp8_block_linear(x[:0], w).shape == (0, 3, 48)
    wl = w.clone().requires_grad_()
    xe = x[:0].clone().requires_grad_()
    fp8_block_linear(xe, wl).sum().backward()
    assert (wl.grad == 0).all() and xe.grad.shape == (0, 3, 64)
    with pytest.raises(RuntimeError, match="twice"):
        torch.autograd.grad(fp8_block_linear(x, wl).sum(), wl, create_graph=True)
    # an expanded (stride 0) gradient, as sum() makes
    wl = w.clone().requires_grad_()
    fp8_block_linear(x, wl).float().sum().backward()
    assert torch.isfinite(wl.grad).all()


# ---------------------------------------------------------------- experts
def make_experts(e, h, u, swiglu, seed, device, bias=True):
    t = {"up": rand(e, u, h, seed=seed) * h ** -0.5, "down": rand(e, h, u, seed=seed + 1) * u ** -0.5}
    if swiglu:
        t["gate"] = rand(e, u, h, seed=seed + 2) * h ** -0.5
    b = {s: rand(e, w.shape[1], seed=seed + 3) * 0.1 if bias else None for s, w in t.items()}
    dev = lambda x: None if x is None else x.to(device)  # noqa: E731
    ex = Fp8BlockExperts(dev(t["up"]), dev(b["up"]), dev(t["down"]), dev(b["down"]), dev(t.get("gate")),
                         dev(b.get("gate")))
    return ex, b


def delta_oracle(ex, b, x, idx, w, quantize=True):
    """(delta, S): fp64 from the definition; S bounds what the activations'
    rounding can move (quantize False: activations left unquantised)."""
    rows = lambda t: (lambda q, s: q.view(torch.float8_e4m3fn).double()  # noqa: E731
                      * s.double().repeat_interleave(128, 1)[:, : t.shape[1]])(*plain_quantize(t, 1))
    d = lambda t: t.dequantize().double().cpu()  # noqa: E731
    up, down, gate = d(ex.w_up), d(ex.w_down), d(ex.w_gate) if ex.w_gate is not None else None
    xq = rows(x)
    n, h = x.shape
    out, s = torch.zeros(n, h, dtype=torch.float64), torch.zeros(n, h, dtype=torch.float64)
    bias = lambda k, e: 0 if b[k] is None else b[k][e].double()  # noqa: E731
    for t in range(n):
        tot = {}
        for j in range(idx.shape[1]):
            e = int(idx[t, j])
            if 0 <= e < ex.num_experts:
                tot[e] = tot.get(e, 0.0) + float(w[t, j])
        for e, we in tot.items():
            if not we > 0:
                continue
            y = up[e] @ xq[t] + bias("up", e)
            if gate is not None:
                y = torch.nn.functional.silu(gate[e] @ xq[t] + bias("gate", e)) * y
            else:
                y = torch.nn.functional.gelu(y)
            a = rows(y[None].float())[0] if quantize else y
            out[t] += we * (down[e] @ a + bias("down", e))
            s[t] += we * (down[e].abs() @ (y.abs() + y.abs().amax() * 2.0 ** -14))
    return out, s


EXPERTS = [(1, 4, 1, 128, 128, True), (1, 4, 2, 64, 100, False), (5, 8, 2, 256, 384, True), (64, 16, 2, 256, 128, True),
           (40, 6, 3, 200, 130, False), (33, 5, 5, 129, 257, True), (300, 4, 2, 512, 256, False), (9, 130, 8, 64, 64, True)]


@pytest.mark.parametrize("n,e,k,h,u,swiglu", EXPERTS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_expert_delta(n, e, k, h, u, swiglu, dtype, cuda_device):
    """Routing and experts together.  Element by element, the result is within the
    activations' half steps (2^-4, plus the products' 2^-12 through the slope) of
    the unquantised-activation FFN; row by row (2-norm), within 2^-5 of the FFN
    with the activations quantised: an activation next to a rounding border may
    land one step (2^-3) away, which at most one in 16 can do (the product's error,
    2^-12 S with S below 16 values, over a step of 2^-3, twice)."""
    ex, b = make_experts(e, h, u, swiglu, 10 * n + e, cuda_device)
    x = rand(n, h, seed=n, dtype=dtype)
    logits = rand(n, e, seed=n + 1)
    idx, w = route_experts(logits.to(cuda_device), k)
    got = fp8_expert_delta(x.to(cuda_device), idx, w, ex)
    check_status(cuda_device)
    assert got.dtype == dtype and got.shape == (n, h)
    want, _ = delta_oracle(ex, b, x, idx.cpu(), w.cpu())
    free, s = delta_oracle(ex, b, x, idx.cpu(), w.cpu(), quantize=False)
    half = 2.0 ** -8 if dtype == torch.bfloat16 else 0.0
    err = (got.double().cpu() - free).abs()
    assert (err <= (2.0 ** -4 + 2.0 ** -6) * s + half * free.abs()).all()
    rowerr = (got.double().cpu() - want).norm(dim=1) / want.norm(dim=1)
    assert rowerr.max() < 2.0 ** -5, float(rowerr.max())
    assert torch.equal(got, fp8_expert_delta(x.to(cuda_device), idx, w, ex))


def test_expert_delta_routing_rules(cuda_device):
    """Repeated ids add their weights; ids outside [0, E) and weights <= 0 are
    skipped; a token with none left gets zeros; int64 ids and strided rows."""
    ex, b = make_experts(4, 64, 48, True, 77, cuda_device)
    x = rand(6, 64, seed=78, dtype=torch.bfloat16)
    idx = torch.tensor([[1, 1], [3, -1], [4, 2], [0, 3], [9, -7], [2, 0]])
    w = torch.tensor([[0.25, 0.5], [1.0, 1.0], [1.0, 0.5], [0.0, 1.0], [1.0, 1.0], [-1.0, 0.5]])
    got = fp8_expert_delta(x.to(cuda_device), idx.to(cuda_device), w.to(cuda_device), ex)
    want, _ = delta_oracle(ex, b, x, idx, w)
    assert (got[4] == 0).all()
    live = want.norm(dim=1) > 0
    assert ((got.double().cpu() - want).norm(dim=1)[live] / want.norm(dim=1)[live]).max() < 2.0 ** -5
    wide = torch.zeros(6, 100, dtype=torch.bfloat16, device=cuda_device)
    wide[:, 8:72] = x.to(cuda_device)
    assert torch.equal(fp8_expert_delta(wide[:, 8:72], idx.int().to(cuda_device), w.to(cuda_device), ex), got)
    assert fp8_expert_delta(x[:0].to(cuda_device), idx[:0].to(cuda_device), w[:0].to(cuda_device), ex).shape == (0, 64)
    three = fp8_expert_delta(x.view(2, 3, 64).to(cuda_device), idx.view(2, 3, 2).to(cuda_device),
                             w.view(2, 3, 2).to(cuda_device), ex)
    assert torch.equal(three.view(6, 64), got)
    with pytest.raises(NotImplementedError):
        fp8_expert_delta(x.to(cuda_device).requires_grad_(), idx.to(cuda_device), w.to(cuda_device), ex)
    with pytest.raises(ValueError):
        fp8_expert_delta(x[:, :63].to(cuda_device), idx.to(cuda_device), w.to(cuda_device), ex)
    # the ranks' parts add up
    parts = sum(ex.delta(x.to(cuda_device), idx.to(cuda_device), w.to(cuda_device), r, 3, torch.float32) for r in range(3))
    torch.testing.assert_close(parts.double().cpu(), ex.delta(x.to(cuda_device), idx.to(cuda_device), w.to(cuda_device),
                                                              out_dtype=torch.float32).double().cpu(), rtol=2.0 ** -20, atol=1e-6)


def test_many_experts(cuda_device):
    """256 experts (the limit), most without a token; one more is refused."""
    g = torch.Generator().manual_seed(3)
    w = torch.randint(0, 120, (256, 32, 16), generator=g).to(torch.uint8).to(cuda_device).view(torch.float8_e4m3fn)
    up = Fp8BlockTensor(w, torch.full((256, 1, 1), 2.0 ** -6, device=cuda_device), 128)
    down = Fp8BlockTensor(w.view(torch.uint8).view(256, 16, 32).view(torch.float8_e4m3fn),
                          torch.full((256, 1, 1), 2.0 ** -6, device=cuda_device), 128)
    ex = Fp8BlockExperts(up, None, down, None)
    x = rand(20, 16, seed=4)
    idx = torch.randint(0, 256, (20, 3), generator=g)
    idx[0] = torch.tensor([0, 255, 128])
    wt = torch.rand(20, 3, generator=g) + 0.1
    got = fp8_expert_delta(x.to(cuda_device), idx.to(cuda_device), wt.to(cuda_device), ex)
    want, _ = delta_oracle(ex, dict(up=None, down=None), x, idx, wt)
    assert ((got.double().cpu() - want).norm(dim=1) / want.norm(dim=1)).max() < 2.0 ** -5
    with pytest.raises(ValueError):
        big = lambda t: Fp8BlockTensor(torch.cat([t.q.view(torch.uint8), t.q[:1].view(torch.uint8)]).view(t.q.dtype),  # noqa: E731
                                       torch.ones(257, 1, 1, device=cuda_device), 128)
        Fp8BlockExperts(big(up), None, big(down), None)


def test_all_routes_dropped(cuda_device):
    """No token keeps an expert: zeros, from kernels without an item."""
    ex, _ = make_experts(6, 64, 48, True, 7, cuda_device)
    for n in (1, 700):
        x = rand(n, 64, seed=8).to(cuda_device)
        idx = torch.full((n, 2), -1, device=cuda_device)
        assert (fp8_expert_delta(x, idx, torch.ones(n, 2, device=cuda_device), ex) == 0).all()
    check_status(cuda_device)


def test_two_graphs_and_a_stream(cuda_device):
    """Two captured steps of different sizes and an eager call, replayed in turn:
    none uses another's scratch."""
    ex, _ = make_experts(8, 128, 96, True, 5, cuda_device)
    w = quantize_fp8_blocks(rand(128, 128, seed=6).to(cuda_device), 128)

    def step(x, logits):
        idx, tw = route_experts(logits, 2)
        return fp8_block_linear(x + fp8_expert_delta(x, idx, tw, ex), w)

    graphs = []
    for n in (3, 150):
        x = rand(n, 128, seed=n, dtype=torch.bfloat16).to(cuda_device)
        lg = rand(n, 8, seed=n + 1).to(cuda_device)
        want = step(x, lg)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            step(x, lg)
        torch.cuda.current_stream().wait_stream(s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(x, lg)
        graphs.append((graph, out, want, x, lg))
    for _ in range(3):
        for graph, *_ in graphs:
            graph.replay()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            eager = step(graphs[1][3], graphs[1][4])
        for graph, *_ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(eager, graphs[1][2])
        for _, out, want, *_ in graphs:
            assert torch.equal(out, want)


def test_training_step_captured(cuda_device):
    """A captured forward + backward equals the eager one.  (No eager graph of the
    same leaves may be alive then: autograd would tie the capture to the stream
    that graph was built on, whatever operator it holds.)"""
    x = rand(40, 64, seed=1).to(cuda_device).requires_grad_()
    w = rand(32, 64, seed=2).to(cuda_device).requires_grad_()
    dy = rand(40, 32, seed=3).to(cuda_device)
    want = torch.autograd.grad(fp8_block_linear(x, w), (x, w), dy)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        torch.autograd.grad(fp8_block_linear(x, w), (x, w), dy)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = torch.autograd.grad(fp8_block_linear(x, w), (x, w), dy)
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    fp8_block_linear(x, w).backward(dy)
    assert torch.equal(x.grad, want[0]) and torch.equal(w.grad, want[1])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_linear_expanded_gradient(dtype, cuda_device):
    """A gradient of stride 0 in both dimensions gives what its dense copy gives."""
    x = rand(37, 200, seed=1, dtype=dtype).to(cuda_device).requires_grad_()
    w = rand(130, 200, seed=2, dtype=dtype).to(cuda_device).requires_grad_()
    one = torch.ones(1, 1, dtype=dtype, device=cuda_device)
    got = torch.autograd.grad(fp8_block_linear(x, w), (x, w), one.expand(37, 130))
    want = torch.autograd.grad(fp8_block_linear(x, w), (x, w), one.repeat(37, 130))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_linear_without_columns(cuda_device):
    """Leading dimensions and no elements to sum over: zeros."""
    y = fp8_block_linear(torch.ones(2, 3, 0, device=cuda_device), torch.ones(5, 0, device=cuda_device))
    assert y.shape == (2, 3, 5) and (y == 0).all()
    y = fp8_block_linear(torch.ones(0, device=cuda_device), torch.ones(5, 0, device=cuda_device))
    assert y.shape == (5,) and (y == 0).all()


def test_expert_ids_of_every_type(cuda_device):
    """64-bit ids do not wrap into [0, E); narrow integers count; other types are refused."""
    ex, _ = make_experts(4, 64, 48, False, 5, cuda_device)
    x = rand(3, 64, seed=6).to(cuda_device)
    w = torch.ones(3, 2, device=cuda_device)
    ids = torch.tensor([[0, 3], [1, -1], [2, 4]], device=cuda_device)
    want = fp8_expert_delta(x, ids.int(), w, ex)
    far = ids.clone()
    far[1, 1], far[2, 1] = 2 ** 32, -(2 ** 32) + 1
    assert torch.equal(fp8_expert_delta(x, far, w, ex), want)
    for dtype in (torch.int16, torch.int8):
        assert torch.equal(fp8_expert_delta(x, ids.to(dtype), w, ex), want)
    parts = sum(ex.delta(x, far, w, r, 2, torch.float32) for r in range(2))
    torch.testing.assert_close(parts, want, rtol=2.0 ** -20, atol=1e-6)
    for dtype in (torch.float32, torch.bool):
        with pytest.raises(TypeError):
            fp8_expert_delta(x, ids.to(dtype), w, ex)


def test_offsets_past_32_bits(cuda_device):
    """Inputs and outputs of more than 2^31 elements: the last rows are those of a small call."""
    m, k = 70000, 32768
    x = torch.zeros(m, k, dtype=torch.bfloat16, device=cuda_device)
    tail = rand(300, k, seed=1, dtype=torch.bfloat16).to(cuda_device)
    x[-300:] = tail
    want = quantize_fp8_blocks(tail)
    got = quantize_fp8_blocks(x)
    assert torch.equal(got.q[-300:].view(torch.uint8), want.q.view(torch.uint8))
    assert torch.equal(got.scale[-300:], want.scale)
    del got
    cut = (m - 300) // 128 * 128  # whole blocks of 128 from here on
    for br in (1, 128):
        want = quantize_fp8_blocks(x[cut:].t(), br)
        got = quantize_fp8_blocks(x.t(), br)
        assert torch.equal(got.q[:, cut:].view(torch.uint8), want.q.view(torch.uint8))
        assert torch.equal(got.scale[:, cut // 128:], want.scale)
        del got
    want = quantize_fp8_blocks(x[cut:], 128)
    got = quantize_fp8_blocks(x, 128)
    assert torch.equal(got.q[cut:].view(torch.uint8), want.q.view(torch.uint8))
    assert torch.equal(got.scale[cut // 128:], want.scale)
    del got, x
    a, b = quantize_fp8_blocks(rand(m, 64, seed=2).to(cuda_device)), quantize_fp8_blocks(rand(k, 64, seed=3).to(cuda_device), 128)
    last = Fp8BlockTensor(a.q[-500:], a.scale[-500:], 1)
    assert torch.equal(F.fp8_block_matmul(a, b)[-500:], F.fp8_block_matmul(last, b))


@pytest.mark.parametrize("n", [3, 600])
def test_gelu_of_large_values(n, cuda_device):
    """GELU far from 0, on the decode and on the row schedule: 0 on the left, -inf
    too; x on the right; NaN stays NaN, in the rows of its expert only."""
    ex, _ = make_experts(2, 64, 48, False, 9, cuda_device)
    x = rand(n, 64, seed=10).to(cuda_device)
    idx = (torch.arange(n, device=cuda_device) % 2).view(n, 1)
    w = torch.ones(n, 1, device=cuda_device)
    out = {}
    for v in (-1e4, -3e38, float("-inf"), float("nan")):
        ex.b_up[0, 7] = v
        out[v] = fp8_expert_delta(x, idx, w, ex)
    a, b, c, d = out.values()
    assert torch.isfinite(a).all() and torch.equal(a, b) and torch.equal(a, c)
    assert torch.isnan(d[::2]).all() and torch.equal(d[1::2], a[1::2])
    ex.b_up.fill_(0.0)
    ex.b_up[0, 7] = 2.0 ** 20  # the block's largest: its column of w_down times 2^20, within two roundings
    got = fp8_expert_delta(x, idx, w, ex)[::2].double()
    ffn = x.double()[::2] @ ex.w_up.dequantize(torch.float64)[0].T
    act = ffn[:, 7:8] + 2.0 ** 20
    want = act * ex.w_down.dequantize(torch.float64)[0, :, 7]
    if ex.b_down is not None:
        want = want + ex.b_down[0].double()
    assert ((got - want).norm(dim=1) / want.norm(dim=1)).max() < 2.0 ** -4
