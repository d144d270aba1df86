"""Layer norm, rotary positions in every layout, token log-probabilities and routing to experts: the HIP kernels (GPU) and the
PyTorch references (CPU) against the definitions in 64 bits.

Tolerances count roundings: half a step of the output's type, `finfo.eps / 2` relative, plus `extra`, a bound on the fp32
arithmetic before it in units of U = 2^-24 (each derived where it is formed; a sum of n terms of one lane or thread and a
tree of t levels is off by at most (n + t) U times the sum of the terms' absolute values)."""

import math

import pytest
import torch

from accelerate_hpc_test_amd.models import moe
from accelerate_hpc_test_amd.ops import apply_rope, layer_norm, rope_tables, route_experts, token_logprobs

U = 2.0 ** -24
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
ON = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
gpu = pytest.mark.gpu


def gen(device, seed=0):
    return torch.Generator(device=device).manual_seed(seed)


def normal(g, *shape, dtype=FP32, scale=1.0):
    return (torch.randn(*shape, generator=g, device=g.device) * scale).to(dtype)


def check(out, ref, extra=0.0, what=""):
    """|out - ref| within half a step of out's type and `extra`; NaN and inf where the reference has them."""
    assert out.shape == ref.shape, (what, out.shape, ref.shape)
    o, r = out.detach().double(), ref.detach().double()
    fi = torch.finfo(out.dtype)
    tol = fi.eps / 2 * (r.abs() + extra) * (1 + 2.0 ** -7) + fi.smallest_normal * fi.eps + extra
    same = (o == r) | (o.isnan() & r.isnan()) | (o == ref.detach().to(out.dtype).double())  # past the type's range: inf
    bad = ~(same | ((o - r).abs() <= tol))
    if bad.any():
        at = bad.nonzero()[0].tolist()
        worst = ((o - r).abs() / tol)[bad].max().item()
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {worst:.3g} x the bound; at {at}: "
                             f"{o[tuple(at)].item()} for {r[tuple(at)].item()}")


# ----------------------------------------------------------------------------------------------------------------- layer norm
def norm_case(device, rows, hidden, dtype, residual, params, seed=0):
    g = gen(device, seed)
    x = normal(g, rows, hidden, dtype=dtype, scale=1.5) + 0.3
    res = normal(g, rows, hidden, dtype=dtype) if residual else None
    pdt = FP32 if params == "wide" else dtype
    w = (1 + 0.2 * normal(g, hidden)).to(pdt) if params != "none" else None
    b = (0.2 * normal(g, hidden)).to(pdt) if params in ("both", "wide") else None
    return x.to(dtype), res, w, b, g


def norm64(x, res, w, b, eps, dy=None, dres=None):
    """Outputs, gradients and the bounds of their fp32 errors."""
    s = x.double() if res is None else (x.double() + res.double()).to(x.dtype).double()
    H = s.shape[-1]
    W = torch.ones(H, dtype=torch.float64, device=x.device) if w is None else w.double()
    B = torch.zeros_like(W) if b is None else b.double()
    mu = s.mean(-1, keepdim=True)
    r = ((s - mu).square().mean(-1, keepdim=True) + eps).rsqrt()
    h = (s - mu) * r
    # a thread adds at most 32 values, then 10 levels: the mean is off by 42 U mean|s|, the variance and so rstd by 30 U relative
    dh = U * (42 * r * s.abs().mean(-1, keepdim=True) + 34 * h.abs())
    out = {"s": s, "y": h * W + B, "y_extra": W.abs() * dh + 3 * U * ((h * W).abs() + B.abs())}
    if dy is not None:
        dy = dy.double()
        q = dy * W
        m1, m2 = q.mean(-1, keepdim=True), (q * h).mean(-1, keepdim=True)
        out["dx"] = r * (q - m1 - h * m2) + (0 if dres is None else dres.double())
        size = q.abs() + q.abs().mean(-1, keepdim=True) + h.abs() * (q * h).abs().mean(-1, keepdim=True)
        out["dx_extra"] = r * (64 * U * size + dh * m2.abs() + h.abs() * (q.abs() * dh).mean(-1, keepdim=True)) + 2 * U * out["dx"].abs()
        rows = s.shape[0]
        n = 64 + rows / 64  # the rows a thread adds, and the joins: 512 blocks and 32 row groups share them
        out["dw"], out["db"] = (dy * h).sum(0), dy.sum(0)
        out["dw_extra"] = n * U * (dy * h).abs().sum(0) + (dy.abs() * dh).sum(0)
        out["db_extra"] = n * U * dy.abs().sum(0)
    return out


NORM_SHAPES = [(1, 1), (3, 1), (5, 2), (2, 7), (4, 8), (17, 33), (64, 256), (9, 511), (7, 513), (33, 1027), (300, 1024),
               (2, 2049), (5, 4096), (70, 4096), (3, 6144), (2, 8200), (2, 16383), (1, 16384)]


def run_norm(device, rows, hidden, dtype, residual, params):
    x, res, w, b, g = norm_case(device, rows, hidden, dtype, residual, params)
    leaves = [t.requires_grad_() for t in (x, res, w, b) if t is not None]
    y, s = layer_norm(x, w, b, 1e-5, res)
    assert y.dtype == dtype and (s is x) == (res is None)
    dy = normal(g, rows, hidden, dtype=dtype)
    dres = normal(g, rows, hidden, dtype=dtype) if residual else None
    grads = dict(zip([id(t) for t in leaves], torch.autograd.grad((y, s) if residual else y, leaves, (dy, dres) if residual else dy)))
    ref = norm64(x.detach(), None if res is None else res.detach(), w, b, 1e-5, dy, dres)
    check(y, ref["y"], ref["y_extra"], "y")
    if residual:
        assert torch.equal(s.detach().double(), ref["s"])
        check(grads[id(res)], ref["dx"], ref["dx_extra"], "dresidual")
    check(grads[id(x)], ref["dx"], ref["dx_extra"], "dx")
    if w is not None:
        assert grads[id(w)].dtype == w.dtype
        check(grads[id(w)], ref["dw"], ref["dw_extra"], "dweight")
    if b is not None:
        check(grads[id(b)], ref["db"], ref["db_extra"], "dbias")
    with torch.no_grad():
        y2, _ = layer_norm(x, w, b, 1e-5, res)
    assert torch.equal(y2, y)


@pytest.mark.parametrize("device", ON)
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("rows,hidden", NORM_SHAPES)
def test_layer_norm(device, dtype, rows, hidden):
    run_norm(device, rows, hidden, dtype, (rows + hidden) % 2 == 0, "both")


@pytest.mark.parametrize("device", ON)
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("params", ["none", "weight", "both", "wide"])
@pytest.mark.parametrize("dtype,hidden", [(BF16, 200), (FP16, 3001), (FP32, 515)])
def test_layer_norm_parameters(device, dtype, hidden, params, residual):
    run_norm(device, 19, hidden, dtype, residual, params)


@gpu
@pytest.mark.parametrize("dtype,hidden", [(BF16, 32768), (BF16, 32767), (FP16, 20001), (FP32, 16384)])
def test_layer_norm_widest_rows(dtype, hidden):
    run_norm("cuda", 5, hidden, dtype, True, "both")


@gpu
@pytest.mark.parametrize("rows,hidden,dtype", [(2500, 256, BF16), (1030, 2048, BF16), (5000, 100, FP32), (1100, 4096, BF16)])
def test_layer_norm_many_rows(rows, hidden, dtype):
    run_norm("cuda", rows, hidden, dtype, True, "both")


@gpu
@pytest.mark.parametrize("rows,hidden,dtype", [(33001, 64, BF16), (33001, 61, BF16), (40003, 32, FP32), (17003, 100, BF16), (9001, 250, FP16),
                                               (700, 9001, BF16), (600, 20001, BF16), (300, 24576, FP16), (300, 16381, FP32)])
def test_layer_norm_rows_past_one_round_of_the_blocks(rows, hidden, dtype):
    # rows that share a wave, and rows of 512 threads: more of each than the blocks of a launch take at once, whole and ragged
    run_norm("cuda", rows, hidden, dtype, True, "both")


@pytest.mark.parametrize("device", ON)
def test_layer_norm_strides_and_broadcast_gradients(device):
    g = gen(device, 1)
    wide = normal(g, 6, 5, 3 * 40, dtype=BF16)
    w, b = normal(g, 40, dtype=BF16).requires_grad_(), normal(g, 40, dtype=BF16).requires_grad_()
    for x in (wide[..., 40:80], wide[::2, :, 1:41], wide[:, :, ::3], wide.transpose(0, 1)[..., :40], wide[:1, :1, :40].expand(6, 5, 40),
              wide[0, 0, :40]):
        leaf = x.detach().requires_grad_()
        y, _ = layer_norm(leaf, w, b)
        ref = norm64(x.reshape(-1, 40), None, w, b, 1e-5, torch.ones(x.numel() // 40, 40, device=device))
        check(y.reshape(-1, 40), ref["y"], ref["y_extra"], "y")
        dx, dw, db = torch.autograd.grad(y.sum(), (leaf, w, b))  # an expanded gradient: strides of zero
        check(dx.reshape(-1, 40), ref["dx"], ref["dx_extra"], "dx")
        check(dw, ref["dw"], ref["dw_extra"], "dweight")
        check(db, ref["db"], ref["db_extra"], "dbias")


@pytest.mark.parametrize("device", ON)
def test_layer_norm_empty_constant_and_poisoned_rows(device):
    w = torch.ones(24, device=device, dtype=BF16, requires_grad=True)
    x = torch.zeros(0, 24, device=device, dtype=BF16, requires_grad=True)
    y, _ = layer_norm(x, w, w, residual=x)
    y.sum().backward()
    assert y.shape == (0, 24) and x.grad.shape == (0, 24) and not w.grad.any()
    x = torch.full((4, 24), 3.0, device=device, dtype=FP32)
    x[1] = torch.randn(24, device=device)
    x[2, 5] = math.nan
    x[3, 7] = math.inf
    y, _ = layer_norm(x)
    assert torch.equal(y[0], torch.zeros_like(y[0])) and y[1].isfinite().all() and y[2].isnan().all() and y[3].isnan().all()


@pytest.mark.parametrize("device", ON)
def test_layer_norm_partial_gradients(device):
    """Only some inputs need gradients; only the residual output is used; a frozen norm inside a graph."""
    g = gen(device, 2)
    x, res = normal(g, 6, 48, dtype=BF16), normal(g, 6, 48, dtype=BF16)
    w, b = normal(g, 48, dtype=BF16), normal(g, 48, dtype=BF16)
    dy = normal(g, 6, 48, dtype=BF16)
    ref = norm64(x, res, w, b, 1e-5, dy)
    for name, leaf in (("dx", x), ("dx", res), ("dw", w), ("db", b)):
        leaf.requires_grad_()
        y, s = layer_norm(x, w, b, 1e-5, res)
        (got,) = torch.autograd.grad(y, leaf, dy)
        check(got, ref[name], ref[name + "_extra"], name)
        leaf.requires_grad_(False)
    x.requires_grad_()
    _, s = layer_norm(x, w, b, 1e-5, res)
    assert torch.equal(torch.autograd.grad(s, x, dy)[0], dy)


def test_layer_norm_gradient_by_differences():
    g = gen("cpu", 3)
    args = [normal(g, 3, 5).double().requires_grad_() for _ in range(2)] + [normal(g, 5).double().requires_grad_() for _ in range(2)]
    assert torch.autograd.gradcheck(lambda x, r, w, b: layer_norm(x, w, b, 1e-5, r), tuple(args))


@pytest.mark.parametrize("device", ON)
def test_layer_norm_refusals(device):
    x = torch.zeros(4, 8, device=device)
    for bad in (dict(weight=torch.zeros(7, device=device)), dict(bias=torch.zeros(8, 1, device=device)),
                dict(residual=torch.zeros(4, 7, device=device)), dict(residual=x.to(BF16))):
        with pytest.raises(ValueError):
            layer_norm(x, **bad)
    for bad in (torch.zeros((), device=device), torch.zeros(3, 0, device=device)):
        with pytest.raises(ValueError):
            layer_norm(bad)
    with pytest.raises(TypeError):
        layer_norm(torch.zeros(3, 4, dtype=torch.int32, device=device))
    if device == "cuda":
        with pytest.raises(ValueError):
            layer_norm(torch.zeros(1, 32769, device=device, dtype=BF16))


# ----------------------------------------------------------------------------------------------------------- rotary positions
def rope64(x, cos, sin, n_rot, positions, interleaved, R):
    """Complex multiplication of the pairs."""
    B, S, H, D = x.shape
    if positions is None:
        positions = torch.arange(S, device=x.device)
    turn = torch.complex(cos.double(), sin.double())[positions.expand(B, S)][:, :, None]
    z = x.double()[:, :, :n_rot, :R]
    z = z.reshape(B, S, n_rot, R // 2, 2) if interleaved else z.reshape(B, S, n_rot, 2, R // 2).transpose(-1, -2)
    z = torch.view_as_real(torch.complex(z[..., 0], z[..., 1]) * turn)
    z = z.reshape(B, S, n_rot, R) if interleaved else z.transpose(-1, -2).reshape(B, S, n_rot, R)
    return torch.cat([torch.cat([z, x.double()[:, :, :n_rot, R:]], -1), x.double()[:, :, n_rot:]], 2)


def rope_extra(x, n_rot, R):
    """Two products and a sum in fp32: 3 U of the pair's length, which is at most the sum of both sizes."""
    e = torch.zeros_like(x, dtype=torch.float64)
    big = x.double()[:, :, :n_rot, :R].abs()
    e[:, :, :n_rot, :R] = 3 * U * 2 * big.amax(-1, keepdim=True)
    return e


def run_rope(device, B, S, n_rot, H, D, R, interleaved, dtype, positions, x=None, table=None):
    g = gen(device, D + R)
    cos, sin = rope_tables(table or 600, R, 10000.0, device)
    x = normal(g, B, S, H, D, dtype=dtype) if x is None else x
    pos = torch.randint(0, cos.shape[0], (B, S), generator=g, device=device) if positions else None
    leaf = x.detach().requires_grad_()
    out = apply_rope(leaf, cos, sin, n_rot, pos, interleaved=interleaved, rotary_dim=R)
    check(out, rope64(x, cos, sin, n_rot, pos, interleaved, R), rope_extra(x, n_rot, R), "out")
    g_out = normal(g, B, S, H, D, dtype=dtype)
    (dx,) = torch.autograd.grad(out, leaf, g_out)
    check(dx, rope64(g_out, cos, -sin, n_rot, pos, interleaved, R), rope_extra(g_out, n_rot, R), "gradient")
    assert torch.equal(out[:, :, n_rot:], x[:, :, n_rot:]) and torch.equal(out[..., R:], x[..., R:])
    with torch.no_grad():
        assert torch.equal(apply_rope(x, cos, sin, n_rot, pos, interleaved=interleaved, rotary_dim=R), out)


ROPE_SIZES = [(128, 128), (64, 64), (256, 64), (96, 24), (80, 74), (80, 78), (64, 2), (5, 2), (7, 6), (6, 4), (48, 12), (33, 10),
              (128, 126), (576, 64), (192, 64), (2, 2), (9, 8)]


@pytest.mark.parametrize("device", ON)
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,R", ROPE_SIZES)
def test_rope(device, D, R, interleaved, dtype):
    run_rope(device, 2, 13, 5, 7, D, R, interleaved, dtype, positions=(D + R) % 3 != 0)


@gpu
@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("D,R", [(8, 8), (9, 8), (16, 16), (17, 16), (19, 18), (23, 18), (24, 18), (31, 22), (40, 30), (1000, 994), (1000, 10),
                                 (999, 998), (1000, 18)])
def test_rope_windows_of_the_halves(D, R, dtype):
    # halves of a window, of one value less or more, copied ends shorter and longer than a window, the widest heads
    run_rope("cuda", 2, 11, 3, 4, D, R, False, dtype, positions=True)


@pytest.mark.parametrize("device", ON)
@pytest.mark.parametrize("B,S,n_rot,H", [(1, 1, 1, 1), (33, 1, 40, 48), (1, 517, 3, 3), (3, 70, 0, 2), (2, 9, 1, 300)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rope_lengths_and_heads(device, B, S, n_rot, H, interleaved):
    for positions in (False, True):
        run_rope(device, B, S, n_rot, H, 64, 32, interleaved, BF16, positions)


@pytest.mark.parametrize("device", ON)
@pytest.mark.parametrize("interleaved", [False, True])
def test_rope_strides(device, interleaved):
    g = gen(device, 5)
    big = normal(g, 2, 9, 8, 100, dtype=BF16)
    for x in (big[..., 3:83], big[:, ::2, 1:6, :80], big.transpose(1, 2)[..., :80], big[:, :, ::3, :80], big[..., ::2][..., :48],
              big[:1, :, :, :80].expand(3, -1, -1, -1)):
        B, S, H, D = x.shape
        run_rope(device, B, S, min(3, H), H, D, 24, interleaved, BF16, True, x=x)


@pytest.mark.parametrize("device", ON)
def test_rope_shared_positions_and_long_tables(device):
    """One row of positions for the whole batch, [S] positions, 32-bit ones, and tables longer than the sequence."""
    g = gen(device, 6)
    cos, sin = rope_tables(64, 32, 10000.0, device)
    x = normal(g, 3, 10, 4, 32, dtype=BF16)
    pos = torch.randperm(64, generator=g, device=device)[:10]
    want = rope64(x, cos, sin, 3, pos, False, 32)
    if device == "cuda":
        for p in (pos, pos[None], pos[None].expand(3, 10), pos[None].expand(3, 10).int(), pos.int()):
            check(apply_rope(x, cos, sin, 3, p), want, rope_extra(x, 3, 32), "positions")
    for interleaved in (False, True):
        check(apply_rope(x, cos, sin, 3, interleaved=interleaved), rope64(x, cos, sin, 3, None, interleaved, 32), rope_extra(x, 3, 32),
              "tables longer than the sequence")


@gpu
@pytest.mark.parametrize("interleaved", [False, True])
def test_rope_positions_outside_the_tables(interleaved):
    cos, sin = rope_tables(16, 8, 10000.0, "cuda")
    x = torch.ones(1, 4, 2, 12, device="cuda", dtype=FP32)
    pos = torch.tensor([[0, 16, -1, 2**40]], device="cuda")
    out = apply_rope(x, cos, sin, 1, pos, interleaved=interleaved, rotary_dim=8)
    assert out[0, 0].isfinite().all() and out[0, 1:, 0, :8].isnan().all()
    assert (out[0, :, 0, 8:] == 1).all() and (out[0, :, 1] == 1).all()


@gpu
@pytest.mark.parametrize("D", [128, 24])
def test_rope_positions_outside_the_tables_whole_heads(D):
    """bf16 heads rotated whole in halves: their own kernel, forward and backward."""
    cos, sin = rope_tables(16, D, 10000.0, "cuda")
    x = torch.ones(1, 5, 3, D, device="cuda", dtype=BF16, requires_grad=True)
    pos = torch.tensor([[3, 16, -1, -(2**40), 15]], device="cuda")
    out = apply_rope(x, cos, sin, 2, pos)
    (d,) = torch.autograd.grad(out, x, torch.ones_like(out))
    for t in (out, d):
        assert t[0, [0, 4]].isfinite().all() and t[0, 1:4, :2].isnan().all() and (t[0, :, 2] == 1).all()
    check(out[0, [0, 4]], rope64(x, cos, sin, 2, torch.tensor([[3, 0, 0, 0, 15]], device="cuda"), False, D)[0, [0, 4]], 6 * U, "inside")


@pytest.mark.parametrize("device", ON)
def test_rope_empty(device):
    cos, sin = rope_tables(8, 4, 10000.0, device)
    for shape in ((0, 3, 2, 6), (2, 0, 2, 6), (1, 3, 0, 6)):
        x = torch.zeros(shape, device=device, dtype=BF16, requires_grad=True)
        y = apply_rope(x, cos, sin, 0, interleaved=True, rotary_dim=4)
        assert y.shape == shape
        y.sum().backward()
        x = torch.zeros(*shape[:3], 8, device=device, dtype=BF16, requires_grad=True)
        y = apply_rope(x, *rope_tables(8, 8, 10000.0, device), 0)
        assert y.shape == x.shape
        y.sum().backward()


@pytest.mark.parametrize("device", ON)
def test_rope_refusals(device):
    cos, sin = rope_tables(8, 4, 10000.0, device)
    x = torch.zeros(1, 4, 2, 6, device=device, dtype=BF16)
    for kw in (dict(rotary_dim=3), dict(rotary_dim=8), dict(rotary_dim=0), dict(rotary_dim=6), dict()):
        with pytest.raises(ValueError):
            apply_rope(x, cos, sin, 1, **kw)
    with pytest.raises(ValueError):
        apply_rope(x, cos, sin, 3, rotary_dim=4)
    with pytest.raises(ValueError):
        apply_rope(torch.zeros(1, 9, 2, 6, device=device), cos, sin, 1, rotary_dim=4)
    if device == "cuda":
        with pytest.raises(ValueError):
            apply_rope(torch.zeros(1, 1, 1, 1002, device=device), cos, sin, 1, rotary_dim=4)


@pytest.mark.parametrize("kind", ["linear", "dynamic", "yarn", "yarn mscale", "llama3"])
def test_rope_tables_scaled(kind):
    """Frequencies and amplitude against the installed transformers' for the same configuration."""
    from transformers import LlamaConfig
    from transformers.modeling_rope_utils import ROPE_INIT_FUNCTIONS

    S, D = 3000, 64
    scaling = {"rope_type": kind.split()[0], "factor": 4.0, "original_max_position_embeddings": 1024}
    if kind == "yarn mscale":
        scaling |= {"mscale": 0.8, "mscale_all_dim": 0.5, "beta_fast": 24.0, "beta_slow": 2.0}
    if kind == "llama3":
        scaling |= {"low_freq_factor": 1.0, "high_freq_factor": 4.0}
    maximum = 1024 if kind == "dynamic" else 4096
    cfg = LlamaConfig(hidden_size=256, num_attention_heads=4, head_dim=D, max_position_embeddings=maximum,
                      rope_parameters=dict(scaling, rope_theta=10000.0))
    cfg.rope_theta, cfg.rope_scaling = 10000.0, dict(scaling, rope_theta=10000.0)
    inv, amplitude = ROPE_INIT_FUNCTIONS[scaling["rope_type"]](cfg, "cpu", seq_len=S)
    cos, sin = rope_tables(S, D, 10000.0, scaling=scaling)
    angle = torch.arange(S, dtype=torch.float64)[:, None] * inv.double()
    # the other side's frequencies are fp32: each may be some roundings off, times up to 3000 positions
    tol = 16 * U * S
    assert (cos - angle.cos() * amplitude).abs().max() < tol and (sin - angle.sin() * amplitude).abs().max() < tol


# ------------------------------------------------------------------------------------------------------ token log-probabilities
def logits_case(device, rows, V, dtype, seed=0, banned=True):
    g = gen(device, seed)
    x = normal(g, rows, V, scale=2.0)
    x.scatter_add_(1, torch.randint(0, V, (rows, 4), generator=g, device=device), torch.full((rows, 4), 8.0, device=device))
    x = x.to(dtype)
    if banned and V > 8:
        x[::3, 1::4] = -math.inf
        x[1::3, 2::5] = torch.finfo(dtype).min
    tokens = torch.randint(0, V, (rows,), generator=g, device=device) // 4 * 4  # never a banned one
    return x, tokens, g


def logprobs64(x, tokens, k, T, ignore, g_lp=None, g_ent=None, g_top=None):
    z = x.double() / T
    m = z.amax(-1, keepdim=True)
    e = (z - m).exp()
    S = e.sum(-1, keepdim=True)
    p = e / S
    lp = z - m - S.log()
    fin = torch.where(p > 0, lp, torch.zeros_like(lp))
    H = -(p * fin).sum(-1, keepdim=True)
    at = tokens.clamp(min=0)[:, None]
    counts = (tokens != ignore)[:, None]
    out = {"lp": torch.where(counts, lp.gather(1, at), 0.0)[:, 0], "ent": torch.where(counts, H, 0.0)[:, 0]}
    # on the GPU a thread adds V / 512 values and 9 levels follow, on the CPU one of 8 vector lanes adds V / 8; e's exponent
    # is rounded: |z - m| U relative, and |z - m| e^-|z - m| < 0.4
    n = 40 + x.shape[1] / (512 if x.is_cuda else 8)
    out["lp_extra"] = U * (n + 4 * out["lp"].abs() + 4 * ((x.double().gather(1, at) / T - m).abs() * counts)[:, 0].nan_to_num(0, 0, 0))
    out["ent_extra"] = U * ((2 * n + 8) * ((p * (z - m).nan_to_num(0, 0, 0)).abs().sum(-1) + 1) + 4 * S.log()[:, 0].abs())
    order = torch.sort(x.double(), dim=-1, descending=True, stable=True)[1][:, :k]
    out["top_lp"] = torch.where(counts, lp.gather(1, order), 0.0)
    out["top_id"] = torch.where(counts, order, -1)
    out["top_extra"] = U * (n + 8 * out["top_lp"].abs().nan_to_num(0, 0, 0) + 8 * S.log().abs())
    if g_lp is not None or g_ent is not None or g_top is not None:
        zero = torch.zeros(x.shape[0], 1, dtype=torch.float64, device=x.device)
        G = zero if g_lp is None else g_lp.double()[:, None]
        E = zero if g_ent is None else g_ent.double()[:, None]
        total = G + (0 if g_top is None else g_top.double().sum(-1, keepdim=True))
        d = -p * (total + E * (fin + H))
        size = p * (total.abs() + E.abs() * (fin.abs() + H)) * (n + 8 + 2 * fin.abs())
        d.scatter_add_(1, at, G)
        if g_top is not None:
            d.scatter_add_(1, order, g_top.double())
            size = size + p * g_top.double().abs().sum(-1, keepdim=True) * k
        out["dx"] = d / T * counts
        out["dx_extra"] = U * (size + 4 * d.abs()) / T * counts
    return out


def run_logprobs(device, rows, V, dtype, k, T=1.0, ignore_every=0, seed=0, banned=True):
    x, tokens, g = logits_case(device, rows, V, dtype, seed, banned)
    if ignore_every:
        tokens[::ignore_every] = -100
    leaf = x.detach().requires_grad_()
    r = token_logprobs(leaf, tokens, top_k=k, temperature=T)
    g_lp, g_ent = normal(g, rows), normal(g, rows)
    g_top = normal(g, rows, k) if k else None
    ref = logprobs64(x, tokens, k, T, -100, g_lp, g_ent, g_top)
    check(r.logprobs, ref["lp"], ref["lp_extra"], "logprobs")
    check(r.entropy, ref["ent"], ref["ent_extra"], "entropy")
    outs, grads = [r.logprobs, r.entropy], [g_lp, g_ent]
    if k:
        assert torch.equal(r.top_tokens, ref["top_id"])
        check(r.top_logprobs, ref["top_lp"], ref["top_extra"], "top_logprobs")
        outs.append(r.top_logprobs)
        grads.append(g_top)
    else:
        assert r.top_logprobs is None and r.top_tokens is None
    (dx,) = torch.autograd.grad(outs, leaf, grads)
    check(dx, ref["dx"], ref["dx_extra"], "dlogits")
    with torch.no_grad():
        again = token_logprobs(x, tokens, top_k=k, temperature=T)
    assert all(a is b is None or torch.equal(a, b) for a, b in zip(again, r))


LOGIT_SHAPES = [(1, 1), (3, 2), (5, 7), (4, 8), (9, 33), (4, 511), (6, 1000), (3, 4097), (2, 32000), (2, 50257)]


@pytest.mark.parametrize("device", ON)
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("rows,V", LOGIT_SHAPES)
def test_token_logprobs(device, dtype, rows, V):
    run_logprobs(device, rows, V, dtype, min(V // 2, 20), T=1.0 if V % 2 else 0.7, ignore_every=3 if rows > 3 else 0)


@pytest.mark.parametrize("device", ON)
@pytest.mark.parametrize("k", [0, 1, 5, 63, 64])
def test_token_logprobs_alternatives(device, k):
    run_logprobs(device, 6, 2000, BF16, k, T=1.5)  # 16-bit logits: many equal ones
    run_logprobs(device, 3, 64, FP32, k, banned=False)


@gpu
@pytest.mark.parametrize("rows,V,dtype,k", [(300, 5003, BF16, 3), (8, 128256, BF16, 20), (2, 200003, FP32, 32), (2, 150000, FP16, 64)])
def test_token_logprobs_large(rows, V, dtype, k):
    run_logprobs("cuda", rows, V, dtype, k, ignore_every=7)


@pytest.mark.parametrize("device", ON)
@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_token_logprobs_alternatives_where_rows_are_orderly(device, dtype):
    """Constant rows, falling and rising ones, and rows whose best values all lie a thread's stride apart."""
    V, k = 40000, 40
    x = torch.zeros(7, V, device=device)
    x[1] = torch.arange(V, device=device) / 256.0
    x[2] = -x[1]
    for step in (2048, 4096):
        x[3 + step // 4096, ::step] = 3.0
    x[5, ::512] = 2.0
    x[6] = -0.0
    x[6, ::2] = 0.0
    # more elements of one thread's chunks than a row's list holds: each thread of 512 has chunks 512 apart
    per = 16 // torch.tensor([], dtype=dtype).element_size()
    big = torch.zeros(2, 512 * per * 80, device=device, dtype=dtype)
    big.view(2, 80, 512, per)[0, :, :8] = 1.0
    big.view(2, 80, 512, per)[1, :, ::13] = torch.arange(80, device=device, dtype=dtype)[:, None, None] / 8
    for rows in (x.to(dtype), big):
        r = token_logprobs(rows, torch.zeros(rows.shape[0], dtype=torch.int64, device=device), top_k=k)
        want = torch.sort(rows.float() + 0.0, dim=-1, descending=True, stable=True)[1][:, :k]
        assert torch.equal(r.top_tokens, want)


@pytest.mark.parametrize("device", ON)
def test_token_logprobs_rows_without_a_distribution(device):
    x = torch.randn(7, 100, device=device)
    x[0, 3] = math.nan
    x[1, 99] = math.inf
    x[2] = -math.inf
    x[3, 1:] = -math.inf  # one possible token
    tokens = torch.tensor([0, 0, 0, 0, 100, -7, -100], device=device)
    leaf = x.clone().requires_grad_()
    r = token_logprobs(leaf, tokens, top_k=2)
    assert r.logprobs[:3].isnan().all() and r.entropy[:3].isnan().all() and (r.top_tokens[:3] == -1).all() and r.top_logprobs[:3].isnan().all()
    assert r.logprobs[3] == 0 and r.entropy[3] == 0 and r.top_tokens[3].tolist() == [0, 1] and r.top_logprobs[3].tolist() == [0, -math.inf]
    assert r.logprobs[4:6].isnan().all() and r.entropy[4:6].isfinite().all()  # tokens outside the vocabulary
    assert r.logprobs[6] == 0 and r.entropy[6] == 0 and r.top_tokens[6].tolist() == [-1, -1] and r.top_logprobs[6].tolist() == [0, 0]
    (d,) = torch.autograd.grad((r.logprobs, r.entropy), leaf, (torch.ones(7, device=device), torch.ones(7, device=device)))
    assert d[:3].isnan().any(-1).all() and not d[3].any() and not d[6].any()


@pytest.mark.parametrize("device", ON)
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("V", [50, 70001])
def test_token_logprobs_masked_rows(device, dtype, V):
    """Rows that masks leave empty or nearly so, in one block and in slices: the type's lowest value everywhere (a uniform
    distribution), -inf everywhere, one finite logit at either end, whole stretches of -inf, NaN and +inf far apart."""
    low = torch.finfo(dtype).min
    x = torch.full((8, V), -math.inf, device=device, dtype=dtype)
    x[0] = low
    x[1, V - 1] = 1.0
    x[2, 0] = low
    x[3, V // 2 :] = torch.linspace(-3, 3, V - V // 2, device=device).to(dtype)
    x[4, V // 3] = math.nan
    x[5, V // 3] = math.inf
    x[6] = low
    x[6, V - 2] = 0.5
    x = x.requires_grad_()
    tokens = torch.tensor([V - 1, V - 1, 0, V - 1, 0, 0, V - 2, 3], device=device)
    r = token_logprobs(x, tokens, top_k=3)
    (d,) = torch.autograd.grad((r.logprobs[:4].sum() + r.entropy[:4].sum() + r.logprobs[6],), x)
    tol = 64 * U * math.log(V) + (V * U / 8 if device == "cpu" else 0)
    assert abs(r.logprobs[0].item() + math.log(V)) < tol and abs(r.entropy[0].item() - math.log(V)) < tol
    assert r.top_tokens[0].tolist() == [0, 1, 2]
    for i, t in ((1, V - 1), (2, 0), (6, V - 2)):
        assert r.logprobs[i] == 0 and r.entropy[i] == 0 and r.top_tokens[i, 0] == t and r.top_logprobs[i, 0] == 0
        assert not d[i].any()
    assert r.top_tokens[1].tolist() == [V - 1, 0, 1] and r.top_logprobs[1].tolist() == [0, -math.inf, -math.inf]
    z = x[3].detach().double()
    lp = torch.log_softmax(z, -1)
    assert abs(r.logprobs[3].item() - lp[V - 1].item()) < tol and d[3].isfinite().all()
    assert r.logprobs[[4, 5, 7]].isnan().all() and r.entropy[[4, 5, 7]].isnan().all() and (r.top_tokens[[4, 5, 7]] == -1).all()


@gpu
def test_token_logprobs_refuses_more_rows_than_a_launch_holds():
    x = torch.zeros(2**24 + 8, 1, device="cuda", dtype=BF16)
    with pytest.raises(RuntimeError):
        token_logprobs(x, torch.zeros(2**24 + 8, dtype=torch.int64, device="cuda"))


@pytest.mark.parametrize("device", ON)
def test_token_logprobs_shapes_strides_and_gradients(device):
    g = gen(device, 4)
    big = normal(g, 3, 4, 90, dtype=FP32)
    tokens = torch.randint(0, 40, (3, 4), generator=g, device=device)
    for x in (big[..., 7:47], big[..., ::2][..., :40], big[:, :1, :40].expand(3, 4, 40), big.transpose(0, 1)[..., :40].transpose(0, 1)):
        leaf = x.detach().requires_grad_()
        r = token_logprobs(leaf, tokens.int() if x.is_contiguous() else tokens, top_k=3)
        ref = logprobs64(x.reshape(12, 40), tokens.reshape(12), 3, 1.0, -100, torch.ones(12, device=device))
        check(r.logprobs.reshape(12), ref["lp"], ref["lp_extra"], "logprobs")
        assert r.entropy.shape == (3, 4) and r.top_tokens.shape == (3, 4, 3) and torch.equal(r.top_tokens.reshape(12, 3), ref["top_id"])
        (d,) = torch.autograd.grad(r.logprobs.sum(), leaf)
        check(d.reshape(12, 40), ref["dx"], ref["dx_extra"], "dlogits")
        (d,) = torch.autograd.grad(token_logprobs(leaf, tokens, top_k=2).top_logprobs[..., 1].sum(), leaf)
        one = torch.tensor([0.0, 1.0], device=device).expand(12, 2)
        ref = logprobs64(x.reshape(12, 40), tokens.reshape(12), 2, 1.0, -100, g_top=one)
        check(d.reshape(12, 40), ref["dx"], ref["dx_extra"], "dlogits of the second alternative")
    r = token_logprobs(big[0, 0], tokens[0, 0], top_k=1)
    assert r.logprobs.shape == () and r.top_tokens.shape == (1,)
    leaf = torch.zeros(0, 5, device=device, requires_grad=True)
    r = token_logprobs(leaf, torch.zeros(0, dtype=torch.int64, device=device), top_k=2)
    r.logprobs.sum().backward()
    assert r.top_tokens.shape == (0, 2) and leaf.grad.shape == (0, 5)


def test_token_logprobs_gradient_by_differences():
    x = normal(gen("cpu", 8), 4, 9).double().requires_grad_()
    tokens = torch.tensor([1, 8, -100, 0])
    assert torch.autograd.gradcheck(lambda t: token_logprobs(t, tokens, top_k=2, temperature=0.8)[:3], (x,))


@pytest.mark.parametrize("device", ON)
def test_token_logprobs_refusals(device):
    x, t = torch.zeros(4, 100, device=device), torch.zeros(4, dtype=torch.int64, device=device)
    for args, kw in (((x, t[:3]), {}), ((x, t[:, None]), {}), ((x, t), dict(top_k=101)), ((x, t), dict(top_k=-1)),
                     ((x, t), dict(temperature=0.0)), ((x, t), dict(temperature=math.inf)), ((x[:, :0], t), {})):
        with pytest.raises(ValueError):
            token_logprobs(*args, **kw)
    for bad in (t.float(), t.bool()):
        with pytest.raises(TypeError):
            token_logprobs(x, bad)
    with pytest.raises(TypeError):
        token_logprobs(x.int(), t)
    if device == "cuda":
        with pytest.raises(ValueError):
            token_logprobs(x, t, top_k=65)


# ---------------------------------------------------------------------------------------------------------- routing to experts
def route64(x, k, scoring, bias, groups, top_groups, renorm, scale, dw=None):
    """Row by row, from the definition."""
    x = x.double()
    T, E = x.shape
    score = torch.softmax(x, -1) if scoring == "softmax" else torch.sigmoid(x)
    key = score + (0 if bias is None else bias.double())
    if bias is None and groups == top_groups:
        key = x
    size = E // groups
    ids = []
    for row in key.tolist():
        open_ = range(E)
        if top_groups < groups:
            rating = [sum(sorted(row[g * size : (g + 1) * size], reverse=True)[:2]) for g in range(groups)]
            best = sorted(range(groups), key=lambda g: (-rating[g], g))[:top_groups]
            open_ = [e for e in open_ if e // size in best]
        ids.append(sorted(open_, key=lambda e: (-row[e], e))[:k])
    ids = torch.tensor(ids, device=x.device).view(T, k)
    s = score.gather(1, ids)
    total = s.sum(-1, keepdim=True) if renorm else torch.ones(T, 1, dtype=torch.float64, device=x.device)
    w = s / total * scale
    if dw is None:
        return w, ids
    u = dw.double() * scale
    ds = (u - (u * s / total).sum(-1, keepdim=True)) / total if renorm else u
    full = torch.zeros_like(score).scatter_(1, ids, ds)
    mag = torch.zeros_like(score).scatter_(1, ids, (u.abs() + (u * s / total).abs().sum(-1, keepdim=True)) / total if renorm else u.abs())
    if scoring == "sigmoid":
        return w, ids, full * score * (1 - score), mag * score
    inner = (full * score).sum(-1, keepdim=True)
    return w, ids, score * (full - inner), score * (mag + (mag * score).sum(-1, keepdim=True))


def run_route(device, T, E, k, scoring, bias, groups, top_groups, renorm, dtype, seed=0, scale=2.5):
    g = gen(device, seed)
    x = normal(g, T, E, dtype=dtype, scale=1.5)
    b = 0.05 * normal(g, E) if bias else None
    leaf = x.detach().requires_grad_()
    w, ids = route_experts(leaf, k, scoring, b, groups, top_groups, renorm, scale)
    dw = normal(g, T, k)
    (dx,) = torch.autograd.grad(w, leaf, dw)
    rw, rids, rdx, mag = route64(x, k, scoring, b, groups, top_groups, renorm, scale, dw)
    assert torch.equal(ids, rids)
    # scores: an exp, a sum of up to 16 values per lane and 6 levels, a division; shares: k more
    n = 40 + k
    check(w, rw, n * U * rw.abs(), "weights")
    check(dx, rdx, 2 * n * U * mag, "dlogits")
    with torch.no_grad():
        w2, ids2 = route_experts(x, k, scoring, b, groups, top_groups, renorm, scale)
    assert torch.equal(w2, w) and torch.equal(ids2, ids)


ROUTES = [(1, 1, 1, 1, 1), (5, 2, 1, 1, 1), (9, 8, 2, 1, 1), (33, 8, 8, 1, 1), (3, 13, 4, 1, 1), (17, 32, 6, 1, 1), (4, 33, 7, 1, 1),
          (6, 64, 8, 1, 1), (5, 100, 10, 1, 1), (7, 256, 8, 8, 4), (2, 256, 16, 4, 1), (3, 60, 6, 6, 2), (4, 24, 3, 12, 5), (5, 8, 2, 4, 2),
          (3, 7, 3, 7, 4), (2, 320, 8, 1, 1), (3, 512, 64, 8, 8), (2, 1000, 20, 40, 3), (2, 1024, 8, 64, 9)]


@pytest.mark.parametrize("device", ON)
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("T,E,k,groups,top_groups", ROUTES)
def test_route_experts(device, T, E, k, groups, top_groups, bias, scoring):
    for renorm, dtype in ((True, FP32), (False, BF16), (k > 1, FP16)):
        if renorm and k == 1:
            continue  # the share of one is 1, its gradient rounding noise around 0
        run_route(device, T, E, k, scoring, bias, groups, top_groups, renorm, dtype)


@gpu
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_route_experts_many_tokens(scoring):
    run_route("cuda", 2051, 8, 2, scoring, False, 1, 1, True, BF16)
    run_route("cuda", 1023, 128, 6, scoring, True, 8, 3, True, FP32)


@pytest.mark.parametrize("device", ON)
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_route_experts_ties_masks_and_poison(device, scoring):
    x = torch.zeros(7, 16, device=device)
    x[1, ::2] = 1.0
    x[2] = -math.inf  # softmax: no distribution; sigmoid: scores of 0
    x[3, :14] = -math.inf
    x[4, 5] = math.nan
    x[5] = -200.0  # sigmoid scores that 32 bits cannot hold
    x[6, 3] = torch.finfo(FP32).min
    w, ids = route_experts(x, 4, scoring, renormalize=True)
    assert ids[0].tolist() == [0, 1, 2, 3] and ids[1].tolist() == [0, 2, 4, 6] and ids[3].tolist()[:2] == [14, 15]
    assert ids[6].tolist() == [0, 1, 2, 4]
    assert all(len(set(r)) == 4 and min(r) >= 0 and max(r) < 16 for r in ids.tolist())
    assert torch.equal(w[:2], torch.full((2, 4), 0.25, device=device))
    if scoring == "softmax":
        assert w[2].isnan().all() and w[4].isnan().all() and torch.equal(w[5], torch.full((4,), 0.25, device=device))
    else:
        assert not w[2].any() and not w[5].any()
    # equal keys of equal groups: the lower group, then the lower expert; a bias of -inf closes an expert
    w, ids = route_experts(x[:2], 4, scoring, n_groups=4, topk_groups=2)
    assert ids.tolist() == [[0, 1, 2, 3], [0, 2, 4, 6]]
    bias = torch.zeros(16, device=device)
    bias[:6] = -math.inf
    assert route_experts(x[:2], 4, scoring, bias)[1].tolist() == [[6, 7, 8, 9], [6, 8, 10, 12]]
    bias[4:] = -math.inf  # fewer possible experts than choices: by index
    assert sorted(route_experts(x[:1], 4, scoring, bias)[1].tolist()[0]) == [0, 1, 2, 3]


@pytest.mark.parametrize("device", ON)
def test_route_experts_order_is_finer_than_32_bits(device):
    """Keys that 32 bits round to one value: the choice follows the scores in 64 bits."""
    x = torch.zeros(2, 64, device=device)
    x[0, 40] = 2.0 ** -22  # its sigmoid is 2^-24 above 1/2: half a step of fp32 there
    x[1] = 9.0
    x[1, 7] = 9.0 + 2.0 ** -20
    bias = torch.zeros(64, device=device)
    for groups, top_groups in ((1, 1), (8, 3)):
        _, ids = route_experts(x, 1, "sigmoid", bias, groups, top_groups)
        assert ids.tolist() == [[40], [7]]


@pytest.mark.parametrize("device", ON)
def test_route_experts_strides_and_empty(device):
    big = normal(gen(device, 9), 6, 100)
    for x in (big[:, 3:43], big[::2, :40], big[:, ::2][:, :40], big[:1, :40].expand(6, 40)):
        w, ids = route_experts(x, 3, "sigmoid")
        rw, rids = route64(x, 3, "sigmoid", None, 1, 1, True, 1.0)
        assert torch.equal(ids, rids)
        check(w, rw, 40 * U * rw, "weights")
    leaf = torch.zeros(0, 8, device=device, requires_grad=True)
    w, ids = route_experts(leaf, 2)
    w.sum().backward()
    assert w.shape == ids.shape == (0, 2) and leaf.grad.shape == (0, 8)


def test_route_experts_gradient_by_differences():
    x = normal(gen("cpu", 10), 3, 12).double().requires_grad_()
    bias = 0.1 * normal(gen("cpu", 11), 12)
    for scoring in ("softmax", "sigmoid"):
        for renorm in (False, True):
            fn = lambda t: route_experts(t, 3, scoring, bias, 4, 2, renorm, 1.5)[0]  # noqa: E731
            assert torch.autograd.gradcheck(fn, (x,))


@pytest.mark.parametrize("device", ON)
def test_route_experts_refusals(device):
    x = torch.zeros(4, 16, device=device)
    for args, kw in (((x, 0), {}), ((x, 17), {}), ((x, 2, "tanh"), {}), ((x, 2), dict(n_groups=3)), ((x, 2), dict(n_groups=4, topk_groups=5)),
                     ((x, 5), dict(n_groups=4, topk_groups=1)), ((x, 2), dict(bias=torch.zeros(15, device=device))),
                     ((x, 2), dict(scale=0.0)), ((x, 2), dict(scale=math.nan)), ((x[0], 2), {}), ((x, 2), dict(n_groups=0))):
        with pytest.raises(ValueError):
            route_experts(*args, **kw)
    with pytest.raises(TypeError):
        route_experts(x.int(), 2)
    if device == "cuda":
        with pytest.raises(ValueError):
            route_experts(torch.zeros(1, 1025, device=device), 2)
        with pytest.raises(ValueError):
            route_experts(torch.zeros(1, 256, device=device), 65)


# --------------------------------------------------------------------------------------------------------- used together
def block64(p, ids, cos, sin, cfg):
    """The block of `block` below in 64 bits; the choice of experts is passed in (it is not differentiable)."""
    x = p["embed"][p["tokens"]]
    B, S, Hd = x.shape
    h = torch.nn.functional.layer_norm(x, (Hd,), p["w1"], p["b1"], 1e-5)
    qkv = (h @ p["qkv"]).view(B, S, 3 * cfg["heads"], cfg["D"])
    n, D, R = cfg["heads"], cfg["D"], cfg["R"]
    c, s = cos.double()[:S, None], sin.double()[:S, None]
    a, b = qkv[:, :, : 2 * n, 0:R:2], qkv[:, :, : 2 * n, 1:R:2]
    rot = torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)
    qk = torch.cat([rot, qkv[:, :, : 2 * n, R:]], -1)
    q, k, v = qk[:, :, :n].transpose(1, 2), qk[:, :, n:].transpose(1, 2), qkv[:, :, 2 * n :].transpose(1, 2)
    att = (q @ k.transpose(-1, -2)) / math.sqrt(D)
    att = att.masked_fill(torch.ones(S, S, dtype=torch.bool, device=x.device).triu(1), -math.inf).softmax(-1)
    o = (att @ v).transpose(1, 2).reshape(B, S, n * D) @ p["proj"]
    x = x + o
    h = torch.nn.functional.layer_norm(x, (Hd,), p["w2"], p["b2"], 1e-5)
    t = h.view(-1, Hd)
    score = torch.sigmoid(t @ p["gate"])
    w = score.gather(1, ids)
    w = w / w.sum(-1, keepdim=True) * cfg["scale"]
    y = torch.einsum("th,ehf->tef", t, p["up"]).relu()
    y = torch.einsum("tef,efh->teh", y, p["down"])
    x = x + (y.gather(1, ids[..., None].expand(-1, -1, Hd)) * w[..., None]).sum(1).view(B, S, Hd)
    h = torch.nn.functional.layer_norm(x, (Hd,), p["w3"], p["b3"], 1e-5)
    logits = h @ p["head"]
    lp = torch.log_softmax(logits, -1)
    return logits, lp.gather(-1, p["targets"][..., None])[..., 0], -(lp.exp() * lp).sum(-1)


def block(p, cos, sin, cfg):
    """Norm, rotary attention, norm, routed experts, norm, log-probabilities, on the four operators; products in fp32."""
    x = p["embed"][p["tokens"]]
    B, S, Hd = x.shape
    n, D, R = cfg["heads"], cfg["D"], cfg["R"]
    h, res = layer_norm(x, p["w1"], p["b1"])
    qkv = apply_rope((h @ p["qkv"]).view(B, S, 3 * n, D), cos, sin, 2 * n, interleaved=True, rotary_dim=R)
    q, k, v = (qkv[:, :, i * n : (i + 1) * n].transpose(1, 2).contiguous() for i in range(3))
    att = (q @ k.transpose(-1, -2).contiguous()) / math.sqrt(D)
    att = att.masked_fill(torch.ones(S, S, dtype=torch.bool, device=x.device).triu(1), -math.inf).softmax(-1)
    o = (att @ v).transpose(1, 2).reshape(B, S, n * D) @ p["proj"]
    h, res = layer_norm(o, p["w2"], p["b2"], residual=res)
    t = h.reshape(-1, Hd)
    w, ids = route_experts(t @ p["gate"], cfg["k"], "sigmoid", p["balance"], cfg["groups"], cfg["top_groups"], True, cfg["scale"])
    y = 0
    for e in range(p["up"].shape[0]):
        share = (w * (ids == e)).sum(-1, keepdim=True)
        y = y + (t @ p["up"][e]).relu() @ p["down"][e] * share
    h, _ = layer_norm(y.view(B, S, Hd), p["w3"], p["b3"], residual=res)
    logits = h @ p["head"]
    return logits, ids, token_logprobs(logits, p["targets"])


@pytest.mark.parametrize("device", ON)
def test_operators_together_in_a_decoder_block(device):
    """A policy loss (log-probabilities and entropy) through the block, forward and every gradient against 64 bits. The fp32
    products of up to 64 terms, chained 12 deep, are off by less than 64 * 12 * 16 U relative to the gradients' norm."""
    g = gen(device, 12)
    Hd, E, F, V, B, S = 64, 8, 32, 100, 2, 11
    cfg = dict(heads=4, D=16, R=12, k=2, groups=4, top_groups=2, scale=1.5)
    shapes = dict(embed=(V, Hd), qkv=(Hd, 3 * 64), proj=(64, Hd), gate=(Hd, E), up=(E, Hd, F), down=(E, F, Hd), head=(Hd, V))
    p = {n: normal(g, *s, scale=1 / math.sqrt(s[-2])) for n, s in shapes.items()}
    for i in (1, 2, 3):
        p[f"w{i}"], p[f"b{i}"] = 1 + 0.1 * normal(g, Hd), 0.1 * normal(g, Hd)
    names = list(p)
    for n in names:
        p[n].requires_grad_()
    p["balance"] = 0.05 * normal(g, E)
    p["tokens"], p["targets"] = (torch.randint(0, V, (B, S), generator=g, device=device) for _ in range(2))
    cos, sin = rope_tables(S, cfg["R"], 10000.0, device, {"rope_type": "linear", "factor": 2.0})
    adv = normal(g, B, S)
    logits, ids, r = block(p, cos, sin, cfg)
    loss = -(r.logprobs * adv).mean() - 0.01 * r.entropy.mean()
    grads = torch.autograd.grad(loss, [p[n] for n in names])
    p64 = {n: v.detach().double().requires_grad_() if n in names else v for n, v in p.items()}
    want, lp, ent = block64(p64, ids, cos, sin, cfg)
    loss64 = -(lp * adv.double()).mean() - 0.01 * ent.mean()
    grads64 = torch.autograd.grad(loss64, [p64[n] for n in names])
    tol = 64 * 12 * 16 * U
    assert (logits - want).norm() < tol * want.norm() and abs(loss.item() - loss64.item()) < tol
    for n, a, b in zip(names, grads, grads64):
        assert (a - b).norm() < tol * b.norm(), (n, ((a - b).norm() / b.norm()).item())


@pytest.mark.parametrize("device", ON)
def test_moe_layer_routes_by_sigmoid_groups_and_bias(device):
    """The layer's own router: output and gradients equal the same layer with its weights and experts taken from 64 bits."""
    torch.manual_seed(0)
    dt = BF16 if device == "cuda" else FP32
    layer = moe.MoELayer(256, 256, 8, 2, scoring="sigmoid", n_groups=4, topk_groups=2, scale=2.0)
    for prm in layer.parameters():
        torch.nn.init.normal_(prm, std=0.05)
    layer = layer.to(device, dt)
    layer.router_bias = 0.05 * torch.randn(8).to(device)
    x = torch.randn(3, 17, 256, device=device).to(dt).requires_grad_()
    out = layer(x)
    gate = layer.gate(x.reshape(-1, 256)).detach()
    w, ids = route64(gate, 2, "sigmoid", layer.router_bias, 4, 2, True, 2.0)
    ex = layer.experts
    t = x.detach().double().reshape(-1, 256)
    want = torch.zeros_like(t)
    for e in range(8):
        gu = t @ ex.w_gate_up[e].detach().double().t()
        y = (torch.nn.functional.silu(gu[:, :256]) * gu[:, 256:]) @ ex.w_down[e].detach().double().t()
        want += y * (w * (ids == e)).sum(-1, keepdim=True)
    # three roundings to dt on the way (hidden, expert output, weight) and one at the end; and two products of 256 terms
    # summed in fp32, 256 U of the terms' absolute sum each, which is up to sqrt(256) = 16 times the sum's size
    assert (out.reshape(-1, 256).double() - want).norm() < (4 * torch.finfo(dt).eps + 2 * 256 * 16 * U) * want.norm()
    out.float().square().mean().backward()
    assert x.grad.isfinite().all() and layer.gate.weight.grad.abs().sum() > 0


@pytest.mark.parametrize("device", ON)
def test_decoder_with_partial_interleaved_rotary_and_routed_groups(device):
    from accelerate_hpc_test_amd.models.mixtral import MixtralConfig, MixtralForCausalLM

    cfg = MixtralConfig(vocab_size=128, hidden_size=256, intermediate_size=256, num_hidden_layers=2, num_attention_heads=2,
                        num_key_value_heads=1, max_position_embeddings=256, num_local_experts=8, rope_interleaved=True,
                        partial_rotary_factor=0.5, router_scoring="sigmoid", router_n_groups=4, router_topk_groups=2,
                        routed_scaling_factor=1.5, rope_scaling={"rope_type": "linear", "factor": 2.0})
    torch.manual_seed(0)
    model = MixtralForCausalLM(cfg)
    model.init_weights()
    model = model.to(device, BF16 if device == "cuda" else FP32)
    ids = torch.randint(0, 128, (1, 128), device=device)
    out = model(ids, labels=ids)
    r = token_logprobs(out.logits, ids, top_k=3)
    (out.loss - 0.01 * r.entropy.mean()).backward()
    assert cfg.rotary_dim == 64 and all(p.grad is not None and p.grad.isfinite().all() for p in model.parameters())


# ------------------------------------------------------------------------------------------------- streams, graphs, repetition
def all_operators(st):
    """One forward and backward of each operator on leaves and gradients held in `st`."""
    y, s = layer_norm(st["x"], st["w"], st["b"], 1e-5, st["res"])
    outs = [y, s, *torch.autograd.grad((y, s), (st["x"], st["res"], st["w"], st["b"]), (st["dy"], st["dres"]))]
    o = apply_rope(st["qkv"], st["cos"], st["sin"], 3, st["pos"], interleaved=True, rotary_dim=24)
    outs += [o, *torch.autograd.grad(o, st["qkv"], st["dqkv"])]
    r = token_logprobs(st["logits"], st["tokens"], top_k=5)
    outs += [*r, *torch.autograd.grad((r.logprobs, r.entropy, r.top_logprobs), st["logits"], (st["g1"], st["g2"], st["g3"]))]
    w, ids = route_experts(st["gate"], 4, "sigmoid", st["bias"], 8, 3)
    return outs + [w, ids, *torch.autograd.grad(w, st["gate"], st["dw"])]


def all_inputs(seed):
    g = gen("cuda", seed)
    st = {"x": normal(g, 300, 520, dtype=BF16), "res": normal(g, 300, 520, dtype=BF16), "w": normal(g, 520, dtype=BF16),
          "b": normal(g, 520, dtype=BF16), "qkv": normal(g, 2, 50, 5, 80, dtype=BF16), "logits": normal(g, 40, 3000, scale=3.0),
          "gate": normal(g, 70, 64)}
    for t in st.values():
        t.requires_grad_()
    st |= {"dy": normal(g, 300, 520, dtype=BF16), "dres": normal(g, 300, 520, dtype=BF16), "dqkv": normal(g, 2, 50, 5, 80, dtype=BF16),
           "pos": torch.randint(0, 100, (2, 50), generator=g, device="cuda"), "bias": 0.1 * normal(g, 64), "dw": normal(g, 70, 4),
           "tokens": torch.randint(-100, 3000, (40,), generator=g, device="cuda"), "g1": normal(g, 40), "g2": normal(g, 40),
           "g3": normal(g, 40, 5)}
    st["tokens"][st["tokens"] < 0] = -100
    st["cos"], st["sin"] = rope_tables(100, 24, 10000.0, "cuda")
    return st


@gpu
def test_operators_repeat_bit_for_bit_and_on_another_stream():
    st = all_inputs(0)
    first = all_operators(st)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        there = all_operators(st)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for a, b, c in zip(first, all_operators(st), there):
        assert torch.equal(a, b) and torch.equal(a, c)


@gpu
def test_backward_is_differentiable_once():
    """A backward that is itself recorded gives the gradients, and an error where they are differentiated again."""
    st = all_inputs(5)
    y, s = layer_norm(st["x"], st["w"], st["b"], 1e-5, st["res"])
    o = apply_rope(st["qkv"], st["cos"], st["sin"], 3, st["pos"], interleaved=True, rotary_dim=24)
    r = token_logprobs(st["logits"], st["tokens"])
    w, _ = route_experts(st["gate"], 4, "sigmoid", st["bias"], 8, 3)
    for out, leaf, grad in ((y, "x", "dy"), (o, "qkv", "dqkv"), (r.logprobs, "logits", "g1"), (w, "gate", "dw")):
        (plain,) = torch.autograd.grad(out, st[leaf], st[grad], retain_graph=True)
        (d,) = torch.autograd.grad(out, st[leaf], st[grad], create_graph=True)
        assert torch.equal(d, plain) and d.requires_grad
        with pytest.raises(RuntimeError, match="not differentiable"):
            d.float().sum().backward()


@gpu
def test_operators_in_a_captured_graph():
    """Forward and backward captured once; replays follow new inputs, with eager work and synchronisations between them."""
    st = all_inputs(1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            all_operators(st)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = all_operators(st)
    for seed in (2, 3, 2, 4):
        fresh = all_inputs(seed)
        with torch.no_grad():
            for n, t in st.items():
                t.copy_(fresh[n])
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in captured]
        for a, b in zip(got, all_operators(fresh)):
            assert torch.equal(a, b)
