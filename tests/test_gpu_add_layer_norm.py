"""op.add_layer_norm (layer norm of a sum, forward and backward) against the formula in 64 bits.

Tolerances, from the arithmetic.  E is half a step of the type that sums are held in (2^-24; 2^-53 for float64), F half a step of the
result's (2^-8 for bfloat16).  A lane adds up to 32 values one after the other before lanes are added in at most 9 steps, so a mean of
values v is off by at most about 42 E mean|v|; what follows is a handful of roundings.  K = 64 E times the sum of the absolute values of
an expression's terms bounds each of them.  xhat is off by K (|z| + mean|z|) rstd (the difference of nearby numbers), relative errors of
rstd come through the variance and are of the order of that of xhat.  The row sums of dweight and dbias: a lane adds at most
rows / 2 values, then at most 8 rows of a workgroup, then 32 + 16 partial sums: (rows / 2 + 64) E times the sum of absolute values."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f64": torch.float64}


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def make(shape, dtype, seed=0, residual=True, affine=True, shift=0.0):
    gen = torch.Generator().manual_seed(seed)
    rand = lambda s, a=1.0: (torch.randn(s, generator=gen, dtype=torch.float64) * a).to(dtype)
    t = dict(x=(rand(shape, 0.5) + shift).to(dtype), dy=rand(shape, 0.25))
    t["residual"] = rand(shape) if residual else None
    t["weight"] = (1 + rand(shape[-1:], 0.2).double()).to(dtype) if affine else None
    t["bias"] = rand(shape[-1:], 0.3) if affine else None
    return t


def reference(t, eps):
    """{name: (value, bound without the result's own rounding)} in 64 bits."""
    dtype = t["x"].dtype
    E = half_step(torch.float64 if dtype == torch.float64 else torch.float32)
    cols = t["x"].shape[-1]
    d = {n: (v.double().reshape(-1, cols) if n in ("x", "residual", "dy") else v.double()) for n, v in t.items() if v is not None}
    z = d["x"] + d.get("residual", 0.0)
    w, b = d.get("weight", torch.ones(cols, dtype=torch.float64)), d.get("bias", torch.zeros(cols, dtype=torch.float64))
    mean = z.mean(1, keepdim=True)
    rstd = 1 / ((z - mean).square().mean(1, keepdim=True) + eps).sqrt()
    xhat = (z - mean) * rstd
    K = 64 * E
    dx = K * ((z.abs() + z.abs().mean(1, keepdim=True)) * rstd + xhat.abs() * (1 + (z.abs().mean(1, keepdim=True) * rstd)))     # of xhat
    y = xhat * w + b
    g = d["dy"] * w
    m1, m2 = g.mean(1, keepdim=True), (g * xhat).mean(1, keepdim=True)
    dz = rstd * (g - m1 - xhat * m2)
    a2 = (g * xhat).abs().mean(1, keepdim=True)
    dz_b = rstd * (K * (g.abs() + g.abs().mean(1, keepdim=True) + xhat.abs() * a2) + dx * m2.abs() + xhat.abs() * (g.abs() * dx).mean(1, keepdim=True))
    dz_b = dz_b + dz.abs() * K * (1 + z.abs().mean(1, keepdim=True) * rstd)                            # rstd's own
    n = (z.size(0) / 2 + 64) * E
    out = {"y": (y, dx * w.abs() + K * (xhat * w).abs() + K * b.abs()), "dz": (dz, dz_b),
           "dweight": ((d["dy"] * xhat).sum(0), n * (d["dy"] * xhat).abs().sum(0) + (d["dy"].abs() * dx).sum(0)),
           "dbias": (d["dy"].sum(0), n * d["dy"].abs().sum(0))}
    return out


def close(got, want, name, dtype):
    value, bound = want
    got = got.detach().cpu().double().reshape(value.shape)
    bound = bound + half_step(dtype) * value.abs() + torch.finfo(torch.float32).tiny
    worst = ((got - value).abs() - bound).max().item() if value.numel() else 0.0
    assert worst <= 0, f"{name}: beyond its bound by {worst:.3e}"


def check(t, eps=1e-5, dev=None):
    from bpt_amd import op
    dev = dev or {n: None if v is None else v.to(DEV).requires_grad_(n != "dy") for n, v in t.items()}
    y = op.add_layer_norm(dev["x"], dev["residual"], dev["weight"], dev["bias"], eps)
    names = [n for n in ("x", "residual", "weight", "bias") if dev[n] is not None]
    grads = dict(zip(names, torch.autograd.grad(y, [dev[n] for n in names], dev["dy"])))
    ref = reference(t, eps)
    dtype = t["x"].dtype
    assert y.dtype == dtype and y.shape == t["x"].shape
    close(y, ref["y"], "y", dtype)
    close(grads["x"], ref["dz"], "dx", dtype)
    if "residual" in grads:
        assert torch.equal(grads["residual"], grads["x"])
    for n in ("weight", "bias"):
        if n in grads:
            close(grads[n], ref["d" + n], "d" + n, dtype)
    with torch.no_grad():
        assert torch.equal(op.add_layer_norm(dev["x"], dev["residual"], dev["weight"], dev["bias"], eps), y)
    return y, grads


SHAPES = [(1, 512), (3, 1), (5, 2), (5, 3), (7, 7), (2, 4), (6, 9), (33, 300), (129, 301), (64, 513), (1000, 40), (17, 1024), (9, 2047), (9, 4096), (5, 4097),
          (3, 8192), (3, 8200), (4, 20001), (2, 3, 5, 64), (512,), (5000, 512)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_matches_the_formula(shape, dtype):
    check(make(shape, TYPES[dtype]))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("residual,affine", [(False, True), (True, False), (False, False)])
@pytest.mark.parametrize("cols", [65, 512])
def test_without_residual_or_weights(cols, residual, affine, dtype):
    check(make((37, cols), TYPES[dtype], residual=residual, affine=affine))


@pytest.mark.parametrize("dtype", ["f32", "f64"])
def test_rows_far_from_zero(dtype):
    """The variance is that of the differences, not a difference of sums."""
    check(make((40, 512), TYPES[dtype], shift=1000.0))


def test_rows_of_one_value():
    """Variance 0: xhat is 0 and the gradient rstd (g - mean g), rstd = eps^-1/2."""
    t = make((8, 256), torch.float32, residual=False)
    t["x"] = torch.full((8, 256), 0.75)
    check(t)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("cols", [64, 301])
def test_tensors_off_16_bytes(cols, dtype):
    t = make((50, cols), TYPES[dtype])
    dev = {}
    for n, v in t.items():
        buf = torch.empty(v.numel() + 1, dtype=v.dtype, device=DEV)
        dev[n] = buf[1:].view(v.shape).copy_(v.to(DEV)).detach().requires_grad_(n != "dy")
        assert dev[n].data_ptr() % 16 != 0
    check(t, dev=dev)


def test_no_rows():
    from bpt_amd import op
    x = torch.empty((0, 64), device=DEV, requires_grad=True)
    w, b = (torch.ones(64, device=DEV, requires_grad=True) for _ in range(2))
    y = op.add_layer_norm(x, None, w, b)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.empty_like(y))
    assert y.shape == dx.shape == (0, 64) and not dw.any() and not db.any()


def test_nan_stays_in_its_row_and_columns_sums():
    from bpt_amd import op
    t = make((20, 300), torch.float32)
    clean = op.add_layer_norm(*(t[n].to(DEV) for n in ("x", "residual", "weight", "bias")))
    t["x"][7, 123] = float("nan")
    t["x"][11, 4] = float("inf")
    y = op.add_layer_norm(*(t[n].to(DEV) for n in ("x", "residual", "weight", "bias")))
    rows = torch.ones(20, dtype=torch.bool)
    rows[[7, 11]] = False
    assert torch.isnan(y[~rows.to(DEV)]).all() and torch.equal(y[rows.to(DEV)], clean[rows.to(DEV)])


def test_the_same_bits_every_time_and_on_another_stream():
    t = make((3000, 512), torch.float32)
    y, grads = check(t)
    side = torch.cuda.Stream()
    for stream in (torch.cuda.current_stream(), side):
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            y2, grads2 = check(t)
        torch.cuda.synchronize()
        assert torch.equal(y, y2) and all(torch.equal(grads[n], grads2[n]) for n in grads)


def test_gradient_against_differences():
    from bpt_amd import op
    t = make((6, 33), torch.float64)
    args = tuple(t[n].to(DEV).requires_grad_(True) for n in ("x", "residual", "weight", "bias"))
    assert torch.autograd.gradcheck(lambda *a: op.add_layer_norm(*a), args)
    assert torch.autograd.gradgradcheck(lambda *a: op.add_layer_norm(*a), args)


def test_gradients_of_some_inputs_only():
    from bpt_amd import op
    t = {n: v.to(DEV) for n, v in make((300, 96), torch.float32).items()}
    names = ("x", "residual", "weight", "bias")
    full = [t[n].clone().requires_grad_(True) for n in names]
    want = torch.autograd.grad(op.add_layer_norm(*full), full, t["dy"])
    for i in range(4):
        args = [t[n] for n in names]
        args[i] = args[i].clone().requires_grad_(True)
        (got,) = torch.autograd.grad(op.add_layer_norm(*args), args[i], t["dy"])
        assert torch.equal(got, want[i])
    x = t["x"].clone().requires_grad_(True)                       # (no residual, no weight: the places move up)
    b = t["bias"].clone().requires_grad_(True)
    dx, db = torch.autograd.grad(op.add_layer_norm(x, None, None, b), (x, b), t["dy"])
    assert torch.equal(db, want[3]) and torch.isfinite(dx).all()


def test_one_tensor_twice():
    """x is residual too: its gradient is both."""
    from bpt_amd import op
    x = make((10, 64), torch.float32)["x"].to(DEV).requires_grad_(True)
    dy = torch.randn_like(x)
    z = (2 * x.detach()).requires_grad_(True)
    (got,) = torch.autograd.grad(op.add_layer_norm(x, x), x, dy)
    (want,) = torch.autograd.grad(op.add_layer_norm(z), z, dy)
    assert torch.equal(got, 2 * want)


def test_replays_of_a_captured_pass_match_the_eager_one():
    from bpt_amd import op
    t = make((700, 320), torch.float32)
    dev = {n: v.to(DEV) for n, v in t.items()}
    leaves = [dev[n].requires_grad_(True) for n in ("x", "residual", "weight", "bias")]

    def step():
        y = op.add_layer_norm(*leaves)
        return (y.detach(),) + torch.autograd.grad(y, leaves, dev["dy"])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for i in range(4):
        with torch.no_grad():
            for n in ("x", "residual", "dy"):
                dev[n].copy_(make((700, 320), torch.float32, seed=i + 1)[n])
        graph.replay()
        torch.cuda.synchronize()
        for got, want in zip(captured, step()):
            assert torch.equal(got, want)


def test_refusals():
    from bpt_amd import op
    t = {n: v.to(DEV) for n, v in make((4, 64), torch.float32).items()}
    x, r, w, b = (t[n] for n in ("x", "residual", "weight", "bias"))
    with pytest.raises(RuntimeError, match="x must be contiguous"):
        op.add_layer_norm(x.t(), None)
    with pytest.raises(RuntimeError, match="residual must be a CUDA tensor"):
        op.add_layer_norm(x, r.cpu())
    with pytest.raises(ValueError, match="residual must have shape"):
        op.add_layer_norm(x, r[:1].contiguous())
    with pytest.raises(RuntimeError, match="one dtype"):
        op.add_layer_norm(x, r, w.double(), b)
    with pytest.raises(ValueError, match="bias must have shape"):
        op.add_layer_norm(x, r, w, b[:32].contiguous())
    with pytest.raises(RuntimeError, match="unsupported dtype"):
        op.add_layer_norm(x.half())
    with pytest.raises(ValueError, match="eps"):
        op.add_layer_norm(x, eps=-1.0)
    with pytest.raises(ValueError, match="last axis"):
        op.add_layer_norm(x[:, :0].contiguous())
