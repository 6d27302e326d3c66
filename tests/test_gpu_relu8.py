"""relu kept in 8 bits (graphop.relu8_forward / relu8_backward) and the feed-forward's second half on it (op.relu_linear8).

The codes, exponents and what they stand for are whole numbers and powers of two: they are compared bit by bit with the definition."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
BLOCK = 64


def drop_scale(n, p, seed):
    """Per element 0 or 1 / (1 - p): the hash that attention_dropout_mask documents, of the element's index."""
    from bpt_amd import graphop
    if p == 0:
        return torch.ones(n)
    eid = torch.empty(n)
    return graphop.attention_dropout_mask(None, None, eid, None, torch.empty(1, 1, 1), None, p, seed).reshape(-1)


def definition(a, p=0.0, seed=0):
    """(y, codes, exps, y8) on the CPU in 64 bits; y rounded to a's type as stored, which the codes are of."""
    x = a.cpu().double().reshape(-1)
    n = x.numel()
    y = torch.where(x <= 0, torch.zeros_like(x), x)
    scale = drop_scale(n, p, seed)
    y = torch.where(scale == 0, torch.zeros_like(y), (y.float() * scale).double())
    y = y.to(a.dtype).double()
    blocks = torch.nn.functional.pad(y, (0, -n % BLOCK)).view(-1, BLOCK)
    bad = ~torch.isfinite(blocks).all(1)
    top = torch.where(bad[:, None], torch.zeros_like(blocks), blocks).amax(1)
    e = torch.full_like(top, -126.0)
    for k in range(-126, 122):                                    # the smallest exponent that reaches
        e = torch.where(255 * 2.0 ** (k - 1) < top, torch.full_like(top, float(k)), e) if k > -126 else e
    codes = torch.where(blocks > 0, (blocks / torch.exp2(e)[:, None]).round().clamp(min=1), torch.zeros_like(blocks))
    codes[bad] = (blocks[bad] != 0).double()
    y8 = codes * torch.exp2(e)[:, None]
    y8[bad] = torch.where(codes[bad] != 0, torch.full_like(codes[bad], float("nan")), torch.zeros_like(codes[bad]))
    e[bad] = 127
    flat = lambda t: t.reshape(-1)[:n].view(a.shape)
    return y.view(a.shape).to(a.dtype), flat(codes).to(torch.uint8), e.to(torch.int8), flat(y8).to(a.dtype)


def same(a, b):
    return torch.equal(torch.nan_to_num(a.cpu().float(), nan=-7.0), torch.nan_to_num(b.float(), nan=-7.0))


def check(a, p=0.0, seed=0):
    from bpt_amd import graphop
    y, codes, exps, y8 = definition(a, p, seed)
    gy, gcodes, gexps = graphop.relu8_forward(a, p, seed)
    assert same(gy, y) and torch.equal(gcodes.cpu(), codes) and torch.equal(gexps.cpu(), exps)
    dy = torch.randn(a.shape, generator=torch.Generator().manual_seed(5)).to(a.dtype).to(DEV)
    da, g8 = graphop.relu8_backward(dy, gcodes, gexps, p)
    inv = torch.tensor(1.0) / (1 - torch.tensor(p, dtype=torch.float32))
    want = torch.where(codes != 0, (dy.cpu().float() * inv).to(a.dtype), torch.zeros_like(y))
    assert same(g8, y8) and same(da, want)
    return gy, gcodes, gexps


def make(n, dtype, seed=0, spread=2.0):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(n, generator=gen) * torch.exp(spread * torch.randn(n, generator=gen))).to(TYPES[dtype]).to(DEV)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [1, 2, 7, 63, 64, 65, 127, 1000, 4095, 4096, 4097, 100003])
def test_matches_the_definition(n, dtype):
    check(make(n, dtype))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("p", [0.1, 0.5])
def test_dropout(p, dtype):
    check(make(20011, dtype), p, 1234567890123)


@pytest.mark.parametrize("dtype", TYPES)
def test_every_magnitude(dtype):
    """Blocks whose largest is each power of two and its neighbours, subnormal ones included; borders of the exponent's rule."""
    t = TYPES[dtype]
    tops = torch.tensor([m * 2.0 ** k for k in range(-140, 128) for m in (1.0, 1.9921875, 1.99609375)], dtype=torch.float64).to(t)
    a = make(tops.numel() * BLOCK, dtype, spread=0.0).view(-1, BLOCK)
    a = (torch.sigmoid(a.float()) * tops.to(DEV).float()[:, None]).to(t)
    a[:, 17] = tops.to(DEV)
    a[:, 33] = -a[:, 33]
    check(a)


@pytest.mark.parametrize("dtype", TYPES)
def test_rounding_is_off_by_half_a_step(dtype):
    a = make(64 * 500, dtype, spread=1.0)
    y, codes, exps = check(a)
    y8 = codes.view(-1, 64).double() * torch.exp2(exps.double())[:, None]
    err, step = (y.view(-1, 64).double() - y8).abs(), torch.exp2(exps.double())[:, None]
    small = (y.view(-1, 64).double() < step / 2) & (y.view(-1, 64) > 0)
    assert (err[~small] <= (step / 2).expand_as(err)[~small]).all() and (err <= step).all()
    assert ((step / 2) <= y.view(-1, 64).double().amax(1, keepdim=True) * 2.0 ** -8 * 1.01).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_infinities_and_nan_mark_their_block(dtype):
    a = make(64 * 6 + 10, dtype, spread=0.0)
    a[70], a[130], a[200], a[64 * 6 + 3] = float("nan"), float("inf"), float("-inf"), float("nan")
    _, _, exps = check(a)
    assert exps.tolist()[1] == 127 and exps.tolist()[2] == 127 and exps.tolist()[3] != 127 and exps.tolist()[6] == 127


def test_all_negative_and_zeros():
    a = torch.cat([-torch.rand(200), torch.zeros(200), torch.full((10,), -0.0)]).to(DEV)
    y, codes, exps = check(a)
    assert not codes.any() and not y.any() and (exps == -126).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_tensors_off_16_bytes(dtype):
    buf = make(1001, dtype)
    check(buf[1:])


def test_nothing():
    from bpt_amd import graphop
    y, codes, exps = graphop.relu8_forward(torch.empty((0, 64), device=DEV))
    assert y.shape == codes.shape == (0, 64) and exps.shape == (0,)
    da, y8 = graphop.relu8_backward(y, codes, exps)
    assert da.shape == y8.shape == (0, 64)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape,outer", [((1, 64), 16), ((33, 100), 48), ((2, 5, 256), 64), ((300, 512), 128)], ids=str)
@pytest.mark.parametrize("p", [0.0, 0.1])
def test_relu_linear(shape, outer, p, dtype):
    """float32 products sum up to 512 terms of size |u||v|, off by (terms + 4) 2^-24 of the sum of their absolute values whatever their order;
    bfloat16 results are rounded once more, dY before the mask too (2^-8 each), and 1 / (1 - p) is one rounding on the way."""
    from bpt_amd import op
    t = TYPES[dtype]
    gen = torch.Generator().manual_seed(3)
    inner = shape[-1]
    a = torch.randn(shape, generator=gen).to(t)
    w = (torch.randn((outer, inner), generator=gen) / inner ** 0.5).to(t)
    b = torch.randn(outer, generator=gen).to(t)
    do = torch.randn(shape[:-1] + (outer,), generator=gen).to(t)
    ad, wd, bd = (x.to(DEV).requires_grad_(True) for x in (a, w, b))
    out = op.relu_linear8(ad, wd, bd, p, 99)
    ga, gw, gb = torch.autograd.grad(out, (ad, wd, bd), do.to(DEV))
    y, codes, _, y8 = definition(a, p, 99)
    d = lambda x: x.double().reshape(-1, x.shape[-1])
    H = torch.finfo(t).eps / 2
    def close(got, u, v, more=0.0, roundings=1, name=""):
        want, terms = u @ v + more, u.shape[1]
        bound = (terms + 4) * 2.0 ** -24 * (u.abs() @ v.abs() + (more.abs() if torch.is_tensor(more) else 0)) + roundings * H * want.abs()
        err = (got.cpu().double().reshape(want.shape) - want).abs() - bound
        assert (err <= 0).all(), (name, err.max())
    close(out.detach(), d(y), w.double().t(), b.double()[None], 2 if dtype == "bf16" else 1, "out")
    inv = 1 / (1 - p)
    mask = d(codes) != 0
    dyw = d(do) @ w.double() * inv * mask
    bound = (outer + 8) * 2.0 ** -24 * (d(do).abs() @ w.double().abs()) * inv + (3 * H) * dyw.abs()
    assert ((ga.cpu().double().reshape(dyw.shape) - dyw).abs() <= bound).all()
    close(gw, d(do).t(), d(y8), 0.0, 1, "dweight")
    ones = torch.ones(d(do).shape[0], 1, dtype=torch.float64)
    close(gb[:, None], d(do).t(), ones, 0.0, 1, "dbias")
    with torch.no_grad():
        again = op.relu_linear8(ad, wd, bd, p, 99)
    assert torch.equal(again, out) or p == 0.0
    assert (again.float() - out.float()).abs().max() <= 2 * H * out.float().abs().max() + 1e-5


def test_relu_linear_keeps_a_byte_an_activation():
    from bpt_amd import op
    a = torch.randn((4096, 2048), device=DEV, requires_grad=True)
    w = torch.randn((64, 2048), device=DEV, requires_grad=True)
    kept = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: kept.append(t) or t, lambda t: t):
        op.relu_linear8(a, w, None, 0.1, 1)
    sizes = sorted(t.numel() * t.element_size() for t in kept)
    assert sum(sizes) == a.numel() + a.numel() // 64 + w.numel() * 4


def test_relu_linear_needs_no_gradient_of_some():
    from bpt_amd import op
    a, w, b = torch.randn(20, 64, device=DEV), torch.randn(8, 64, device=DEV), torch.randn(8, device=DEV)
    do = torch.randn(20, 8, device=DEV)
    full = [t.clone().requires_grad_(True) for t in (a, w, b)]
    want = torch.autograd.grad(op.relu_linear8(*full), full, do)
    for i in range(3):
        args = [a, w, b]
        args[i] = args[i].clone().requires_grad_(True)
        (got,) = torch.autograd.grad(op.relu_linear8(*args), args[i], do)
        assert torch.equal(got, want[i])


def test_relu_linear_of_no_rows_and_to_no_outputs():
    from bpt_amd import op
    for rows, outer in ((0, 16), (5, 0), (0, 0)):
        a, w, b = (torch.randn(*s, device=DEV, requires_grad=True) for s in ((rows, 64), (outer, 64), (outer,)))
        y = op.relu_linear8(a, w, b)
        grads = torch.autograd.grad(y, (a, w, b), torch.ones_like(y))
        assert y.shape == (rows, outer) and [g.shape for g in grads] == [a.shape, w.shape, b.shape] and not any(g.any() for g in grads)


@pytest.mark.parametrize("dtype", TYPES)
def test_relu_linear_inside_autocast(dtype):
    """The products are of the tensors as they are."""
    from bpt_amd import op
    a, w = (torch.randn(s, device=DEV).to(TYPES[dtype]).requires_grad_(True) for s in ((20, 64), (8, 64)))
    do = torch.randn(20, 8, device=DEV).to(TYPES[dtype])
    want = torch.autograd.grad(op.relu_linear8(a, w), (a, w), do)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        out = op.relu_linear8(a, w)
        got = torch.autograd.grad(out, (a, w), do)
    assert out.dtype == TYPES[dtype] and all(torch.equal(x, y) for x, y in zip(got, want))


def test_replays_of_a_captured_pair_match_the_eager_one():
    from bpt_amd import graphop
    a, dy = make(50000, "f32"), make(50000, "f32", 1)
    step = lambda: graphop.relu8_forward(a, 0.1, 7) + graphop.relu8_backward(dy, *graphop.relu8_forward(a, 0.1, 7)[1:], 0.1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for i in range(3):
        a.copy_(make(50000, "f32", i + 2))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(captured, step()))


def test_refusals():
    from bpt_amd import graphop, op
    a = torch.randn(4, 64, device=DEV)
    y, codes, exps = graphop.relu8_forward(a)
    with pytest.raises(RuntimeError, match="unsupported dtype"):
        graphop.relu8_forward(a.double())
    with pytest.raises(RuntimeError, match="a must be contiguous"):
        graphop.relu8_forward(a.t())
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        graphop.relu8_forward(a.cpu())
    for p in (-0.1, 1.0, float("nan")):
        with pytest.raises(ValueError, match="dropout_p"):
            graphop.relu8_forward(a, p)
    with pytest.raises(ValueError, match="codes must have shape"):
        graphop.relu8_backward(a, codes[:2].contiguous(), exps)
    with pytest.raises(ValueError, match="exps must have shape"):
        graphop.relu8_backward(a, codes, exps[:2].contiguous())
    with pytest.raises(ValueError, match="uint8"):
        graphop.relu8_backward(a, exps, exps)
    with pytest.raises(ValueError, match="last axis"):
        op.relu_linear8(a[:, :0].contiguous(), torch.randn(8, 0, device=DEV))
    with pytest.raises(ValueError, match="weight must be"):
        op.relu_linear8(a, torch.randn(8, 32, device=DEV))
    w = torch.randn(8, 64, device=DEV, requires_grad=True)
    with pytest.raises(RuntimeError, match="twice"):
        torch.autograd.grad(op.relu_linear8(a, w).sum(), w, create_graph=True)
