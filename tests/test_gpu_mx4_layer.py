"""Layers in 4 bits put together: several on one input, a decoder layer trained and served, graphs, streams."""
import pytest
import torch

from conftest import bits_equal, make_gen, randn_bf16
from oracle import mx4 as oracle

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def T():
    import triton_int8_amd
    return triton_int8_amd


def layers_of(T, dev, k, features, bias=False, seed=0):
    gen = make_gen(seed)
    out = []
    for n in features:
        m = T.Mx4Linear(k, n, bias=bias, device=dev)
        with torch.no_grad():
            m.weight.copy_(randn_bf16(gen, n, k, std=k ** -0.5))
            if bias:
                m.bias.copy_(randn_bf16(gen, n))
        out.append(m)
    return out


@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("tokens", [1, 37, 300])
def test_several_layers_on_one_input(T, dev, tokens, bias):
    """The bits of separate calls: outputs, gradients of the weights, and x's, added up as autograd adds it up."""
    layers = layers_of(T, dev, 200, (96, 40, 513), bias)
    gen = make_gen(tokens)
    x = randn_bf16(gen, 2, tokens, 200).to(dev)
    dys = [randn_bf16(gen, 2, tokens, m.out_features).to(dev) for m in layers]
    got = []
    for together in (True, False):
        for m in layers:
            m.zero_grad()
        h = x.clone().requires_grad_()
        ys = T.mx4.linears(h, layers) if together else [m(h) for m in layers]
        torch.autograd.backward(ys, dys)
        got.append([*(y.detach() for y in ys), h.grad, *(p.grad for m in layers for p in m.parameters())])
        with torch.no_grad():
            got[-1] += list(T.mx4.linears(x, layers) if together else [m(x) for m in layers])
    assert len(got[0]) == len(got[1]) and all(bits_equal(a, b) for a, b in zip(*got))


def test_bias_gradient(T, dev):
    (m,) = layers_of(T, dev, 64, (1000,), True)
    dy = randn_bf16(make_gen(2), 777, 1000).to(dev)
    m(torch.zeros(777, 64, dtype=torch.bfloat16, device=dev, requires_grad=True)).backward(dy)
    want, mag = dy.double().sum(0), dy.double().abs().sum(0)
    assert bool(((m.bias.grad.double() - want).abs() <= 2.0 ** -8 * want.abs() + 777 * 2.0 ** -24 * mag).all())


def test_gradients_against_differences(T, dev):
    """Values that have codes, moved to their neighbours: the layer is exact there, and so are the differences that its gradients stand for."""
    gen = make_gen(4)
    tokens, k, n = 24, 32, 16
    grid = lambda *s: (torch.randint(-1, 2, s, generator=gen).float() * torch.randint(1, 3, s, generator=gen) / 2 * (torch.rand(s, generator=gen) < 0.5)).bfloat16()  # noqa: E731
    x, w, dy = grid(tokens, k), grid(n, k), grid(tokens, n)
    for t in (x, w, dy):        # (so that every group has the same scale, with room for a step more)
        t[:, 0] = t[0] = 2.0
    (m,) = layers_of(T, dev, k, (n,))

    def value(x, w):
        with torch.no_grad():
            m.weight.copy_(w.to(dev))
            return float((m(x.to(dev)).double() * dy.to(dev).double()).sum())
    xd = x.to(dev).requires_grad_()
    with torch.no_grad():
        m.weight.copy_(w.to(dev))
    m(xd).backward(dy.to(dev))
    base = value(x, w)
    y = x.double() @ w.double().t()
    assert base == float((y.bfloat16().double() * dy.double()).sum())
    dx, dw = xd.grad.double().cpu(), m.weight.grad.double().cpu()
    assert torch.equal(dx, (dy.double() @ w.double()).bfloat16().double()) and torch.equal(dw, (dy.double().t() @ x.double()).bfloat16().double())
    exact_x, exact_w = dy.double() @ w.double(), dy.double().t() @ x.double()
    for r, c in ((1, 1), (5, 30), (23, 7)):
        up = x.clone()
        up[r, c] += 0.5
        rounding = 2.0 ** -8 * float((y[r].abs() * dy[r].double().abs()).sum()) * 2
        assert abs(value(up, w) - base - 0.5 * float(exact_x[r, c])) <= rounding
    for r, c in ((1, 1), (15, 30), (7, 7)):
        up = w.clone()
        up[r, c] += 0.5
        rounding = 2.0 ** -8 * float((y[:, r].abs() * dy[:, r].double().abs()).sum()) * 2
        assert abs(value(x, up) - base - 0.5 * float(exact_w[r, c])) <= rounding


def decoder(T, dev, hidden=512, heads=4, mlp=1280):
    layer = T.DecoderLayer(hidden, heads, mlp, scheme="mx4", device=dev)
    gen = make_gen(hidden)
    with torch.no_grad():
        for p in layer.parameters():
            p.copy_(randn_bf16(gen, *p.shape, std=p.shape[1] ** -0.5) if p.dim() == 2 else 1.0 + randn_bf16(gen, *p.shape, std=0.1))
    return layer


def test_decoder_layer_trains(T, dev, monkeypatch):
    """Forward and backward; the projections that share an input give the bits of separate calls."""
    layer = decoder(T, dev)
    assert sum(isinstance(m, T.Mx4Linear) for m in layer.modules()) == 7
    gen = make_gen(1)
    x, dy = randn_bf16(gen, 2, 100, 512).to(dev), randn_bf16(gen, 2, 100, 512).to(dev)
    got = []
    for together in (True, False):
        if not together:
            monkeypatch.setattr(T.mx4, "all_as_written", lambda layers: False)
        layer.zero_grad()
        h = x.clone().requires_grad_()
        y = layer(h)
        y.backward(dy)
        got.append([y.detach(), h.grad, *(p.grad for p in layer.parameters())])
    assert all(torch.isfinite(t).all() and t.abs().sum() > 0 for t in got[0])
    assert all(bits_equal(a, b) for a, b in zip(*got))
    # beside its twin in bf16: 4 bits leave an eighth of an element's size at most, over seven products
    twin = T.DecoderLayer(512, 4, 1280, int8=False, device=dev)
    twin.copy_weights_from(layer)
    with torch.no_grad():
        a, b = layer(x).double() - x.double(), twin(x).double() - x.double()
    assert float((a - b).norm() / b.norm()) < 0.5


def served(T, layer, x, cache, rotary, counts=None):
    """The layer on new tokens, piece by piece: the oracle's norm, each linear on its own, torch's sums."""
    import triton_int8_amd.decoder as D
    B, S, H = x.shape
    eps = layer.input_norm.eps
    norm = lambda t, m, r=None: oracle.norm(t.cpu(), m.weight.detach().cpu(), eps, None if r is None else r.cpu())  # noqa: E731
    h = norm(x, layer.input_norm)[0].to(x.device)
    at = (cache.positions[:, None] + torch.arange(S, device=x.device)).flatten().long()
    q, k, v = (m(h).view(1, B * S, layer.heads, layer.head_dim) for m in (layer.q_proj, layer.k_proj, layer.v_proj))
    q, k = D._RopeFunction.apply(q, k, rotary[0][at].contiguous(), rotary[1][at].contiguous())
    q, k, v = (t.reshape(B, S, layer.heads, layer.head_dim) for t in (q, k, v))
    cache.append(k, v, counts=counts)
    a = layer.o_proj(cache.attend(q, counts=counts).view(B, S, H))
    h, _, x = (t.to(a.device) for t in norm(a, layer.post_norm, x))
    return x + layer.down_proj(T.ops.swiglu(layer.gate_proj(h), layer.up_proj(h)))


@pytest.mark.parametrize("packed", [False, True])
def test_decoder_layer_serves(T, dev, packed):
    """Prompts, parts of them and single tokens, ragged ones among them: the bits of the pieces."""
    layer = decoder(T, dev)
    rotary = T.decoder.rope_tables(256, layer.head_dim, dev)
    x = randn_bf16(make_gen(3), 3, 120, 512).to(dev)
    counts = torch.tensor([40, 17, 0], dtype=torch.int32, device=dev)
    one, other = (T.Cache4(3, 200, 4, layer.head_dim, page_size=16, device=dev) for _ in range(2))
    with torch.no_grad():
        want = [served(T, layer, x[:, :40], one, rotary, counts)]
        want += [served(T, layer, x[:, a:b], one, rotary) for a, b in ((40, 41), (41, 46), (46, 120))]
        if packed:
            layer.pack()
            assert not list(layer.input_norm.buffers()) and all(m.packed for m in layer._linears())
        got = [layer.serve(x[:, :40], other, rotary, counts=counts)]
        got += [layer.serve(x[:, a:b], other, rotary) for a, b in ((40, 41), (41, 46), (46, 120))]
    rows = torch.arange(40, device=dev) < counts[:, None]
    assert bits_equal(got[0][rows], want[0][rows]) and all(bits_equal(a, b) for a, b in zip(got[1:], want[1:]))
    assert torch.equal(one.lengths, other.lengths)


def test_blank_rows_may_hold_anything(T, dev):
    layer = decoder(T, dev).pack()
    rotary = T.decoder.rope_tables(64, layer.head_dim, dev)
    counts = torch.tensor([5, 9], dtype=torch.int32, device=dev)
    x = randn_bf16(make_gen(3), 2, 9, 512).to(dev)
    dirty = x.clone()
    dirty[0, 5:] = float("nan")
    with torch.no_grad():
        ys = [layer.serve(t, T.Cache4(2, 64, 4, layer.head_dim, device=dev), rotary, counts=counts, blank=True) for t in (x, dirty)]
    assert bits_equal(*ys) and not ys[0][0, 5:].any()


def test_hooks_and_replaced_parts_are_seen(T, dev):
    """A module of the layer that does more than it is written to do is called."""
    layer = decoder(T, dev)
    rotary = T.decoder.rope_tables(64, layer.head_dim, dev)
    x = randn_bf16(make_gen(3), 2, 9, 512).to(dev)
    serve = lambda: layer.serve(x, T.Cache4(2, 64, 4, layer.head_dim, device=dev), rotary)  # noqa: E731
    plain = serve()
    seen = []
    for m in (layer.q_proj, layer.post_norm):
        handle = m.register_forward_hook(lambda mod, i, o: seen.append(mod))
        serve()
        handle.remove()
    assert seen == [layer.q_proj, layer.post_norm]
    layer.gate_proj.forward = lambda h: torch.zeros(*h.shape[:-1], 1280, dtype=h.dtype, device=h.device)
    assert not torch.equal(serve(), plain)
    del layer.gate_proj.forward
    assert bits_equal(serve(), plain)


def test_other_schemes_are_not_packed(T, dev):
    with pytest.raises(ValueError, match="mx4"):
        T.DecoderLayer(256, 2, 256, device=dev).pack()


# (the last of them in parts along the tokens, with a workspace)
@pytest.mark.parametrize("tokens,k,n", [(5, 300, 200), (130, 512, 96), (4000, 64, 72)])
def test_captured_steps(T, dev, tokens, k, n):
    """A step recorded once and replayed with other inputs, eager work between the replays, another graph beside it."""
    gen = make_gen(tokens)
    sets = [[randn_bf16(gen, tokens, k).to(dev), randn_bf16(gen, n, k, std=0.05).to(dev), randn_bf16(gen, tokens, n).to(dev)] for _ in range(3)]
    want = [[t.clone() for t in T.mx4.linear_fwd_bwd(*s)] for s in sets]
    steps = [T.GraphedStep(T.mx4.linear_fwd_bwd, *sets[0]) for _ in range(2)]
    for turn in range(4):
        for step in steps:
            got = step(*sets[turn % 3])
            torch.cuda.synchronize()
            assert all(bits_equal(a, b) for a, b in zip(got, want[turn % 3]))
            T.mx4.linear_fwd_bwd(*sets[(turn + 1) % 3])


def test_captured_layer_with_its_backward(T, dev):
    """(Leaves of the step's own: none that an eager graph outside holds.)"""
    weights = [randn_bf16(make_gen(n), n, 256, std=0.06).to(dev) for n in (96, 500)]
    x, dy = randn_bf16(make_gen(5), 70, 256).to(dev), [randn_bf16(make_gen(6), 70, w.shape[0]).to(dev) for w in weights]

    def step(x, *dys):
        leaves = [t.detach().requires_grad_() for t in (x, *weights)]
        ys = T.mx4.Mx4LinearFunction.apply(*leaves)
        return (*(y.detach() for y in ys), *torch.autograd.grad(ys, leaves, dys))
    want = [t.clone() for t in step(x, *dy)]
    graphed = T.GraphedStep(step, x, *dy)
    for _ in range(3):
        got = graphed(x, *dy)
        torch.cuda.synchronize()
        assert all(bits_equal(a, b) for a, b in zip(got, want))
        step(x, *dy)


def test_captured_norm_and_products(T, dev):
    layer = decoder(T, dev).pack()
    w = layer.input_norm.weight.detach()
    x, r = (randn_bf16(make_gen(s), 33, 512).to(dev) for s in (1, 2))

    def run(x, r):
        q, s, rstd, h = T.ops.rmsnorm_quant(x, w, 1e-5, residual=r)
        p, t, *_ = T.ops.rmsnorm_quant(x, w, 1e-5, to="int8", group=128)
        return T.mx4.gemm_nt(q, s, *layer.q_proj.quantised()), rstd, h, T.mx4.dequant(q, s, 512), T.ops.dequant_row(p, t)
    with torch.no_grad():
        graphed = T.GraphedStep(run, x, r)
        for a, b in ((x, r), (r, x), (x, x)):
            want = [t.clone() for t in run(a, b)]
            got = graphed(a, b)
            torch.cuda.synchronize()
            assert all(bits_equal(u, v) for u, v in zip(got, want))


# (the first launch in two parts along the contraction, with a workspace; the second for all products)
@pytest.mark.parametrize("sizes", [((5, 40, 16384), (300, 100, 600)), ((20, 300, 1000), (20, 70, 1000), (20, 900, 1000))])
def test_captured_products_together(T, dev, sizes):
    gen = make_gen(1)
    inputs = [[t for m, n, k in sizes for t in (*T.mx4.quant_row(randn_bf16(gen, m, k).to(dev)), *T.mx4.quant_row(randn_bf16(gen, n, k, std=0.1).to(dev)))] for _ in range(2)]

    def run(*t):
        return tuple(T.mx4.gemm_nt_multi([t[i:i + 4] for i in range(0, len(t), 4)]))
    want = [[t.clone() for t in run(*i)] for i in inputs]
    steps = [T.GraphedStep(run, *inputs[0]) for _ in range(2)]
    for turn in range(4):
        for step in steps:
            got = step(*inputs[turn % 2])
            torch.cuda.synchronize()
            assert all(bits_equal(a, b) for a, b in zip(got, want[turn % 2]))
            run(*inputs[(turn + 1) % 2])


def test_on_other_streams(T, dev):
    """Calls on two streams at once, each behind what made its inputs there."""
    gen = torch.Generator(device=dev).manual_seed(3)
    x, w, dy = (torch.randn(s, generator=gen, device=dev).bfloat16() for s in ((3000, 512), (640, 512), (3000, 640)))
    want = T.mx4.linear_fwd_bwd(x, w, dy)
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                a, b, c = ((t.float() * 2.0).mul_(0.5).bfloat16() for t in (x, w, dy))      # (exact)
                got.append(T.mx4.linear_fwd_bwd(a, b, c))
    torch.cuda.synchronize()
    assert all(bits_equal(u, v) for g in got for u, v in zip(g, want))


@pytest.mark.parametrize("native", [True, False])
def test_both_ways_from_python(T, dev, native, monkeypatch):
    """The calls made from C++ and those made from Python are the same."""
    gen = make_gen(7)
    x, w, dy, r = (randn_bf16(gen, *s).to(dev) for s in ((50, 256), (70, 256), (50, 70), (50, 256)))
    nw = randn_bf16(gen, 256).to(dev)

    def run():
        q, s = T.mx4.quant_row(x)
        out = [q, s, *T.mx4.quant_row(x.view(5, 10, 256)), *T.mx4.quant_col_t(x), *T.mx4.quant_row_col_t(x), T.mx4.dequant(q, s, 256), *T.mx4.linear_fwd_bwd(x, w, dy)]
        out += [T.mx4.gemm_nt(q, s, *T.mx4.quant_row(w), out_dtype=d) for d in (torch.bfloat16, torch.float32)]
        out += [y for n in (1, 2, 3) for y in T.mx4.gemm_nt_multi([(q, s, *T.mx4.quant_row(w)), (q, s, q, s), (q[3:], s[:, 3:], q, s)][:n])]
        for kw in (dict(), dict(residual=r), dict(to="int8"), dict(to="int8", group=128, residual=r, inv_mode=1)):
            out += T.ops.rmsnorm_quant(x, nw, 1e-5, **kw)
        out += [T.ops.dequant_row(*T.ops.rmsnorm_quant(x, nw, 1e-5, to="int8", group=g)[:2]) for g in (0, 128)]
        return out
    assert T._lib.native() is not None
    want = run()
    if not native:
        monkeypatch.setattr(T._lib, "native", lambda: None)
    got = run()
    assert all(a.dtype == b.dtype and a.shape == b.shape and a.is_contiguous() and bits_equal(a, b) for a, b in zip(got, want))


def test_inference_mode(T, dev):
    (m,) = layers_of(T, dev, 256, (96,))
    x = randn_bf16(make_gen(1), 7, 256).to(dev)
    with torch.no_grad():
        want = m(x)
    with torch.inference_mode():
        y = m(x)
        assert y.is_inference() and bits_equal(y.clone(), want)
        w = torch.ones(256, dtype=torch.bfloat16, device=dev)
        assert all(t.is_inference() for t in (*T.ops.rmsnorm_quant(x, w, 1e-5, residual=x), *T.mx4.quant_row_col_t(x)))
    assert not any(t.is_inference() for t in (*T.ops.rmsnorm_quant(x, w.clone(), 1e-5, residual=x), *T.mx4.quant_row_col_t(x)))
    assert not m(x.requires_grad_()).is_inference()


def test_weights_that_change_are_quantised_again(T, dev):
    """Nothing is kept of an unpacked weight, however it is changed."""
    (m,) = layers_of(T, dev, 256, (96,))
    x = randn_bf16(make_gen(1), 7, 256).to(dev)
    with torch.no_grad():
        first = m(x)
        m.weight.data.mul_(2.0)
        assert bits_equal(m(x), first * 2)


def test_packed_layers_are_saved_and_loaded(T, dev):
    """Into a layer that is packed too."""
    for bias in (False, True):
        (m,) = layers_of(T, dev, 520, (96,))
        m = T.Mx4Linear(520, 96, bias=bias, device=dev).pack()
        x = randn_bf16(make_gen(1), 7, 520).to(dev)
        other = T.Mx4Linear(520, 96, bias=bias, device=dev).pack()
        with torch.no_grad():
            assert not bits_equal(m(x), other(x))
            other.load_state_dict({k: v.clone() for k, v in m.state_dict().items()})
            assert bits_equal(m(x), other(x)) and set(m.state_dict()) == {"codes", "scales"} | ({"bias"} if bias else set())


@pytest.mark.parametrize("native", [True, False])
def test_products_of_column_slices(T, dev, native, monkeypatch):
    """Slices of columns that begin at a tile, in place, by the call from C++ and by the one from Python."""
    if not native:
        monkeypatch.setattr(T._lib, "native", lambda: None)
    gen = make_gen(4)
    a, b = randn_bf16(gen, 40, 1300), randn_bf16(gen, 70, 1300)
    (qa, sa), (qb, sb) = T.mx4.quant_row(a.to(dev)), T.mx4.quant_row(b.to(dev))
    want = T.mx4.gemm_nt(*T.mx4.quant_row(a[:, 512:1024].to(dev)), *T.mx4.quant_row(b[:, 512:1024].to(dev)))
    part = slice(256, 512)
    assert bits_equal(T.mx4.gemm_nt(qa[:, part], sa[2:4], qb[:, part], sb[2:4]), want)
    assert bits_equal(T.mx4.dequant(qa[:, part], sa[2:4], 512), T.mx4.dequant(*T.mx4.quant_row(a[:, 512:1024].to(dev)), 512))


def test_tangents_and_traces_are_refused(T, dev):
    from torch.autograd import forward_ad
    x, w = randn_bf16(make_gen(1), 7, 256).to(dev), torch.ones(256, dtype=torch.bfloat16, device=dev)
    layer = T.Mx4Linear(256, 96, device=dev).requires_grad_(False)
    with forward_ad.dual_level():
        d = forward_ad.make_dual(x, x)
        for call in (lambda: layer(d), lambda: T.ops.rmsnorm_quant(d, w, 1e-5)):
            with pytest.raises(ValueError, match="tangent"):
                call()
    for call in (layer, T.mx4.quant_row, lambda t: T.ops.rmsnorm_quant(t, w, 1e-5)[0]):
        with pytest.raises(ValueError, match="traced"):
            torch.jit.trace(call, (x,), check_trace=False)


def test_broadcast_inputs_and_gradients(T, dev):
    """An input that is one row expanded, and a gradient that is one number expanded: what copies of them give; the row's gradient is the sum of the copies'."""
    (m,) = layers_of(T, dev, 256, (96,))
    row = randn_bf16(make_gen(1), 256).to(dev)
    grads = []
    for expanded in (True, False):
        leaf = (row.clone() if expanded else row.expand(5, 256).clone()).requires_grad_()
        m.weight.grad = None
        y = m(leaf.expand(5, 256) if expanded else leaf)
        (y.sum() if expanded else (y * torch.ones_like(y)).sum()).backward()
        grads.append((y.detach(), m.weight.grad, leaf.grad if expanded else leaf.grad.sum(0)))
    assert all(bits_equal(a, b) for a, b in zip(*grads))


def test_the_same_weight_twice(T, dev):
    """Its gradient is the sum of both uses'."""
    (m,) = layers_of(T, dev, 256, (96,))
    x, dy = randn_bf16(make_gen(1), 7, 256).to(dev), [randn_bf16(make_gen(s), 7, 96).to(dev) for s in (2, 3)]
    single = []
    for d in dy:
        m.weight.grad = None
        m(x).backward(d)
        single.append(m.weight.grad)
    m.weight.grad = None
    a, b = T.mx4.linears(x, (m, m))
    assert bits_equal(a, b)
    torch.autograd.backward((a, b), dy)
    assert bits_equal(m.weight.grad, single[0] + single[1]) or bits_equal(m.weight.grad, single[1] + single[0])


def test_threads(T, dev):
    """Calls from several threads at once, each on a stream of its own."""
    import threading
    work = []
    for n, k, tokens in ((96, 256, 50), (640, 512, 300), (64, 1000, 7)):
        gen = make_gen(n)
        x, w, dy = (randn_bf16(gen, *s).to(dev) for s in ((tokens, k), (n, k), (tokens, n)))
        work.append(((x, w, dy), [t.clone() for t in T.mx4.linear_fwd_bwd(x, w, dy)]))
    torch.cuda.synchronize()
    wrong = []

    def run(inputs, want):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got = T.mx4.linear_fwd_bwd(*inputs)
                torch.cuda.current_stream().synchronize()
                if not all(bits_equal(a, b) for a, b in zip(got, want)):
                    wrong.append(inputs[0].shape)
    threads = [threading.Thread(target=run, args=w) for w in work]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
