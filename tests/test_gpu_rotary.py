"""GPU tests of qk_norm_rope: forward, backward, layouts, padding, graphs, against the formulas in 64 bits."""

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32 = 2.0 ** -24       # half a step of a 32-bit float


@pytest.fixture(scope="module")
def rot():
    import flash_attention_amd.rotary as rot

    return rot


def reference(x, w, table, positions, eps, interleaved, dout=None):
    """x [rows, D] float64, positions [rows]; returns out, its bound's scale, and with dout: dx, its scale, dw, its scale"""
    R = table.shape[1]
    pos = positions.clamp(0, table.shape[0] - 1)
    c, s = table[pos, : R // 2].double(), table[pos, R // 2:].double()
    first = torch.arange(0, R, 2) if interleaved else torch.arange(R // 2)
    second = first + (1 if interleaved else R // 2)
    pad, far = positions < 0, positions >= table.shape[0]
    r = 1 / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    y = x * r * w

    def turn(v, sign):
        o, m = v.clone(), v.abs()
        a, b = v[:, first], v[:, second]
        o[:, first], o[:, second] = a * c - sign * b * s, sign * a * s + b * c
        m[:, first], m[:, second] = (a * c).abs() + (b * s).abs(), (a * s).abs() + (b * c).abs()
        return o, m

    out, mag = turn(y, 1)
    out[pad], out[far] = 0, float("nan")
    if dout is None:
        return out, mag
    g, gm = turn(dout, -1)
    g[far] = float("nan")                 # (an output that is NaN whatever the inputs: so are its gradients, the weights' among them)
    xhat, t = x * r, g * w
    dot = (t * xhat).mean(-1, keepdim=True)
    dx = r * (t - xhat * dot)
    dxm = r * (gm * w.abs() + xhat.abs() * (gm * w.abs() * xhat.abs()).mean(-1, keepdim=True))
    live = ~pad
    dw, dwm = (g * xhat)[live].sum(0), (gm * xhat.abs())[live].sum(0)
    dx[pad], dx[far] = 0, float("nan")
    return out, mag, dx, dxm, dw, dwm


def rows(t):
    """[B, H, L, D] or [T, H, D] -> [rows, D] in the order (b, l, h)"""
    t = t.detach().cpu().double()
    return (t.transpose(1, 2) if t.ndim == 4 else t).reshape(-1, t.shape[-1])


def close(got, want, mag, dtype, steps):
    """one rounding to the type, and `steps` roundings of 32 bits against the size of what is added up"""
    u = torch.finfo(dtype).eps / 2
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    tol = u * want.abs() + steps * F32 * mag * (1 + u) + 1e-37 + (2.0 ** -25 if dtype == torch.float16 else 0)
    fine = ~torch.isnan(want)
    assert bool(((got - want).abs() <= tol)[fine].all()), float(((got - want).abs() - tol)[fine].max())


def check(rot, layout, B, L, H, Hk, D, R, dtype, interleaved, wdtype="same", positions="random", grad=True, eps=1e-6, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed)

    def operand(h):
        x = torch.randn(B, L, h, D, generator=g).mul(scale).to(dtype)
        if layout == "thd":
            return x.reshape(B * L, h, D).to(DEV)
        return x.to(DEV).transpose(1, 2) if layout == "inner" else x.transpose(1, 2).contiguous().to(DEV)

    q, k = operand(H), operand(Hk)
    wt = None if wdtype is None else dtype if wdtype == "same" else wdtype
    wq, wk = (None if wt is None else (1 + 0.2 * torch.randn(D, generator=g)).to(wt).to(DEV) for _ in "qk")
    table = rot.rotary_table(2 * L + 3, R, device=DEV)
    if positions is None:
        pos, full = None, torch.arange(L).repeat(B) if layout != "thd" else torch.arange(B * L)
        if layout == "thd":
            table = rot.rotary_table(B * L, R, device=DEV)
    else:
        shape = (B * L,) if layout == "thd" else (B, L) if positions != "shared" else (L,)
        pos = torch.randint(0, 2 * L + 3, shape, generator=g)
        if positions == "holes":
            pos[torch.rand(shape, generator=g) < 0.3] = -1
            pos.view(-1)[-1] = 2 * L + 3
            pos.view(-1)[0] = 2 ** 31 - 1
        full = pos.reshape(-1) if positions != "shared" else pos.repeat(B)
        pos = pos.to(torch.int32 if seed % 2 else torch.int64).to(DEV)
    leaves = [t for t in (q, k, wq, wk) if t is not None]
    for t in leaves:
        t.requires_grad_(grad)
    qo, ko = rot.qk_norm_rope(q, k, wq, wk, table, pos, eps=eps, interleaved=interleaved)
    assert qo.shape == q.shape and ko.dtype == dtype
    assert [a for a, n in zip(qo.stride(), q.shape) if n > 1] == [a for a, n in zip(q.stride(), q.shape) if n > 1]      # (a dimension of one has no stride)
    dq, dk = torch.randn(q.shape, generator=g).to(dtype).to(DEV), torch.randn(k.shape, generator=g).to(dtype).to(DEV)
    grads = torch.autograd.grad((qo, ko), leaves, (dq, dk)) if grad else ()
    for i, (x, w, h, o, d) in enumerate(((q, wq, H, qo, dq), (k, wk, Hk, ko, dk))):
        p = full.repeat_interleave(h)
        wd = torch.ones(D, dtype=torch.float64) if w is None else w.detach().cpu().double()
        out, mag, dx, dxm, dw, dwm = reference(rows(x), wd, table.cpu(), p, eps, interleaved, rows(d))
        # sum of D squares in partial sums of at most 16 and a tree: 12 roundings of r at most, two for x r w, three for the rotation
        close(rows(o), out, mag, dtype, 24)
        if grad:
            close(rows(grads[i]), dx, dxm, dtype, 64)
            assert [a for a, n in zip(grads[i].stride(), x.shape) if n > 1] == [a for a, n in zip(x.stride(), x.shape) if n > 1]
            if w is not None:
                # a lane adds at most all rows one after the other
                if torch.isnan(dw).any():
                    assert bool(torch.isnan(grads[2 + i]).all())
                else:
                    close(grads[2 + i].cpu().double(), dw, dwm, w.dtype, p.numel() + 64)


DT = pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])


@DT
@pytest.mark.parametrize("layout", ["thd", "bhld", "inner"])
@pytest.mark.parametrize("D,R", [(64, 64), (128, 128), (256, 256), (32, 32), (128, 64), (256, 32), (64, 16)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_wide(rot, dtype, layout, D, R, interleaved):
    check(rot, layout, 2, 37, 6, 2, D, R, dtype, interleaved, seed=D + R)


@DT
@pytest.mark.parametrize("layout", ["thd", "bhld", "inner"])
@pytest.mark.parametrize("D,R", [(2, 2), (80, 80), (96, 48), (10, 6), (512, 512), (512, 256), (66, 64), (128, 24), (300, 300)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_any_head_dim(rot, dtype, layout, D, R, interleaved):
    check(rot, layout, 3, 11, 5, 1, D, R, dtype, interleaved, seed=D + R + 1)


@DT
@pytest.mark.parametrize("positions", [None, "shared", "holes"])
@pytest.mark.parametrize("layout", ["thd", "bhld"])
@pytest.mark.parametrize("D", [64, 80])
def test_positions(rot, dtype, positions, layout, D):
    if positions == "shared" and layout == "thd":
        pytest.skip("packed tokens have a position each")
    check(rot, layout, 2, 50, 3, 3, D, D // 2 if D == 64 else D, dtype, False, positions=positions, seed=3)


@DT
@pytest.mark.parametrize("wdtype", [None, torch.float32, "same"])
@pytest.mark.parametrize("D", [128, 80])
def test_weights(rot, dtype, wdtype, D):
    check(rot, "inner", 1, 29, 4, 2, D, D, dtype, False, wdtype=wdtype, seed=5)


@DT
@pytest.mark.parametrize("B,L,H,Hk,D", [(1, 1, 1, 1, 64), (1, 1, 32, 8, 128), (700, 1, 5, 5, 64), (1, 3001, 7, 1, 128), (4, 515, 12, 12, 64), (2, 400, 9, 3, 80)])
def test_sizes(rot, dtype, B, L, H, Hk, D):
    """from one row to launches whose lane groups take several heads and whose backward strides over its rows"""
    check(rot, "bhld", B, L, H, Hk, D, D, dtype, False, seed=7)
    check(rot, "inner", B, L, H, Hk, D, D, dtype, True, seed=8, grad=False)


@DT
def test_many_rows(rot, dtype):
    check(rot, "bhld", 2, 2048, 24, 8, 128, 128, dtype, False, seed=11)


@pytest.mark.parametrize("dtype,scale", [(torch.float32, 1e-12), (torch.float32, 1e12), (torch.bfloat16, 1e15), (torch.float16, 1e-6), (torch.float16, 1e3)])
def test_small_and_large_values(rot, dtype, scale):
    """the norm's 32-bit sum neither overflows nor loses eps against the mean where the result is a normal number"""
    check(rot, "thd", 1, 33, 4, 2, 64, 64, dtype, False, seed=13, scale=scale, grad=dtype != torch.float16)


def test_rows_of_zeros_and_nan(rot):
    q = torch.zeros(3, 2, 64, device=DEV)
    q[1, 0, 5] = float("nan")
    q[2] = 1
    table = rot.rotary_table(4, 64, device=DEV)
    out, _ = rot.qk_norm_rope(q, q, None, None, table)
    assert bool((out[0] == 0).all()) and bool(torch.isnan(out[1, 0]).all()) and bool(torch.isfinite(out[1, 1]).all()) and bool(torch.isfinite(out[2]).all())


def test_unaligned_rows_and_slices_of_a_projection(rot):
    B, L, H, D = 2, 19, 4, 64
    fused = torch.randn(B, L, 3 * H * D, device=DEV).bfloat16()
    q, k = (fused[..., i * H * D:(i + 1) * H * D].unflatten(2, (H, D)).transpose(1, 2) for i in (0, 1))
    table = rot.rotary_table(64, D, device=DEV)
    a = rot.qk_norm_rope(q, k, None, None, table)
    b = rot.qk_norm_rope(q.contiguous(), k.contiguous(), None, None, table)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    odd = torch.randn(B, H, L, D + 1, device=DEV).bfloat16()[..., 1:]
    for x, y in zip(rot.qk_norm_rope(odd, odd, None, None, table), rot.qk_norm_rope(odd.contiguous(), odd.contiguous(), None, None, table)):
        torch.testing.assert_close(x, y, rtol=2.0 ** -7, atol=0)       # (another summation order: a step of bfloat16 at most)
    spread = torch.randn(B, H, L, 2 * D, device=DEV).bfloat16()[..., ::2]
    for x, y in zip(rot.qk_norm_rope(spread, spread, None, None, table), rot.qk_norm_rope(spread.contiguous(), spread.contiguous(), None, None, table)):
        assert torch.equal(x, y)


def test_gradient_against_differences(rot):
    """the chain with a scalar loss against central differences in 64 bits"""
    g = torch.Generator().manual_seed(1)
    q, k = torch.randn(1, 2, 5, 64, generator=g), torch.randn(1, 1, 5, 64, generator=g)
    wq, wk = 1 + 0.1 * torch.randn(64, generator=g), 1 + 0.1 * torch.randn(64, generator=g)
    table = rot.rotary_table(9, 32, device=DEV)
    pos = torch.tensor([3, 0, 8, 1, 2])
    a, b = torch.randn(q.shape, generator=g), torch.randn(k.shape, generator=g)
    leaves = [t.to(DEV).requires_grad_() for t in (q, k, wq, wk)]
    o = rot.qk_norm_rope(*leaves, table, pos.to(DEV))
    grads = torch.autograd.grad((o[0] * a.to(DEV)).sum() + (o[1] * b.to(DEV)).sum(), leaves)

    def loss(q, k, wq, wk):
        out = 0
        for x, w, d in ((q, wq, a), (k, wk, b)):
            y, _ = reference(rows(x), w.double(), table.cpu(), pos.repeat_interleave(x.shape[1]), 1e-6, False)
            out = out + (y * rows(d)).sum()
        return float(out)

    base = [t.double() for t in (q, k, wq, wk)]
    for i, gr in enumerate(grads):
        flat = base[i].reshape(-1)
        for j in range(0, flat.numel(), max(1, flat.numel() // 7)):
            h, keep = 1e-5, float(flat[j])
            flat[j] = keep + h
            up = loss(*base)
            flat[j] = keep - h
            down = loss(*base)
            flat[j] = keep
            # the third difference is h^2 and the 32-bit result off by some 2^-18 of terms up to about 10
            assert abs(float(gr.reshape(-1)[j]) - (up - down) / (2 * h)) < 1e-4


def test_partial_gradients_and_double_backward(rot):
    table = rot.rotary_table(8, 64, device=DEV)
    q, k, w = torch.randn(2, 3, 8, 64, device=DEV), torch.randn(2, 1, 8, 64, device=DEV), torch.ones(64, device=DEV)
    full = [t.clone().requires_grad_() for t in (q, k, w, w)]
    want = torch.autograd.grad(sum((o * o * o).sum() for o in rot.qk_norm_rope(*full, table)), full)
    for only in range(4):
        args = [t.clone().requires_grad_(i == only) for i, t in enumerate((q, k, w, w))]
        (got,) = torch.autograd.grad(sum((o * o * o).sum() for o in rot.qk_norm_rope(*args, table)), [args[only]])
        assert torch.equal(got, want[only])
    args = [t.clone().requires_grad_() for t in (q, k, w, w)]
    qo, ko = rot.qk_norm_rope(*args, table)
    (g,) = torch.autograd.grad((qo * qo).sum(), [args[0]], create_graph=True)        # (k's output takes no part)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_broadcast_operands(rot):
    """operands, positions and incoming gradients with strides of zero, one weight for both sides"""
    g = torch.Generator().manual_seed(12)
    B, H, Hk, L, D = 3, 4, 2, 37, 64
    table = rot.rotary_table(L + 9, D, device=DEV)
    q0, k0 = (torch.randn(*s, generator=g).to(DEV).requires_grad_() for s in ((1, H, L, D), (B, 1, L, D)))
    w = (1 + 0.2 * torch.randn(D, generator=g)).to(DEV).requires_grad_()
    pos = torch.randint(0, L + 9, (1, L), generator=g)
    q, k = q0.expand(B, H, L, D), k0.expand(B, Hk, L, D)
    o = rot.qk_norm_rope(q, k, w, w, table, pos.to(DEV).expand(B, L))
    gq, gk, gw = torch.autograd.grad([t.sum() for t in o], (q0, k0, w))
    dws = []
    for x, h, y, got, dims in ((q, H, o[0], gq, 0), (k, Hk, o[1], gk, 1)):
        full = pos.repeat(B, 1).reshape(-1).repeat_interleave(h)
        out, mag, dx, dxm, dw, dwm = reference(rows(x), w.detach().cpu().double(), table.cpu(), full, 1e-6, False, torch.ones(B * L * h, D, dtype=torch.float64))
        close(rows(y), out, mag, torch.float32, 24)
        back = lambda t: t.reshape(B, L, h, D).transpose(1, 2).sum(dims, keepdim=True)  # noqa: E731
        close(rows(got), rows(back(dx)), rows(back(dxm)), torch.float32, 64 + 3)
        dws.append((dw, dwm))
    close(gw.cpu().double(), dws[0][0] + dws[1][0], dws[0][1] + dws[1][1], torch.float32, B * L * H + 65)


def test_only_one_output_used(rot):
    table = rot.rotary_table(8, 64, device=DEV)
    q, k = torch.randn(5, 3, 64, device=DEV, requires_grad=True), torch.randn(5, 1, 64, device=DEV, requires_grad=True)
    qo, _ = rot.qk_norm_rope(q, k, None, None, table)
    gq, gk = torch.autograd.grad(qo.sum(), (q, k), allow_unused=True)
    assert float(gq.abs().sum()) > 0 and (gk is None or float(gk.abs().sum()) == 0)


def test_captured_forward_and_backward(rot):
    """a captured training step against the eager one, replayed with other work between"""
    table = rot.rotary_table(64, 128, device=DEV)
    q, k, wq, wk = (torch.randn(*s, device=DEV).bfloat16().requires_grad_() for s in ((2, 8, 40, 128), (2, 2, 40, 128), (128,), (128,)))
    dq, dk = torch.randn_like(q), torch.randn_like(k)

    def step():
        o = rot.qk_norm_rope(q, k, wq, wk, table)
        return (*o, *torch.autograd.grad(o, (q, k, wq, wk), (dq, dk)))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for i in range(5):
        with torch.no_grad():
            q.copy_(torch.randn_like(q))
            dq.copy_(torch.randn_like(q))
        graph.replay()
        torch.randn(1 << 18, device=DEV).sum().item()
        want = step()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_other_stream_and_reproducible(rot):
    table = rot.rotary_table(1024, 64, device=DEV)
    leaves = [torch.randn(*s, device=DEV).half().requires_grad_() for s in ((4, 12, 1000, 64), (4, 12, 1000, 64), (64,), (64,))]

    def step():
        o = rot.qk_norm_rope(*leaves, table)
        return (*o, *torch.autograd.grad(o, leaves, [t.detach() for t in o]))

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert all(torch.equal(a, b) for a, b in zip(step(), want))


def test_compiled(rot):
    table = rot.rotary_table(64, 64, device=DEV)
    leaves = [torch.randn(*s, device=DEV).bfloat16().requires_grad_() for s in ((2, 4, 40, 64), (2, 2, 40, 64), (64,), (64,))]

    def loss(q, k, wq, wk):
        a, b = rot.qk_norm_rope(q * 1.0, k * 1.0, wq, wk, table)
        return (a.float() ** 2).sum() + b.float().sum()

    want = torch.autograd.grad(loss(*leaves), leaves)
    got = torch.autograd.grad(torch.compile(loss, fullgraph=True, backend="aot_eager")(*leaves), leaves)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_empty(rot):
    table = rot.rotary_table(4, 64, device=DEV)
    q, k, w = torch.zeros(0, 3, 64, device=DEV, requires_grad=True), torch.zeros(0, 1, 64, device=DEV), torch.ones(64, device=DEV, requires_grad=True)
    o, _ = rot.qk_norm_rope(q, k, w, None, table)
    assert o.shape == (0, 3, 64)
    o.sum().backward()
    assert float(w.grad.abs().sum()) == 0


def test_refusals(rot):
    table = rot.rotary_table(8, 64, device=DEV)
    q, k, w = torch.zeros(2, 3, 8, 64, device=DEV), torch.zeros(2, 1, 8, 64, device=DEV), torch.ones(64, device=DEV)
    call = lambda **kw: rot.qk_norm_rope(**{**dict(q=q, k=k, q_weight=w, k_weight=w, table=table), **kw})  # noqa: E731
    for bad in (dict(q=q.cpu()), dict(q=q[0, 0]), dict(k=k[:1]), dict(k=k[..., :32]), dict(k=k.half()), dict(q=q.double(), k=k.double()), dict(q_weight=w[:32]), dict(q_weight=w.half()),
                dict(table=table.double()), dict(table=table[:, :63]), dict(table=table.cpu()), dict(table=table[:, ::2]), dict(table=rot.rotary_table(8, 128, device=DEV)),
                dict(positions=torch.zeros(8, device=DEV)), dict(positions=torch.zeros(7, dtype=torch.int32, device=DEV)), dict(positions=torch.zeros(8, dtype=torch.int32)),
                dict(eps=-1.0), dict(eps=float("nan")), dict(q=torch.zeros(2, 3, 8, 63, device=DEV), k=torch.zeros(2, 1, 8, 63, device=DEV))):
        with pytest.raises((ValueError, TypeError)):
            call(**bad)
    for bad in ((0, 64), (8, 63), (8, 0)):
        with pytest.raises(ValueError):
            rot.rotary_table(*bad)
