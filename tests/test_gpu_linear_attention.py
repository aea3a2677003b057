"""functional.linear_attention, its gradients and its step for single tokens against the
recurrence in 64 bits: lengths from nothing to several segments, heads that no tile
divides, padded batches, decays from none to all, states, layouts, streams, graphs.

Bounds (u = 2^-24).  Every result is a sum of products of decays and inputs; with A the
same sum of magnitudes, f32 arithmetic is within N u A: N counts the additions on the
longest path (a head's width, a chunk, one a chunk behind it), some for pieces left out
of f32 products (2^-22) and the relative error of e^d, up to (16 + 4 |d|) u for the |d|
< 88 that is not 0.  From bf16 inputs the scores and the states that outputs read may be
rounded to bf16 once, 2^-8 A.  A decay's gradient sums q dq and k dk behind its token,
unrounded ones."""
import math

import pytest
import torch

from tests import row_ref as R

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f32": torch.float32}
U = R.U


def _F():
    from pratchya_amd import functional
    return functional


def recurrence(q, k, v, g, state, lengths, scale, dout, dstate):
    """All results in 64 bits, by the recurrences themselves; CPU arrays."""
    B, T, H, D = q.shape
    E = v.shape[-1]
    live = torch.ones(T, B, 1, dtype=torch.bool)
    if lengths is not None:
        live = (torch.arange(T)[:, None] < lengths[None, :])[..., None]
    zero = torch.zeros((), dtype=torch.float64)
    q, k, v, do = (torch.where(live[..., None], t.double().movedim(1, 0), zero) for t in (q, k, v, dout))
    a = torch.where(live, torch.exp(g.double().movedim(1, 0)), 1 + zero)[..., None, None]
    S = torch.zeros(B, H, D, E, dtype=torch.float64) if state is None else state.double().clone()
    out, dq, kept = torch.empty_like(v), torch.empty_like(q), []
    for t in range(T):
        kept.append(S)
        S = a[t] * S + k[t][..., :, None] * v[t][..., None, :]
        out[t] = scale * (q[t][..., None] * S).sum(-2)
        dq[t] = scale * (do[t][..., None, :] * S).sum(-1)
    Rr = torch.zeros_like(S) if dstate is None else dstate.double().clone()
    dk, dv, dg = torch.empty_like(k), torch.empty_like(v), torch.empty(T, B, H, dtype=torch.float64)
    for t in range(T - 1, -1, -1):
        Rr = Rr + scale * q[t][..., :, None] * do[t][..., None, :]
        dk[t] = (Rr * v[t][..., None, :]).sum(-1)
        dv[t] = (Rr * k[t][..., :, None]).sum(-2)
        Rr = a[t] * Rr
        dg[t] = (Rr * kept[t]).sum((-1, -2))
    dk, dv = torch.where(live[..., None], dk, zero), torch.where(live[..., None], dv, zero)
    dg = torch.where(live, dg, zero)
    back = [x.movedim(0, 1) for x in (out, dq, dk, dv, dg)]
    return dict(out=back[0], state=S, dq=back[1], dk=back[2], dv=back[3], dg=back[4], dstate=Rr)


def reference(q, k, v, g, state, lengths, scale, dout, dstate):
    want = recurrence(q, k, v, g, state, lengths, scale, dout, dstate)
    mag = recurrence(*(None if t is None else t.abs() for t in (q, k, v)), g, None if state is None else state.abs(),
                     lengths, abs(scale), dout.abs(), None if dstate is None else dstate.abs())
    T, D, E = q.shape[1], q.shape[-1], v.shape[-1]
    N = 700 + D + E + T / 8
    rel = N * U
    half = 2.0 ** -8 if q.dtype == torch.bfloat16 else 0.0
    tiny = 1e-30
    bound = {n: (rel + half) * mag[n] + tiny for n in ("out", "dq", "dk", "dv")}
    bound.update({n: rel * mag[n] + tiny for n in ("state", "dstate")})
    terms = (q.double().abs() * mag["dq"]).sum(-1) + (k.double().abs() * mag["dk"]).sum(-1)
    if lengths is not None:
        terms = torch.where((torch.arange(T)[None, :] < lengths[:, None])[..., None], terms.nan_to_num(0), 0.0)
    ends = 0.0 if dstate is None else (mag["state"] * dstate.double().abs()).sum((-1, -2))[:, None]
    bound["dg"] = 2 * rel * (terms.flip(1).cumsum(1).flip(1) + ends) + tiny
    return want, bound


def make(B, T, H, D, E, dtype, seed=0, gates="any", gdt=torch.float32):
    gen = torch.Generator().manual_seed(seed)
    q, k = (torch.randn((B, T, H, D), generator=gen).to(dtype) for _ in range(2))
    v, dout = (torch.randn((B, T, H, E), generator=gen).to(dtype) for _ in range(2))
    u = torch.rand((B, T, H), generator=gen)
    g = {"any": -torch.exp(-6 * u), "none": 0 * u, "strong": -40 * u, "grow": 0.02 * u,
         "resets": torch.where(u < 0.1, -math.inf, torch.where(u < 0.2, -1e30, -0.1 * u))}[gates].to(gdt)
    state, dstate = (torch.randn((B, H, D, E), generator=gen) for _ in range(2))
    return q, k, v, g, state, dout, dstate


def check(q, k, v, g, state, lengths, scale, dout, dstate):
    F = _F()
    leaves = [t.cuda().requires_grad_(True) for t in (q, k, v, g)]
    s0 = None if state is None else state.cuda().requires_grad_(True)
    lens = None if lengths is None else lengths.cuda()
    r = F.linear_attention(*leaves, state=s0, lengths=lens, scale=scale)
    assert r.out.dtype == q.dtype and r.state.dtype == torch.float32 and r.out.shape == v.shape
    leaves += [] if s0 is None else [s0]
    ends, gs = ([r.out], [dout.cuda()]) if dstate is None else ([r.out, r.state], [dout.cuda(), dstate.cuda()])
    got = torch.autograd.grad(ends, leaves, gs)
    want, bound = reference(q, k, v, g, state, lengths, scale, dout, dstate)
    for name, t in zip(("out", "state", "dq", "dk", "dv", "dg", "dstate"), (r.out, r.state) + got):
        R.close(t, want[name], bound[name], name)
    # without a gradient of the decays: the same but for roundings; without any: the same bits
    leaves[3] = g.cuda()
    r2 = F.linear_attention(*leaves[:4], state=s0, lengths=lens, scale=scale)
    names = ["dq", "dk", "dv"] + ([] if s0 is None else ["dstate"])
    got = torch.autograd.grad([r2.out, r2.state][:len(ends)], leaves[:3] + leaves[4:], gs)
    for name, t in zip(names, got):
        R.close(t, want[name], bound[name], name)
    plain = F.linear_attention(*[t.detach() for t in leaves[:4]], state=None if s0 is None else s0.detach(),
                               lengths=lens, scale=scale)
    assert not plain.out.requires_grad
    assert torch.equal(plain.out, r.out.detach()) and torch.equal(plain.state, r.state.detach())


SIZES = [(1, 1, 1, 1, 1), (2, 5, 3, 8, 16), (1, 64, 2, 64, 64), (2, 65, 1, 64, 64), (3, 130, 2, 16, 48), (1, 257, 2, 128, 128),
         (2, 100, 2, 128, 64), (1, 100, 3, 40, 100), (1, 1030, 1, 64, 64), (2, 777, 2, 33, 65), (1, 31, 1, 65, 7)]


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("carry", [False, True])
@pytest.mark.parametrize("B,T,H,D,E", SIZES)
def test_values_and_gradients(B, T, H, D, E, carry, dt):
    q, k, v, g, state, dout, dstate = make(B, T, H, D, E, DT[dt], seed=T)
    if not carry:
        state = dstate = None
    check(q, k, v, g, state, None, D ** -0.5, dout, dstate)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("gates", ["none", "strong", "grow", "resets"])
@pytest.mark.parametrize("T", [40, 150, 600])
def test_decays(T, gates, dt):
    q, k, v, g, state, dout, dstate = make(2, T, 2, 64, 64, DT[dt], seed=T, gates=gates)
    check(q, k, v, g, state, None, 1.0, dout, dstate)
    if gates != "grow":
        check(q, k, v, g.bfloat16(), None, None, -0.5, dout, None)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("T", [1, 70, 600])
def test_padded(T, dt):
    """Tokens from a sequence's length on are not read, whatever they hold."""
    lengths = torch.tensor([T, 0, 1, -3, T + 9, (2 * T) // 3, min(T, 64)])
    q, k, v, g, state, dout, dstate = make(7, T, 2, 24, 40, DT[dt], seed=T)
    for i, n in enumerate(lengths.tolist()):
        for t in (q, k, v, g, dout):
            t[i, max(n, 0):] = float("nan")
    check(q, k, v, g, state, lengths, 0.25, dout, dstate)
    check(q, k, v, g, None, lengths, 0.25, dout, None)


def test_padded_int32_lengths():
    F = _F()
    q, k, v, g, state, _, _ = (t.cuda() for t in make(3, 80, 2, 16, 16, torch.float32))
    n = torch.tensor([80, 3, 41])
    a = F.linear_attention(q, k, v, g, lengths=n.cuda())
    b = F.linear_attention(q, k, v, g, lengths=n.to(torch.int32).cuda())
    assert torch.equal(a.out, b.out) and torch.equal(a.state, b.state)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_layouts(dt):
    """Slices of one projection's output, transposed and expanded arrays, decays of a head, cotangents of any layout."""
    F = _F()
    B, T, H, D = 2, 90, 3, 32
    gen = torch.Generator().manual_seed(5)
    wide = torch.randn((B, T, H * D * 3 + 5), generator=gen).to(DT[dt])
    q, k, v = (wide[..., 1 + i * H * D:1 + (i + 1) * H * D].unflatten(-1, (H, D)) for i in range(3))
    heads_first = torch.randn((B, H, T, D), generator=gen).to(DT[dt]).movedim(1, 2)
    slow = -torch.rand(H, generator=gen)
    dev = wide.cuda()
    dq, dk_, dv_ = (dev[..., 1 + i * H * D:1 + (i + 1) * H * D].unflatten(-1, (H, D)) for i in range(3))
    for kk, dkk in ((k, dk_), (heads_first, heads_first.movedim(2, 1).cuda().movedim(1, 2)),
                    (k[:, :1].expand(B, T, H, D), dk_[:, :1].expand(B, T, H, D))):
        leaf = slow.cuda().requires_grad_(True)
        args = [dq.detach().requires_grad_(True), dkk.detach().requires_grad_(True), dv_.detach().requires_grad_(True)]
        r = F.linear_attention(*args, leaf.expand(B, T, H))
        for dout in (torch.randn((B, T, H, D), generator=gen).to(DT[dt]), torch.ones((), dtype=DT[dt]).expand(B, T, H, D),
                     torch.randn((B, H, T, D), generator=gen).to(DT[dt]).movedim(1, 2)):
            got = torch.autograd.grad(r.out, args + [leaf], dout.cuda(), retain_graph=True)
            want, bound = reference(q, kk, v, slow.expand(B, T, H), None, None, 1.0, dout, None)
            R.close(r.out, want["out"], bound["out"], "out")
            for name, t in zip(("dq", "dk", "dv"), got):
                R.close(t, want[name], bound[name], name)
            R.close(got[3], want["dg"].sum((0, 1)), bound["dg"].sum((0, 1)) + B * T * U * want["dg"].abs().sum((0, 1)), "dg")


def test_one_output_alone():
    """A cotangent of the state without one of the outputs, and the other way round."""
    F = _F()
    q, k, v, g, state, dout, dstate = make(2, 300, 2, 32, 48, torch.float32)
    leaves = [t.cuda().requires_grad_(True) for t in (q, k, v, g, state)]
    r = F.linear_attention(*leaves[:4], state=leaves[4])
    got = torch.autograd.grad(r.state, leaves, dstate.cuda())
    want, bound = reference(q, k, v, g, state, None, 1.0, torch.zeros_like(dout), dstate)
    for name, t in zip(("dq", "dk", "dv", "dg", "dstate"), got):
        R.close(t, want[name], bound[name], name)


def test_pieces_of_a_sequence():
    """A sequence in pieces, the state handed on, is the whole one's recurrence: also token by token."""
    F = _F()
    for dt in ("bf16", "f32"):
        q, k, v, g, state, dout, _ = make(2, 200, 3, 64, 64, DT[dt], seed=9)
        want, bound = reference(q, k, v, g, state, None, 0.125, dout, None)
        dev = [t.cuda() for t in (q, k, v, g)]
        s, outs = state.cuda(), []
        for lo, hi in ((0, 1), (1, 67), (67, 67), (67, 200)):
            r = F.linear_attention(*[t[:, lo:hi] for t in dev], state=s, scale=0.125)
            s = r.state
            outs.append(r.out)
        R.close(torch.cat(outs, 1), want["out"], bound["out"], "out")
        R.close(s, want["state"], bound["state"], "state")
        s, outs = state.cuda(), []
        for t in range(200):
            outs.append(F.linear_attention_step(*[x[:, t] for x in dev], s, scale=0.125))
        R.close(torch.stack(outs, 1), want["out"], bound["out"], "out of steps")
        R.close(s, want["state"], bound["state"], "state of steps")


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("B,H,D,E", [(1, 1, 1, 1), (3, 2, 64, 64), (2, 5, 128, 128), (1, 3, 17, 33), (2, 2, 128, 5), (4, 1, 3, 100)])
def test_step(B, H, D, E, dt):
    F = _F()
    for gates in ("any", "resets", "grow"):
        q, k, v, g, state, dout, _ = make(B, 1, H, D, E, DT[dt], seed=E, gates=gates)
        want, bound = reference(q, k, v, g, state, None, 0.3, dout, None)
        s = state.cuda()
        y = F.linear_attention_step(*[t[:, 0].cuda() for t in (q, k, v, g)], s, scale=0.3)
        R.close(y, want["out"][:, 0], bound["out"][:, 0], "out")
        R.close(s, want["state"], bound["state"], "state")
        s2 = state.cuda()
        strided = [torch.cat([t[:, 0], t[:, 0]], -1).cuda()[..., :t.shape[-1]] for t in (q, k, v)]
        y2 = F.linear_attention_step(*strided, g[:, 0].to(torch.float32).cuda(), s2, scale=0.3)
        assert torch.equal(y, y2) and torch.equal(s, s2)


def test_empty():
    F = _F()
    for B, T in ((0, 5), (2, 0)):
        q, k, v, g, state, dout, dstate = (t.cuda() for t in make(B, T, 2, 16, 24, torch.bfloat16))
        leaves = [t.requires_grad_(True) for t in (q, k, v, g, state)]
        r = F.linear_attention(*leaves[:4], state=leaves[4])
        assert r.out.shape == (B, T, 2, 24) and torch.equal(r.state, state)
        got = torch.autograd.grad((r.out, r.state), leaves, (dout, dstate))
        assert torch.equal(got[4], dstate) and all(a.shape == b.shape for a, b in zip(got, leaves))
    z = F.linear_attention(q, k, v, g)
    assert not bool(z.state.any())


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("T", [90, 700])
def test_same_bits_streams_and_graphs(T, dt):
    F = _F()
    data = make(2, T, 2, 64, 64, DT[dt], seed=3)
    q, k, v, g, state = (t.cuda().requires_grad_(True) for t in data[:5])
    dout, dstate = data[5].cuda(), data[6].cuda()

    def work():
        r = F.linear_attention(q, k, v, g, state=state, scale=0.125)
        return (r.out.detach(), r.state.detach()) + torch.autograd.grad((r.out, r.state), (q, k, v, g, state), (dout, dstate))
    want = [t.clone() for t in work()]
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(work(), want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = work()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = work()
    for rep in range(3):
        new = make(2, T, 2, 64, 64, DT[dt], seed=10 + rep)
        with torch.no_grad():
            for a, b in zip((q, k, v, g, state, dout, dstate), new):
                a.copy_(b)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, work())), rep


def test_step_in_a_graph():
    F = _F()
    q, k, v, g, state, _, _ = (t.cuda() for t in make(3, 1, 2, 64, 64, torch.bfloat16))
    one = [t[:, 0].contiguous() for t in (q, k, v, g)]
    s, eager = state.clone(), state.clone()
    graph = torch.cuda.CUDAGraph()
    F.linear_attention_step(*one, state.clone())
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        y = F.linear_attention_step(*one, s)
    s.copy_(state)
    for rep in range(4):
        for t in one[:3]:
            t.copy_(torch.randn_like(t))
        torch.cuda.synchronize()
        graph.replay()
        want = F.linear_attention_step(*one, eager)
        assert torch.equal(y, want) and torch.equal(s, eager), rep


def test_changed_arrays():
    F = _F()
    q, k, v, g, state, _, dstate = (t.cuda() for t in make(2, 70, 2, 16, 16, torch.float32))
    for i in range(4):
        args = [t.clone().requires_grad_(True) for t in (q, k, v, g)]
        used = [a * 1 for a in args]
        r = F.linear_attention(*used)
        with torch.no_grad():
            used[i] += 1
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            r.out.sum().backward()
    # the state that came back, updated by steps: refused where the backward pass reads it
    args = [t.clone().requires_grad_(True) for t in (q, k, v, g)]
    r = F.linear_attention(*args)
    with torch.no_grad():
        F.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], g[:, 0], r.state.detach())
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        r.state.backward(dstate)
    r = F.linear_attention(*args)
    r.out.sum().backward()
    with pytest.raises(RuntimeError, match="second time"):
        r.out.sum().backward()


def test_differences():
    """Gradients against differences of the results in 32 bits along random directions."""
    F = _F()
    q, k, v, g, state, dout, dstate = make(1, 90, 2, 32, 32, torch.float32, seed=4)
    leaves = [t.cuda().requires_grad_(True) for t in (q, k, v, g, state)]
    r = F.linear_attention(*leaves[:4], state=leaves[4], scale=0.2)
    grads = torch.autograd.grad((r.out, r.state), leaves, (dout.cuda(), dstate.cuda()))

    def value(args):
        with torch.no_grad():
            r = F.linear_attention(*args[:4], state=args[4], scale=0.2)
        return float((r.out.double() * dout.cuda()).sum() + (r.state.double() * dstate.cuda()).sum())
    base = [t.detach() for t in leaves]
    for i, gr in enumerate(grads):
        way = torch.randn(base[i].shape, generator=torch.Generator().manual_seed(i)).cuda()
        h = 2.0 ** -7
        up, down = list(base), list(base)
        up[i], down[i] = base[i] + h * way, base[i] - h * way
        slope, want = (value(up) - value(down)) / (2 * h), float((gr.double() * way).sum())
        # the results' f32 noise over 2 h, and the third derivative's h^2 (decays: powers of e^(h way))
        scale = float((gr.double().abs() * way.abs()).sum())
        assert abs(slope - want) <= scale * (2.0 ** -20 / h + (h * h * 40 if i == 3 else 2.0 ** -12)), (i, slope, want)


def test_refusals():
    F = _F()
    q = torch.zeros((2, 5, 3, 8), device="cuda")
    v, g, s = torch.zeros((2, 5, 3, 4), device="cuda"), torch.zeros((2, 5, 3), device="cuda"), torch.zeros((2, 3, 8, 4), device="cuda")
    from pratchya_amd import _lib
    call = F.linear_attention
    for bad, error in ((lambda: call(q.half(), q.half(), v.half(), g), TypeError), (lambda: call(q, q.bfloat16(), v, g), TypeError),
                       (lambda: call(q, q[:, :4], v, g), ValueError), (lambda: call(q, q, v[:, :, :2], g), ValueError),
                       (lambda: call(q, q, v, g[..., 0]), ValueError), (lambda: call(q, q, v, g.double()), TypeError),
                       (lambda: call(q[0], q[0], v[0], g[0]), ValueError), (lambda: call(q, q, v, g, state=s[:1]), ValueError),
                       (lambda: call(q, q, v, g, state=s.bfloat16()), TypeError),
                       (lambda: call(q, q, v, g, lengths=torch.ones(3, device="cuda").long()), ValueError),
                       (lambda: call(q, q, v, g, lengths=torch.ones(2, device="cuda")), TypeError),
                       (lambda: call(q, q, v, g, lengths=torch.ones(2).long()), RuntimeError),
                       (lambda: call(q.cpu(), q, v, g), RuntimeError), (lambda: call(q, q, v, [1]), TypeError),
                       (lambda: call(*[torch.zeros((1, 2, 1, 129), device="cuda")] * 3, torch.zeros((1, 2, 1), device="cuda")),
                        _lib.PratchyaUnsupported)):
        with pytest.raises(error):
            bad()
    one = (q[:, 0], q[:, 0], v[:, 0], g[:, 0])
    for bad, error in ((lambda: F.linear_attention_step(*one, s.bfloat16()), TypeError),
                       (lambda: F.linear_attention_step(*one, s[:, :2]), ValueError),
                       (lambda: F.linear_attention_step(*one, s.transpose(2, 3).contiguous().transpose(2, 3)), ValueError),
                       (lambda: F.linear_attention_step(*one, s.cpu()), RuntimeError),
                       (lambda: F.linear_attention_step(q, q, v, g, s), ValueError),
                       (lambda: F.linear_attention_step(q[:, 0].requires_grad_(True), *one[1:], s), ValueError),
                       (lambda: F.linear_attention_step(*one, None), TypeError)):
        with pytest.raises(error):
            bad()
    x = q.clone().requires_grad_(True)
    d, = torch.autograd.grad(call(x, q, v, g).out.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="again"):
        d.sum().backward()
    import torch.autograd.forward_ad as fwd
    with fwd.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
        call(fwd.make_dual(q, torch.ones_like(q)), q, v, g)
