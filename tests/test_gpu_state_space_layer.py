"""The state space layer's operators together, as a model runs them: the norm of
the residual stream, projections, the short convolution, the scan with its gate,
the gated norm by heads into the residual, over packed prompts with gradients;
then generation from its states; and the convolution and the gated norm around
the gated delta rule."""
import pytest
import torch

from oracle import state_space as O

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
HID, D, N, W, HEAD = 48, 96, 16, 4, 32
H = 2.0 ** -8


def weights(T, seed=0):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    p = dict(x=r(1, T, HID), res=r(1, T, HID), w1=1 + 0.1 * r(HID), s1=0.5 + 0.1 * r(HID), win=r(2 * D, HID) / HID ** 0.5,
             cw=r(D, W) / 2, cb=0.1 * r(D), wbc=r(2 * N, D) / D ** 0.5, wdt=0.3 * r(D, D) / D ** 0.5,
             dtb=torch.log(torch.expm1(torch.exp(-5 + 3 * torch.rand(D, generator=gen)))),
             A=-torch.arange(1.0, N + 1) * torch.exp(0.2 * r(D, N)), Dp=1 + 0.1 * r(D), wout=r(HID, D) / D ** 0.5,
             w2=1 + 0.1 * r(HEAD), s2=0.5 + 0.1 * r(HEAD))
    low = ("x", "win", "wbc", "wdt", "wout")
    return {n: t.to(BF16 if n in low else F32) for n, t in p.items()}


class Ours:
    def __init__(self, cu=None, states=None, slots=None):
        self.cu, self.states, self.slots = cu, states, slots

    def before(self, x, r, w, s):
        from uttt_amd.norm import norm_before_block
        return norm_before_block(x, r, w, scale=s)

    def conv(self, x, w, b):
        from uttt_amd.state_space import causal_conv, causal_conv_step
        if self.slots is not None:
            return causal_conv_step(x, w, self.states[0], b, activation="silu", state_indices=self.slots), self.states[0]
        return causal_conv(x, w, b, activation="silu", output_final_state=True, cu_seqlens=self.cu)

    def scan(self, x, dt, A, B, C, Dp, z, dtb):
        from uttt_amd.state_space import selective_scan, selective_scan_step
        kw = dict(D=Dp, gate=z, dt_bias=dtb, dt_softplus=True)
        if self.slots is not None:
            return selective_scan_step(x, dt, A, B, C, self.states[1], state_indices=self.slots, **kw), self.states[1]
        return selective_scan(x, dt, A, B, C, output_final_state=True, cu_seqlens=self.cu, **kw)

    def after(self, x, w, z, r, s):
        from uttt_amd.norm import norm_after_block
        return norm_after_block(x, w, gate=z, residual=r, scale=s)


class Exact:
    """The same in 64 bits on the CPU, differentiable."""

    def __init__(self, cu=None):
        self.cu = cu

    def before(self, x, r, w, s):
        return O.norm_before_block(x, r, w, s)

    def conv(self, x, w, b):
        return O.causal_conv(x, w, b, True, None, self.cu)

    def scan(self, x, dt, A, B, C, Dp, z, dtb):
        ys, states = [], []
        for b, s, e in O.spans(1, x.shape[1], self.cu):
            h, step = torch.zeros_like(A), torch.nn.functional.softplus(dt + dtb, threshold=100.0)
            for t in range(s, e):
                h = h * torch.exp(step[0, t, :, None] * A) + (step[0, t] * x[0, t])[:, None] * B[0, t]
                ys.append(((h * C[0, t]).sum(-1) + Dp * x[0, t]) * torch.nn.functional.silu(z[0, t]))
            states.append(h)
        return torch.stack(ys)[None], torch.stack(states)

    def after(self, x, w, z, r, s):
        return O.norm_after_block(x, w, z, r, s)


def layer(ops, p, x, res):
    """Tokens x and the residual stream [B, T, HID] through one block: the stream after
    it, the block's normed heads, and the states."""
    B, T = x.shape[:2]
    h, stream = ops.before(x, res, p["w1"], p["s1"])
    xz = (h @ p["win"].t()).view(B, T, 2, D)
    u, cs = ops.conv(xz[:, :, 0], p["cw"], p["cb"])
    bc = (u @ p["wbc"].t()).view(B, T, 2, 1, N)
    y, hs = ops.scan(u, u @ p["wdt"].t(), p["A"], bc[:, :, 0], bc[:, :, 1], p["Dp"], xz[:, :, 1], p["dtb"])
    heads = y.view(B, T, D // HEAD, HEAD)
    o = ops.after(heads, p["w2"], xz[:, :, 1].view(heads.shape), heads, p["s2"])
    return o.reshape(B, T, D) @ p["wout"].t(), stream, cs, hs


def close(a, b, n):
    return (a.detach().double().cpu() - b.detach()).norm() <= n * H * b.detach().norm()


def test_prompts_gradients_and_generation():
    """Tolerance: on the way to the block's output each of eight steps rounds to bf16
    once (norm, three projections, convolution, scan, gated norm, projection), as
    many again on the way back; a step's rounding is carried on by the steps behind
    it with their slopes, about 1 each, and a sum of two of them. In the 2-norm."""
    T, cu = 130, [0, 57, 57, 130]
    p = weights(T + 6)
    leaf = {n: t.cuda().requires_grad_() for n, t in p.items()}
    ref = {n: t.double().requires_grad_() for n, t in p.items()}
    out, stream, cs, hs = layer(Ours(torch.tensor(cu, device="cuda")), leaf, leaf["x"][:, :T], leaf["res"][:, :T])
    want, wstream, wcs, whs = layer(Exact(cu), ref, ref["x"][:, :T], ref["res"][:, :T])
    assert close(out, want, 16) and close(stream, wstream, 1e-3) and close(cs, wcs, 4) and close(hs, whs, 8)
    gen = torch.Generator().manual_seed(3)
    g1, g2 = torch.randn(want.shape, generator=gen).to(BF16), torch.randn(wstream.shape, generator=gen)
    names = list(leaf)
    got = torch.autograd.grad([out, stream], [leaf[n] for n in names], [g1.cuda(), g2.cuda()])
    exact = torch.autograd.grad([want, wstream], [ref[n] for n in names], [g1.double(), g2.double()])
    for n, a, b in zip(names, got, exact):
        assert close(a, b, 32), n
    # generation: the first and last sequences carry on, token by token, with a padded row
    with torch.no_grad():
        states = [torch.zeros(5, W - 1, D, device="cuda", dtype=BF16), torch.zeros(5, D, N, device="cuda")]
        slots = torch.tensor([3, 1, -1], device="cuda")
        for s, v in zip(states, (cs, hs)):
            s[slots[:2]] = v[[0, 2]]
        ops, outs = Ours(states=states, slots=slots), []
        for t in range(T, T + 6):
            cut = lambda v: v[:, t:t + 1].expand(3, -1, -1)  # noqa: E731
            outs.append(layer(ops, leaf, cut(leaf["x"]), cut(leaf["res"]))[0])
        outs = torch.cat(outs, 1)
        assert (states[0][[0, 2, 4]] == 0).all() and (states[1][[0, 2, 4]] == 0).all()
        for i, (s, e) in enumerate(((0, 57), (57, 130))):
            keep = list(range(s, e)) + list(range(T, T + 6))
            want, _, wcs, whs = layer(Exact(), ref, ref["x"][:, keep], ref["res"][:, keep])
            assert close(outs[i], want[0, -6:], 16)
            assert close(states[0][slots[i]], wcs[0], 4) and close(states[1][slots[i]], whs[0], 8)


def test_a_training_step_gives_the_same_bits_twice():
    p = weights(100)

    def step():
        leaf = {n: t.cuda().requires_grad_() for n, t in p.items()}
        out, stream, *_ = layer(Ours(torch.tensor([0, 30, 100], device="cuda")), leaf, leaf["x"], leaf["res"])
        (out.float().square().sum() + stream.square().sum()).backward()
        return [t.grad for t in leaf.values()]

    for a, b in zip(step(), step()):
        assert torch.equal(a, b)


def test_around_the_gated_delta_rule():
    """q, k and v through the short convolution, the rule's outputs normed by heads with
    their gate: against the same calls' 64-bit definitions, each from the other's
    inputs (a rounding of its own each, the rule's as its tests have them)."""
    from oracle.delta import gated_delta_rule as exact_rule
    from uttt_amd.delta import gated_delta_rule
    from uttt_amd.norm import norm_after_block
    from uttt_amd.state_space import causal_conv
    gen = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    T, heads, width = 90, 2, 64
    qkv, z = r(1, T, 3 * heads * width).to(BF16), r(1, T, heads, width).to(BF16)
    w, nw = r(3 * heads * width, 4) / 2, 1 + 0.1 * r(width)
    g, beta = -0.1 * r(1, T, heads).abs(), torch.sigmoid(r(1, T, heads))
    y, _ = causal_conv(qkv.cuda(), w.cuda(), activation="silu")
    want, _ = O.causal_conv(qkv.double(), w.double(), None, True)
    assert close(y, want, 1)
    q, k, v = y.view(1, T, 3, heads, width).unbind(2)
    unit = lambda t: (t.float() / t.float().norm(dim=-1, keepdim=True)).to(BF16)  # noqa: E731
    q, k = unit(q), unit(k)
    o, _ = gated_delta_rule(q, k, v, g.cuda(), beta.cuda())
    d = lambda t: t.double().cpu()  # noqa: E731
    want, _ = exact_rule(d(q), d(k), d(v), g.double(), beta.double(), width ** -0.5, None, None)
    assert close(o, want, 2)
    assert close(norm_after_block(o, nw.cuda(), gate=z.cuda()), O.norm_after_block(d(o), nw.double(), z.double()), 1)
