"""The operators of a memory layer together, as a model runs them: layer norm,
several-axes rotary on q and k, their l2 norm (uttt_amd.moe.rows_preprocess),
the gated delta rule over packed prompts, and generation from its states."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
HEADS, WIDTH, SECTIONS = 2, 64, [8, 12, 12]
HID = HEADS * WIDTH


def build(T, seed=0):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    p = dict(x=r(1, T, HID), w=1 + 0.1 * r(HID), b=0.1 * r(HID), wqkv=r(3 * HID, HID) / HID ** 0.5,
             wgb=r(2 * HEADS, HID) / HID ** 0.5)
    pos = torch.stack([torch.arange(T) // 64, torch.arange(T) // 8 % 8, torch.arange(T) % 8], -1)
    return p, pos[None].to(torch.int32)


def project(p, x, pos, dtype, norm, rotary, unit):
    """q, k, v, g, beta of tokens x [B, T, HID]."""
    B, T = x.shape[:2]
    h = norm(x, p["w"], p["b"])
    qkv = (h @ p["wqkv"].to(dtype).t()).view(B, T, 3, HEADS, WIDTH)
    gb = h @ p["wgb"].to(dtype).t()
    q, k = (unit(rotary(qkv[:, :, i], pos)) for i in (0, 1))
    return q, k, qkv[:, :, 2], -torch.nn.functional.softplus(gb[..., :HEADS]), torch.sigmoid(gb[..., HEADS:])


def ours(p, x, pos):
    from uttt_amd.moe import rows_preprocess
    from uttt_amd.norm import layer_norm
    from uttt_amd.positions import axis_frequencies, rotary_axes
    freq = axis_frequencies(SECTIONS, device="cuda")
    unit = lambda t: rows_preprocess(t.reshape(*t.shape[:2], HID), norm="l2", rows_of=WIDTH).view(t.shape)  # noqa: E731
    return project(p, x, pos, BF16, layer_norm, lambda t, s: rotary_axes(t, s, freq, SECTIONS), unit)


def exact(p, x, pos, cu):
    """The same layer in 64 bits on the CPU."""
    from oracle.delta import gated_delta_rule
    from uttt_amd.positions import axis_frequencies
    freq = axis_frequencies(SECTIONS).double()
    axis = [a for a, m in enumerate(SECTIONS) for _ in range(m)]

    def norm(x, w, b):
        return torch.nn.functional.layer_norm(x, (HID,), w, b)

    def rotary(t, pos):
        ang = (pos.double()[..., axis] * freq)[:, :, None]
        a, b = t[..., :32], t[..., 32:]
        return torch.cat([a * ang.cos() - b * ang.sin(), a * ang.sin() + b * ang.cos()], -1)

    unit = lambda t: t / (t.norm(dim=-1, keepdim=True) + 1e-5)  # noqa: E731
    q, k, v, g, beta = project(p, x, pos, torch.float64, norm, rotary, unit)
    return gated_delta_rule(q, k, v, g, beta, WIDTH ** -0.5, None, cu)


def test_prompts_gradients_and_generation():
    """Tolerance: every step of the layer rounds to bf16 once (norm, projection,
    rotary, l2 norm, gates, rule: six half steps of 2^-8 in a row on the way to o,
    as many again on the way back), in the 2-norm."""
    from uttt_amd.delta import gated_delta_rule, gated_delta_step
    H = 2.0 ** -8
    T, cu = 150, [0, 67, 150]
    p, pos = build(T + 8)
    leaf = {n: t.to(BF16 if n in ("x", "wqkv", "wgb") else torch.float32).cuda().requires_grad_() for n, t in p.items()}
    ref = {n: t.detach().double().cpu().requires_grad_() for n, t in leaf.items()}
    q, k, v, g, beta = ours(leaf, leaf["x"][:, :T], pos[:, :T].cuda())
    o, S = gated_delta_rule(q, k, v, g, beta, output_final_state=True, cu_seqlens=torch.tensor(cu, device="cuda"))
    ro, rS = exact(ref, ref["x"][:, :T], pos[:, :T], cu)
    close = lambda a, b, n: (a.double().cpu() - b).norm() <= n * H * b.norm()  # noqa: E731
    assert close(o, ro, 6) and close(S, rS, 6)
    w = torch.randn(o.shape, generator=torch.Generator().manual_seed(1)).to(BF16)
    names = list(leaf)
    got = torch.autograd.grad(o, [leaf[n] for n in names], w.cuda(), retain_graph=True)
    want = torch.autograd.grad(ro, [ref[n] for n in names], w.double(), retain_graph=True)
    for n, a, b in zip(names, got, want):
        assert close(a, b, 12), n
    # generation: both sequences carry on from their states, token by token, with a padded row
    with torch.no_grad():
        state = torch.zeros(5, HEADS, WIDTH, WIDTH, device="cuda")
        slots = torch.tensor([3, 1, -1], device="cuda")
        state[slots[:2]] = S
        outs = []
        for t in range(T, T + 8):
            x = leaf["x"][:, t:t + 1].expand(3, -1, -1)
            outs.append(gated_delta_step(*ours(leaf, x, pos[:, t:t + 1].cuda().expand(3, -1, -1)), state,
                                         state_indices=slots))
        outs = torch.cat(outs, 1)
        assert (outs[2] == 0).all() and (state[[0, 2, 4]] == 0).all()
        for i in range(2):
            keep = list(range(cu[i], cu[i + 1])) + list(range(T, T + 8))
            ro, rS = exact(ref, ref["x"][:, keep], pos[:, keep], None)
            assert close(outs[i], ro[0, -8:], 6) and close(state[slots[i]], rS[0], 6)


def test_a_training_step_gives_the_same_bits_twice():
    """Two identical steps give identical gradients."""
    from uttt_amd.delta import gated_delta_rule
    p, pos = build(130)

    def step():
        leaf = {n: t.to(BF16 if n in ("x", "wqkv", "wgb") else torch.float32).cuda().requires_grad_() for n, t in p.items()}
        o, S = gated_delta_rule(*ours(leaf, leaf["x"], pos.cuda()), output_final_state=True)
        (o.float().square().sum() + S.square().sum()).backward()
        return [t.grad for t in leaf.values()]

    for a, b in zip(step(), step()):
        assert torch.equal(a, b)
