"""The selective scan on the GPU against the 64-bit formulas (tolerances:
tests/state_space_cases.py)."""
import pytest
import torch

from state_space_cases import BF16, F16, F32, call, check, check_scan, scan_exact, scan_inputs, up

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T", [1, 2, 3, 4, 5, 15, 16, 17, 31, 33, 63, 64, 65, 127, 129, 300])
def test_lengths(T):
    check_scan(*scan_inputs(B=2, T=T, D=20, N=16, dtype=BF16, seed=T))


@pytest.mark.parametrize("N", [1, 2, 3, 4, 5, 7, 8, 9, 15, 16, 17, 24, 31, 32, 33, 48, 63, 64])
@pytest.mark.parametrize("gate", [False, True])
def test_states(N, gate):
    check_scan(*scan_inputs(B=1, T=90, D=37, N=N, gate=gate, seed=N))


@pytest.mark.parametrize("D,G", [(1, 1), (2, 2), (3, 1), (12, 4), (63, 1), (64, 2), (65, 1), (129, 3), (256, 1), (257, 1),
                                 (390, 2), (515, 5)])
@pytest.mark.parametrize("N", [4, 16, 40])
def test_channels_and_groups(D, G, N):
    check_scan(*scan_inputs(B=1, T=40, D=D, N=N, G=G, dtype=F16, seed=D))


@pytest.mark.parametrize("dtype,dt_dtype", [(F32, F32), (BF16, F32), (BF16, BF16), (F16, F32), (F16, F16)])
@pytest.mark.parametrize("soft,bias", [(False, False), (False, True), (True, False), (True, True)])
@pytest.mark.parametrize("rest", [False, True])
def test_types_and_options(dtype, dt_dtype, soft, bias, rest):
    check_scan(*scan_inputs(B=2, T=50, D=18, N=6, dtype=dtype, dt_dtype=dt_dtype, soft=soft, bias=bias, gate=rest,
                            skip=rest, state=rest))


@pytest.mark.parametrize("lens,front,behind", [
    ([1], 0, 0), ([0], 3, 2), ([0, 0, 5, 0], 0, 0), ([17, 64, 0, 1, 130, 16, 15], 0, 0), ([70, 3, 0], 5, 40),
    ([1] * 40, 0, 1), ([200, 1, 65], 64, 64), ([0, 0], 0, 0), ([0], 0, 0)])
@pytest.mark.parametrize("N", [8, 24])
def test_packed(lens, front, behind, N):
    """Empty sequences keep their state and hand its gradient back; tokens of no
    sequence get zeros."""
    cu = [front + sum(lens[:i]) for i in range(len(lens) + 1)]
    a = scan_inputs(T=cu[-1] + behind, D=70, N=N, G=2, dtype=BF16, seqs=len(lens), seed=N)
    got = check_scan(*a, cu=cu)
    loose = [t for t in range(cu[-1] + behind) if t < front or t >= cu[-1]]
    for n in ("x", "dt", "gate", "B", "C"):
        assert (got[n][:, loose] == 0).all(), n


def test_long_sequences_in_runs():
    """Long enough for many runs of a sequence, forward and backward."""
    check_scan(*scan_inputs(B=1, T=1500, D=9, N=5, seed=1))
    cu = [0, 900, 901, 1400]
    check_scan(*scan_inputs(T=1400, D=6, N=17, dtype=BF16, seqs=3, seed=2), cu=cu)


def test_many_sequences_as_single_runs():
    check_scan(*scan_inputs(B=300, T=20, D=130, N=4, dtype=BF16, seed=1))


def test_int64_offsets():
    from uttt_amd.state_space import selective_scan
    a, soft, _ = scan_inputs(T=30, D=8, N=4, seqs=2)
    cu = torch.tensor([0, 11, 30], device="cuda")
    y, h = selective_scan(*(a[n] for n in ("x", "dt", "A", "B", "C")), dt_softplus=soft, dt_bias=a["dt_bias"],
                          initial_state=a["initial_state"], output_final_state=True, cu_seqlens=cu)
    y2, h2 = selective_scan(*(a[n] for n in ("x", "dt", "A", "B", "C")), dt_softplus=soft, dt_bias=a["dt_bias"],
                            initial_state=a["initial_state"], output_final_state=True, cu_seqlens=cu.int())
    assert torch.equal(y, y2) and torch.equal(h, h2)


def test_no_tokens():
    """Unpacked sequences of no tokens: the state goes through, its gradient too."""
    a, soft, (dy, dhT) = scan_inputs(B=3, T=0, D=10, N=6)
    a["initial_state"].requires_grad_()
    a["A"].requires_grad_()
    y, h = call(a, soft)
    assert y.shape == (3, 0, 10) and torch.equal(h, a["initial_state"])
    dh0, dA = torch.autograd.grad([y, h], [a["initial_state"], a["A"]], [dy, dhT])
    assert torch.equal(dh0, dhT) and (dA == 0).all()


def test_views():
    """Slices, other strides and addresses of every input, with the bits of their copies."""
    a, soft, grads = scan_inputs(B=2, T=45, D=33, N=8, G=3, dtype=BF16)
    want = {n: g for n, g in check_scan(a, soft, grads).items()}

    def wide(t, front):
        big = t.new_zeros(*t.shape[:-1], t.shape[-1] + 5)
        big[..., front:front + t.shape[-1]] = t
        return big[..., front:front + t.shape[-1]]

    def crossed(t):   # batch and tokens, or rows and columns, the other way round in memory
        return t.transpose(0, 1).contiguous().transpose(0, 1)

    def last(t):      # no contiguous last axis: taken as a copy
        return t.transpose(-1, -2).contiguous().transpose(-1, -2)

    for change in (lambda t: wide(t, 1), lambda t: wide(t, 3), crossed, last):
        b = {n: t if t is None or t.dim() < 2 else change(t) for n, t in a.items()}
        b["D"], b["dt_bias"] = wide(a["D"], 2), wide(a["dt_bias"], 1)
        got = check_scan(b, soft, (change(grads[0]), change(grads[1])))
        for n in want:
            assert torch.equal(got[n], want[n]), n


def test_expanded_inputs():
    """Steps of a head for all its channels and rates of a head for all its states
    are views without memory of their own; their gradients are sums."""
    a, soft, grads = scan_inputs(B=2, T=30, D=24, N=8, bias=False, seed=3)
    heads = a["dt"][:, :, ::6].contiguous().requires_grad_()
    rates = a["A"][::6, :1].contiguous().requires_grad_()
    e = dict(a, dt=heads[..., None].expand(-1, -1, -1, 6).flatten(2),
             A=rates[:, None].expand(-1, 6, 8).reshape(24, 8))
    y, h = call(e, soft)
    got = torch.autograd.grad([y, h], [heads, rates], list(grads))
    val, err = scan_exact(e, soft, grads)
    check(y, val["y"], err["y"], "y")
    # torch's own sums of 6 and 48 gradients: as many roundings of their sizes
    for g, v, b in ((got[0], val["d_dt"].unflatten(2, (4, 6)), err["d_dt"].unflatten(2, (4, 6))),
                    (got[1], val["d_A"].view(4, 48), err["d_A"].view(4, 48))):
        check(g.view(v.shape[:-1]), v.sum(-1), b.sum(-1) + 48 * 2.0 ** -24 * v.abs().sum(-1), "sum")


def test_far_strides():
    """Tokens and rows so far apart that offsets pass 32 bits; past 2^24 elements
    between tokens inputs are copied."""
    a, soft, grads = scan_inputs(B=2, T=140, D=8, N=4, dtype=BF16)
    want = call(a, soft)
    far = torch.empty(140 * 2 + 1, (1 << 23) + 8, dtype=BF16, device="cuda")   # 4.7 GB
    x = far.as_strided((2, 140, 8), (far.stride(0) * 140, far.stride(0), 1))
    x.copy_(a["x"])
    assert torch.equal(call(a, soft, x=x)[0], want[0])
    leaf = x.detach().requires_grad_()
    y, h = call(a, soft, x=leaf)
    ref = a["x"].detach().requires_grad_()
    y2, h2 = call(a, soft, x=ref)
    assert torch.equal(torch.autograd.grad([y, h], leaf, list(grads))[0], torch.autograd.grad([y2, h2], ref, list(grads))[0])
    wide = far.view(-1).as_strided((2, 17, 8), ((1 << 24) * 17 // 2 + 4, 1 << 24, 1))
    wide.copy_(a["x"][:, :17])
    b = {n: t if t is None or t.dim() != 3 or n in ("initial_state",) else t[:, :17] for n, t in a.items()}
    b.update(B=a["B"][:, :17], C=a["C"][:, :17])
    assert torch.equal(call(dict(b, x=wide), soft)[0], call(b, soft)[0])


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("name", ["x", "dt", "B", "C", "gate"])
def test_values_that_are_not_finite(name, bad):
    """They reach their token and later ones of their sequence, no other sequence and
    (of x, dt and the gate) no other channel; what lies in tokens of no sequence
    reaches nothing."""
    cu = [4, 60, 95]
    a, soft, grads = scan_inputs(T=120, D=40, N=8, dtype=BF16, seqs=2, seed=5)
    clean, state = call(a, soft, cu)
    t = a[name].clone()
    t[0, :4] = bad
    t[0, 95:] = bad
    y, h = call(dict(a, **{name: t}), soft, cu)
    assert torch.equal(y, clean) and torch.equal(h, state)
    leaf = {n: v if v is None else v.detach().requires_grad_() for n, v in dict(a, **{name: t}).items()}
    pure = {n: v if v is None else v.detach().requires_grad_() for n, v in a.items()}
    names = [n for n in leaf if leaf[n] is not None]
    for n, g, w in zip(names, torch.autograd.grad(call(leaf, soft, cu), [leaf[n] for n in names], list(grads)),
                       torch.autograd.grad(call(pure, soft, cu), [pure[n] for n in names], list(grads))):
        assert torch.equal(g, w), n
    # in the last token of the first sequence, whose tile has empty places behind it
    t = a[name].clone()
    at = (0, 59, 0, 3) if name in "BC" else (0, 59, 7)
    t[at] = bad
    y, h = call(dict(a, **{name: t}), soft, cu)
    assert torch.equal(y[:, :59], clean[:, :59]) and torch.equal(y[:, 60:], clean[:, 60:])
    assert torch.equal(h[1], state[1])
    if name not in "BC":
        keep = [c for c in range(40) if c != 7]
        assert torch.equal(y[..., keep], clean[..., keep]) and torch.equal(h[:, keep], state[:, keep])


def test_a_bad_last_token_costs_the_rates_no_more_than_its_own_gradient():
    """x of the last token is infinite and its outputs' gradient zero: the rates'
    gradient comes from the states before it, which are finite."""
    a, soft, (dy, dhT) = scan_inputs(T=21, D=5, N=4, gate=False, state=False)
    a["x"] = a["x"].clone()
    dy[:, 20] = 0
    A = a["A"].detach().requires_grad_()
    want = torch.autograd.grad(call(a, soft, A=A)[0], A, dy)[0]
    a["x"][:, 20] = float("inf")
    got = torch.autograd.grad(call(a, soft, A=A)[0], A, dy)[0]
    assert torch.equal(got, want)


def test_rates_of_minus_infinity_forget():
    """e^{dt A} is 0 wherever there is a step; the empty places behind a sequence's
    last token, which have none, do not make NaN of it."""
    a, soft, grads = scan_inputs(T=19, D=6, N=5, gate=False)
    a["A"][:, 2] = -float("inf")
    y, h = call(a, soft)
    want = (up(a["x"])[0, 18] * torch.logaddexp(up(a["dt"] + a["dt_bias"])[0, 18], torch.zeros(6).double()))
    off = (h[0, :, 2].double().cpu() - want * up(a["B"])[0, 18, 0, 2]).abs()
    assert torch.isfinite(y).all() and (off <= 2.0 ** -20 * (want * up(a["B"])[0, 18, 0, 2]).abs() + 1e-30).all()


def test_same_bits_twice():
    a, soft, grads = scan_inputs(B=3, T=200, D=300, N=16, dtype=BF16)
    first, second = (check_free(a, soft, grads) for _ in range(2))
    for s, t in zip(first, second):
        assert torch.equal(s, t)


def check_free(a, soft, grads):
    leaf = {n: None if t is None else t.detach().requires_grad_() for n, t in a.items()}
    y, h = call(leaf, soft)
    return [y, h, *torch.autograd.grad([y, h], [t for t in leaf.values() if t is not None], list(grads))]


def test_one_gradient_alone():
    """Of the outputs or of the states, the other not given."""
    a, soft, grads = scan_inputs(B=1, T=40, D=12, N=8, seed=2)
    val = [scan_exact(a, soft, g) for g in ((grads[0], torch.zeros_like(grads[1])), (torch.zeros_like(grads[0]), grads[1]))]
    for i in range(2):
        leaf = {n: None if t is None else t.detach().requires_grad_() for n, t in a.items()}
        out = call(leaf, soft)
        names = ["x", "dt", "A", "initial_state"]
        for n, g in zip(names, torch.autograd.grad(out[i], [leaf[n] for n in names], grads[i])):
            key = dict(x="d_x", dt="d_dt", A="d_A", initial_state="d_h0")[n]
            check(g, val[i][0][key], val[i][1][key], n)


def test_on_another_stream():
    a, soft, grads = scan_inputs(B=2, T=70, D=40, N=8, dtype=BF16)
    want = check_free(a, soft, grads)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = check_free(a, soft, grads)
    s.synchronize()
    for x, y in zip(got, want):
        assert torch.equal(x, y)


@pytest.mark.parametrize("packed", [False, True])
def test_in_a_graph(packed):
    """Captured and replayed with other inputs and, packed, other offsets in place."""
    a, soft, _ = scan_inputs(T=200, D=40, N=8, dtype=BF16, seqs=3 if packed else None)
    from uttt_amd.state_space import selective_scan
    cu = torch.tensor([0, 50, 51, 180], device="cuda") if packed else None

    def run():
        return selective_scan(*(a[n] for n in ("x", "dt", "A", "B", "C")), D=a["D"], gate=a["gate"], dt_bias=a["dt_bias"],
                              dt_softplus=soft, initial_state=a["initial_state"], output_final_state=True, cu_seqlens=cu)

    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for i in range(4):
        a["x"].copy_(torch.randn(a["x"].shape, device="cuda"))
        if packed:
            cu.copy_(torch.tensor([[0, 50, 51, 180], [10, 10, 200, 200], [0, 64, 128, 150], [0, 1, 2, 3]][i], device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        want = run()
        torch.cuda.synchronize()
        for x, y in zip(out, want):
            assert torch.equal(x, y), i


def test_backward_in_a_graph():
    """A whole training pass captured, with no eager graph of the same leaves alive."""
    a, soft, grads = scan_inputs(T=150, D=40, N=16, dtype=BF16)
    leaf = {n: None if t is None else t.detach().requires_grad_() for n, t in a.items()}
    wanted = [t for t in leaf.values() if t is not None]

    def run():
        y, h = call(leaf, soft)
        return [y.detach(), h.detach(), *torch.autograd.grad([y, h], wanted, list(grads))]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        run()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for i in range(3):
        with torch.no_grad():
            leaf["dt"].copy_(torch.randn(leaf["dt"].shape, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(out, run()):
            assert torch.equal(x, y), i
        torch.cuda.synchronize()


# --------------------------------------------------------------- by tokens --
def step(a, soft, state, idx=None):
    from uttt_amd.state_space import selective_scan_step
    return selective_scan_step(*(a[n] for n in ("x", "dt", "A", "B", "C")), state, D=a["D"], gate=a["gate"],
                               dt_bias=a["dt_bias"], dt_softplus=soft, state_indices=idx)


@pytest.mark.parametrize("D,N,G", [(1, 1, 1), (5, 3, 1), (64, 16, 1), (66, 16, 2), (130, 7, 1), (300, 64, 3), (257, 8, 1), (90, 33, 2)])
@pytest.mark.parametrize("T", [1, 2, 5])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_step(D, N, G, T, dtype):
    a, soft, _ = scan_inputs(B=4, T=T, D=D, N=N, G=G, dtype=dtype, gate=T != 2, bias=T != 5, seed=D + T)
    val, err = scan_exact(a, soft)
    state = a["initial_state"].clone()
    y = step(a, soft, state)
    check(y, val["y"], err["y"], "y")
    check(state, val["state"], err["state"], "state")


def test_step_rows_of_a_pool():
    """Padded rows, indices that are no slot, slots of a pool of all layers, rows that
    name one slot (one after another), and slots that nobody names."""
    a, soft, _ = scan_inputs(B=7, T=2, D=70, N=16, dtype=BF16, seed=1)
    pool = torch.randn(6, 3, 70, 16, device="cuda")
    before = pool.clone()
    for dtype in (torch.int32, torch.int64):
        pool.copy_(before)
        idx = torch.tensor([4, -1, 0, 4, 9, 2, 4], dtype=dtype, device="cuda")
        y = step(a, soft, pool[:, 1], idx)
        ref = before.clone()
        want = torch.zeros_like(y)
        for row, slot in enumerate(idx.tolist()):
            if 0 <= slot < 6:
                one = {n: t if t is None or n in ("A", "D", "dt_bias") else t[row:row + 1] for n, t in a.items()}
                s = ref[slot:slot + 1, 1].clone()
                want[row] = step(one, soft, s)[0]
                ref[slot, 1] = s[0]
        assert torch.equal(y, want) and torch.equal(pool, ref)
        assert (y[1] == 0).all() and (y[4] == 0).all()


def test_step_many_rows_of_one_slot():
    a, soft, _ = scan_inputs(B=600, T=1, D=8, N=4, seed=1)
    idx = torch.zeros(600, dtype=torch.int32, device="cuda")
    state = torch.randn(2, 8, 4, device="cuda")
    h = state[:1].clone()
    y = step(a, soft, state, idx)
    whole = {n: t if t is None or n in ("A", "D", "dt_bias") else t.transpose(0, 1) for n, t in a.items()}
    val, err = scan_exact(dict(whole, initial_state=h), soft)
    check(y.transpose(0, 1), val["y"], err["y"], "y")
    check(state[:1], val["state"], err["state"], "state")


def test_step_carries_a_prompt_on():
    """A prompt's final state, then tokens one by one, against the whole sequence."""
    a, soft, _ = scan_inputs(B=2, T=40, D=30, N=12, seed=4)
    val, err = scan_exact(a, soft)
    cut = lambda s: {n: t if t is None or t.dim() < 3 or n == "initial_state" else t[:, s] for n, t in a.items()}  # noqa: E731
    _, state = call(cut(slice(0, 33)), soft)
    for t in range(33, 40):
        y = step(cut(slice(t, t + 1)), soft, state)
        check(y, val["y"][:, t:t + 1], err["y"][:, t:t + 1], t)
    check(state, val["state"], err["state"], "state")


def test_step_without_rows_or_tokens():
    a, soft, _ = scan_inputs(B=3, T=1, D=8, N=4)
    state = torch.randn(3, 8, 4, device="cuda")
    before = state.clone()
    none = {n: t if t is None or t.dim() < 3 else t[:, :0] for n, t in a.items()}
    assert step(none, soft, state).shape == (3, 0, 8) and torch.equal(state, before)
    none = {n: t if t is None or t.dim() < 3 else t[:0] for n, t in a.items()}
    assert step(none, soft, state).shape == (0, 1, 8) and torch.equal(state, before)


def test_step_in_a_graph():
    a, soft, _ = scan_inputs(B=3, T=1, D=70, N=16, dtype=BF16)
    state = torch.randn(5, 70, 16, device="cuda")
    idx = torch.tensor([3, 0, -1], dtype=torch.int32, device="cuda")
    eager = state.clone()
    step(a, soft, state.clone(), idx)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(a, soft, state, idx)
    for i in range(4):
        a["x"].copy_(torch.randn(a["x"].shape, device="cuda"))
        idx.copy_(torch.tensor([[3, 0, -1], [1, 1, 1], [4, 2, 0], [-1, 7, 3]][i], device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        want = step(a, soft, eager, idx)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(state, eager), i
