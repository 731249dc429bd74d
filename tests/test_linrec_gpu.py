"""The gated linear recurrence (csrc/linrec.hip) against its definition in 64 bits, frame by frame.

Tolerances. u = 2^-24. A step's z and 1 - z are off by at most 4u relative (exponential, reciprocal, one product), its two products and one sum
add less than 4u more, so a step adds at most 8u M to a state bounded by M = max(|n|, |h0|); earlier errors shrink by z per step, so the sum stays
below 8u M L with L = min(longest recording, 1 / min(1 - z)). 16u M L leaves a factor of two for the order of composition. lambda likewise with
its own bound; a product's error is the sum of its factors' relative errors. Outputs in bf16 are rounded once: 2^-8 of the value on top."""
import pytest
import torch

U = 2.0 ** -24


def rounding(dtype):
    return 2.0 ** -8 if dtype == torch.bfloat16 else U


def reference(g, n, lens, h0, reverse, dh, dlast):
    """(h, h_last, dg, dn, dh0, lambda) by loops over frames, float64 on the CPU."""
    g, n, dh = g.double().cpu(), n.double().cpu(), dh.double().cpu()
    z, y = torch.sigmoid(g), torch.sigmoid(-g)
    h, dg, dn, lam = (torch.zeros_like(g) for _ in range(4))
    last, dh0 = h0.double().cpu().clone(), dlast.double().cpu().clone()
    row = 0
    for s, ln in enumerate(lens):
        order = list(range(row, row + ln))
        order = order[::-1] if reverse else order
        row += ln
        prev, before = last[s].clone(), {}
        for r in order:
            before[r] = prev
            prev = z[r] * prev + y[r] * n[r]
            h[r] = prev
        last[s] = prev
        mu = dh0[s].clone()
        for r in order[::-1]:
            lam[r] = dh[r] + mu
            dn[r] = lam[r] * y[r]
            dg[r] = lam[r] * (before[r] - n[r]) * z[r] * y[r]
            mu = z[r] * lam[r]
        dh0[s] = mu
    return h, last, dg, dn, dh0, lam


def close(name, got, ref, absolute, relative):
    got = got.double().cpu()
    over = (got - ref).abs() - relative * ref.abs() - absolute
    print(f"{name}: max|d|={(got - ref).abs().max().item() if ref.numel() else 0:.3e} allowed {absolute:.3e} + {relative:.1e} |ref|")
    assert got.shape == ref.shape and bool((over <= 0).all()), name


def make(dev, dtype, lens, C, seed, gate=1.0, spread=1.5):
    k = torch.Generator().manual_seed(seed)
    N = sum(lens)
    both = torch.randn(N, 2 * C, generator=k)
    both[:, :C] = both[:, :C] * spread + gate
    both = both.to(dtype).to(dev)
    dh = torch.randn(N, C, generator=k).to(dtype).to(dev)
    h0, dlast = (torch.randn(len(lens), C, generator=k).to(dev) for _ in range(2))
    return both, dh, h0, dlast


def run_and_check(dev, dtype, lens, C, reverse, seed, gate=1.0, spread=1.5):
    from pseldnets_amd import ops
    both, dh, h0, dlast = make(dev, dtype, lens, C, seed, gate, spread)
    g, n = both[:, :C], both[:, C:]                       # row-strided views of one projection's output
    plan = ops.packed_plan(lens, device=dev)
    h, last, saved = ops.linrec_fwd(g, n, plan, h0=h0, reverse=reverse)
    dgn = torch.full((sum(lens), 2 * C), float('nan'), dtype=dtype, device=dev)
    dg, dn, dh0 = ops.linrec_bwd(dh, g, n, saved, plan, dh_last=dlast, h0=h0, reverse=reverse, dg=dgn[:, :C], dn=dgn[:, C:])
    rh, rlast, rdg, rdn, rdh0, lam = reference(g, n, lens, h0, reverse, dh, dlast)
    y = torch.sigmoid(-g.double().cpu())
    L = min(max(lens), 1 / y.min().item() if y.numel() else 1) if max(lens) else 1
    M = max(n.double().abs().max().item() if n.numel() else 0, h0.abs().max().item())
    G = max(lam.abs().max().item() if lam.numel() else 0, dlast.abs().max().item())
    eh, el, r = 16 * U * M * L, 16 * U * G * L, rounding(dtype)
    close("h", h, rh, eh, r)
    close("h_last", last, rlast, eh, 0)
    close("dn", dn, rdn, el, r)
    close("dg", dg, rdg, el * 2 * M + G * eh + 16 * U * G * M, r)
    close("dh0", dh0, rdh0, el, 0)
    return h, last, dg, dn, dh0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("lens,C", [([1], 8), ([0], 16), ([7, 0, 1, 128, 129, 3], 64), ([127, 255, 256, 257], 72), ([1] * 37, 136),
                                    ([1000, 3, 0, 511], 40), ([2049], 8)])
def test_against_the_definition(dev, dtype, reverse, lens, C):
    run_and_check(dev, dtype, lens, C, reverse, 1)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("lens,C", [([12000, 1, 700, 9001], 24), ([257, 4000], 264)])
def test_recordings_cut_into_segments(dev, dtype, lens, C):
    """Long enough that one recording is shared between workgroups (the composition launch runs)."""
    from pseldnets_amd import _lib
    assert _lib.lib().pseld_linrec_workspace(sum(lens), len(lens), max(lens), C) > 0
    run_and_check(dev, dtype, lens, C, False, 2)
    run_and_check(dev, dtype, lens, C, True, 3)


@pytest.mark.gpu
def test_gates_that_saturate(dev):
    """Gates of +-60: states that never change (z rounds to one) and states that forget at once."""
    run_and_check(dev, torch.float32, [300, 20], 16, False, 4, gate=0.0, spread=60.0)


@pytest.mark.gpu
def test_gradient_against_differences(dev):
    """The gradients of <h, dh> + <h_last, dlast> against central differences of the forward pass in f32. A difference over 2e has an error of
    e^2 / 6 times a third derivative (below 10 here: products of factors below one, summed over 12 frames) plus the sum's rounding over 2 e:
    with e = 2^-6 that is 4e-4 + 2^-24 * 400 / 2^-5 = 1.2e-3; 4e-3 is allowed."""
    from pseldnets_amd import ops
    lens, C = [5, 12], 8
    both, dh, h0, dlast = make(dev, torch.float32, lens, C, 5)
    g, n = both[:, :C].contiguous(), both[:, C:].contiguous()
    plan = ops.packed_plan(lens, device=dev)

    def value(g, n, h0):
        h, last, _ = ops.linrec_fwd(g, n, plan, h0=h0, need_saved=False)
        return (h.double() * dh.double()).sum().item() + (last.double() * dlast.double()).sum().item()
    _, _, saved = ops.linrec_fwd(g, n, plan, h0=h0)
    grads = ops.linrec_bwd(dh, g, n, saved, plan, dh_last=dlast, h0=h0)
    e = 2.0 ** -6
    for which in range(3):
        for r, c in ((0, 0), (1, 5), (1, 2)):
            args = [[g.clone(), n.clone(), h0.clone()] for _ in range(2)]
            args[0][which][r, c] += e
            args[1][which][r, c] -= e
            diff = (value(*args[0]) - value(*args[1])) / (2 * e)
            assert abs(diff - grads[which][r, c].item()) < 4e-3, (which, r, c)


@pytest.mark.gpu
def test_frame_by_frame_equals_whole(dev):
    """A stream stepped one frame at a time through h0 / h_last gives the whole recording's states, to the rounding of a step each."""
    from pseldnets_amd import ops
    T, C, streams = 40, 32, 3
    both, _, h0, _ = make(dev, torch.float32, [T] * streams, C, 6)
    g, n = both[:, :C].contiguous().view(streams, T, C), both[:, C:].contiguous().view(streams, T, C)
    whole, last, _ = ops.linrec_fwd(g.view(-1, C), n.view(-1, C), ops.packed_plan([T] * streams, device=dev), h0=h0)
    step = ops.packed_plan([1] * streams, device=dev)
    s, M = h0, max(n.abs().max().item(), h0.abs().max().item())
    for t in range(T):
        h, s, _ = ops.linrec_fwd(g[:, t], n[:, t], step, h0=s, need_saved=False)
        close(f"frame {t}", h, whole.view(streams, T, C)[:, t].double().cpu(), 32 * U * M * T, 0)
    close("last", s, last.double().cpu(), 32 * U * M * T, 0)


@pytest.mark.gpu
def test_no_initial_state_optional_arguments_and_repeatability(dev):
    from pseldnets_amd import ops
    lens, C = [300, 5000], 16
    both, dh, _, _ = make(dev, torch.bfloat16, lens, C, 7)
    g, n = both[:, :C], both[:, C:]
    plan = ops.packed_plan(lens, device=dev)
    zero = torch.zeros(2, C, device=dev)
    a, la, sa = ops.linrec_fwd(g, n, plan)
    b, lb, sb = ops.linrec_fwd(g, n, plan, h0=zero)
    assert torch.equal(a, b) and torch.equal(la, lb)
    da = ops.linrec_bwd(dh, g, n, sa, plan)
    db = ops.linrec_bwd(dh, g, n, sb, plan, dh_last=zero, h0=zero)
    assert da[2] is None and torch.equal(da[0], db[0]) and torch.equal(da[1], db[1])
    for _ in range(3):
        c, lc, _ = ops.linrec_fwd(g, n, plan)
        assert torch.equal(a, c) and torch.equal(la, lc)


@pytest.mark.gpu
def test_side_stream_and_captured_graph(dev):
    from pseldnets_amd import ops
    lens, C = [700, 40], 24
    both, dh, h0, dlast = make(dev, torch.float32, lens, C, 8)
    plan = ops.packed_plan(lens, device=dev)
    x = both.clone()

    def step():
        h, last, saved = ops.linrec_fwd(x[:, :C], x[:, C:], plan, h0=h0)
        return (h, last) + ops.linrec_bwd(dh, x[:, :C], x[:, C:], saved, plan, dh_last=dlast, h0=h0)
    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for k in range(3):
        x.copy_(both * (1 + 0.25 * k))
        graph.replay()
        eager = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, eager))


@pytest.mark.gpu
def test_refusals(dev):
    from pseldnets_amd import _lib, ops
    plan = ops.packed_plan([4, 3], device=dev)
    g = torch.zeros(7, 16, device=dev)
    ok = torch.zeros(2, 16, device=dev)
    bad = [lambda: ops.linrec_fwd(g[:6], g[:6], plan),                              # rows that are not the plan's
           lambda: ops.linrec_fwd(g, g.bfloat16(), plan),                           # two types
           lambda: ops.linrec_fwd(g.half(), g.half(), plan),                        # a type the kernels are not built for
           lambda: ops.linrec_fwd(g[:, :12], g[:, :12], plan),                      # channels
           lambda: ops.linrec_fwd(torch.zeros(16, 7, device=dev).t(), g, plan),     # columns apart
           lambda: ops.linrec_fwd(torch.zeros(7, 18, device=dev)[:, 1:17], g, plan),  # rows off their boundary
           lambda: ops.linrec_fwd(g, g, plan, h0=ok[:1]),
           lambda: ops.linrec_fwd(g, g, plan, h0=ok.bfloat16()),
           lambda: ops.linrec_fwd(g.cpu(), g.cpu(), plan),
           lambda: ops.linrec_bwd(g, g, g, None, plan),
           lambda: ops.linrec_bwd(g, g, g, ok, plan),
           lambda: ops.packed_plan([], device=dev), lambda: ops.packed_plan([-1], device=dev), lambda: ops.packed_plan([3], [4], k_cap=3, device=dev),
           lambda: ops.packed_plan([1 << 30, 1 << 30], device=dev)]
    for k, call in enumerate(bad):
        with pytest.raises(_lib.PseldError):
            call()
            print("not refused:", k)


def test_c_entry_refuses_without_a_launch():
    """Argument checks come before anything touches a device: callable here without one."""
    import os
    from pseldnets_amd import _lib
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip("libpseld_hip.so not built")
    L = _lib.lib()
    P = 4096                                                # an address that is never followed
    fwd = lambda dtype=0, g=P, ldg=8, C=8, rows=4, longest=4, seqs=1, h=P, ws=None, nb=0: L.pseld_linrec_fwd(  # noqa: E731
        dtype, g, ldg, P, 8, None, h, 8, P, None, P, P, seqs, rows, longest, C, 0, ws, nb, None)
    for bad in (dict(dtype=7), dict(g=None), dict(ldg=9), dict(g=P + 4), dict(C=12), dict(C=0), dict(seqs=0), dict(longest=5), dict(rows=-1), dict(h=None),
                dict(rows=5000, longest=5000)):
        assert fwd(**bad) == -1, bad
    assert b"workspace" in L.pseld_last_error()
    assert L.pseld_linrec_bwd(0, None, 8, P, 8, P, 8, P, None, P, 8, P, 8, None, P, P, 1, 4, 4, 8, 0, None, 0, None) == -1
    assert L.pseld_linrec_workspace(60000, 2, 60000, 512) > 0 and L.pseld_linrec_workspace(100, 4, 40, 64) == 0


def test_c_entry_refuses_overlapping_results_and_too_many_rows():
    import os
    from pseldnets_amd import _lib
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip("libpseld_hip.so not built")
    L = _lib.lib()
    P, Q, R, S = (4096 * i for i in range(1, 5))            # addresses that are never followed

    def fwd(h=R, ldh=8, rows=4, longest=4):
        return L.pseld_linrec_fwd(0, P, 8, Q, 8, None, h, ldh, P, None, P, P, 1, rows, longest, 8, 0, None, 0, None)

    def bwd(dg=S, lddg=8, dn=5 * 4096, lddn=8):
        return L.pseld_linrec_bwd(0, R, 8, P, 8, Q, 8, P, None, dg, lddg, dn, lddn, None, P, P, 1, 4, 4, 8, 0, None, 0, None)
    for bad in (dict(h=P), dict(h=Q), dict(ldh=4), dict(ldh=0), dict(rows=(1 << 30) + 1)):
        assert fwd(**bad) == -1, bad
    for bad in (dict(dg=P), dict(dg=Q), dict(dg=R), dict(dn=P), dict(dn=Q), dict(dn=R), dict(dn=S), dict(lddg=4), dict(lddn=0)):
        assert bwd(**bad) == -1, bad


def test_plan_fails_loudly_without_gpu():
    import torch as t
    from pseldnets_amd import _lib, ops
    with pytest.raises(_lib.PseldError):
        ops.packed_plan([3, 4], device='cpu')
    assert not t.cuda.is_available() or ops.packed_plan([3, 4]).rows == 7


@pytest.mark.gpu
def test_backward_refuses_states_whose_rows_lie_apart(dev):
    """A strided view of the kept states has their shape and would be read as if it were packed: wrong gradients without an error."""
    from pseldnets_amd import _lib, ops
    lens, C = [100, 30], 16
    both, dh, _, _ = make(dev, torch.float32, lens, C, 9)
    g, n = both[:, :C], both[:, C:]
    plan = ops.packed_plan(lens, device=dev)
    _, _, saved = ops.linrec_fwd(g, n, plan)
    apart = torch.stack([saved, saved + 1], 1)[:, 0]
    assert torch.equal(apart, saved) and not apart.is_contiguous()
    with pytest.raises(_lib.PseldError):
        ops.linrec_bwd(dh, g, n, apart, plan)
    want = ops.linrec_bwd(dh, g, n, saved, plan)
    got = ops.linrec_bwd(dh, g, n, apart.contiguous(), plan)
    assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_states_into_a_view_of_the_caller(dev, dtype):
    from pseldnets_amd import ops
    lens, C = [65, 0, 300], 40
    both, _, h0, _ = make(dev, dtype, lens, C, 10)
    plan = ops.packed_plan(lens, device=dev)
    wide = torch.full((sum(lens), 3 * C), float('nan'), dtype=dtype, device=dev)
    for reverse in (False, True):
        want, last, _ = ops.linrec_fwd(both[:, :C], both[:, C:], plan, h0=h0, reverse=reverse)
        got, last2, _ = ops.linrec_fwd(both[:, :C], both[:, C:], plan, h0=h0, reverse=reverse, out=wide[:, C:2 * C])
        assert got.data_ptr() == wide[:, C:].data_ptr() and torch.equal(got, want) and torch.equal(last, last2)
        assert bool(torch.isnan(wide[:, :C]).all()) and bool(torch.isnan(wide[:, 2 * C:]).all())
