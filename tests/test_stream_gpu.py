"""The causal decoder for whole recordings and running streams (models/components/stream.py): its forward and backward pass against autograd in 64 bits,
its frame-by-frame form against its whole form, and the network that contains it."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def rel(a, b):
    a, b = a.double().cpu(), b.double().cpu()
    return ((a - b).norm() / b.norm().clamp_min(1e-30)).item()


def bucket(rel_pos, n, m):
    d = max(0, -rel_pos)
    e = n // 2
    return d if d < e else e + max(k for k in range(n - e) if k == 0 or d ** (n - e) * e ** k >= m ** k * e ** (n - e))


def make(dev, D, L):
    from pseldnets_amd.models.components.arena import ParamArena
    from pseldnets_amd.models.components.stream import StreamDecoder
    arena = ParamArena()
    dec = StreamDecoder(arena, 's.', D, L)
    g = torch.Generator().manual_seed(5)
    init = {}
    for name in arena.entries:
        shape = arena.offsets[name][1]
        t = torch.randn(shape, generator=g) * (0.5 if 'table' in name else 1.0 / math.sqrt(shape[-1]) if len(shape) == 2 else 0.1)
        init[name] = t + 1.0 if 'norm' in name and name.endswith('weight') else t
    arena.materialize(dev, init)
    return dec, arena, init


def definition(dec, p, x, lens):
    """The decoder in plain torch, 64 bits, recording by recording; x and p require gradients as the caller set them."""
    D, hq, hk, hd = dec.D, dec.heads, dec.kv_heads, dec.hd
    F = torch.nn.functional
    out, row = [], 0
    for n in lens:
        y = x[row:row + n]
        row += n
        for li in range(dec.L):
            w = lambda k: p[f's.layers.{li}.{k}']      # noqa: E731
            qkv = F.linear(F.layer_norm(y, (D,), w('norm1.weight'), w('norm1.bias'), 1e-5), w('self_attn.in_proj_weight'), w('self_attn.in_proj_bias'))
            q, k, v = qkv.split([hq * hd, hk * hd, hk * hd], 1)
            idx = torch.tensor([[bucket(j - i, dec.num_buckets, dec.max_distance) for j in range(n)] for i in range(n)])
            future = torch.ones(n, n).triu(1).bool()
            heads = []
            for h in range(hq):
                kv = h // (hq // hk)
                s = q[:, h * hd:(h + 1) * hd] @ k[:, kv * hd:(kv + 1) * hd].t() / math.sqrt(hd) + w('self_attn.relative_position_bias_table')[idx, h]
                heads.append(torch.softmax(s.masked_fill(future, -math.inf), -1) @ v[:, kv * hd:(kv + 1) * hd])
            y = y + F.linear(torch.cat(heads, 1), w('self_attn.out_proj.weight'), w('self_attn.out_proj.bias'))
            u = F.linear(F.layer_norm(y, (D,), w('norm2.weight'), w('norm2.bias'), 1e-5), w('linear1.weight'), w('linear1.bias'))
            state, hs = torch.zeros(D, dtype=torch.float64), []
            for t in range(n):
                z = torch.sigmoid(u[t, :D])
                state = z * state + (1 - z) * u[t, D:]
                hs.append(state)
            y = y + F.linear(torch.stack(hs), w('linear2.weight'), w('linear2.bias'))
        out.append(y)
    return torch.cat(out)


# 2-norms over a tensor: f32 rounds at 2^-24 some 20 times a layer and sums at most 128 terms, 1e-5 covers it. bf16 rounds every stored activation and gradient
# once (2^-9 of its 2-norm at the root mean square), about 8 of them a layer and direction add up as roots of sums of squares: 2 layers, both directions: 2^-9 * sqrt(32) =
# 1.1e-2, and weights are rounded too: 3e-2.
@pytest.mark.parametrize("dtype,tol", [(torch.float32, 1e-5), (torch.bfloat16, 3e-2)])
@pytest.mark.parametrize("D", [64, 256])
def test_against_autograd(dev, dtype, tol, D):
    from pseldnets_amd import ops
    lens, L = [33, 1, 70], 2
    dec, arena, init = make(dev, D, L)
    g = torch.Generator().manual_seed(1)
    x, dy = (torch.randn(sum(lens), D, generator=g).to(dtype).to(dev) for _ in range(2))
    y, saved = dec.forward_packed(x, ops.packed_plan(lens, device=dev))
    dx = dec.backward(dy, saved)
    p = {k: v.double().requires_grad_(True) for k, v in init.items()}
    xr = x.double().cpu().requires_grad_(True)
    yr = definition(dec, p, xr, lens)
    yr.backward(dy.double().cpu())
    assert rel(y, yr.detach()) < tol and rel(dx, xr.grad) < tol
    for name, t in p.items():
        assert rel(arena.g(name), t.grad) < 4 * tol, name      # a parameter's gradient sums over rows whose errors share a sign at worst


@pytest.mark.parametrize("dtype,tol", [(torch.float32, 1e-5), (torch.bfloat16, 3e-2)])
def test_stream_equals_recording(dev, dtype, tol):
    """Three streams stepped frame by frame give what the whole recordings give, and a full cache refuses the next frame."""
    from pseldnets_amd import _lib
    T, S, D = 45, 3, 256
    dec, _, _ = make(dev, D, 2)
    x = torch.randn(S, T, D, generator=torch.Generator().manual_seed(2)).to(dtype).to(dev)
    whole, _ = dec.forward(x.reshape(S * T, D), S, T)
    state = dec.stream_state(S, T, dev, dtype)
    for t in range(T):
        y = dec.step(x[:, t].contiguous(), state)
        assert rel(y, whole.view(S, T, D)[:, t]) < tol, t
    with pytest.raises(_lib.PseldError):
        dec.step(x[:, 0].contiguous(), state)


def test_stream_step_in_a_captured_graph(dev):
    S, D, cap = 2, 64, 40
    dec, _, _ = make(dev, D, 2)
    x = torch.randn(S, 8, D, generator=torch.Generator().manual_seed(3)).to(dev)
    eager, held = dec.stream_state(S, cap, dev, torch.float32), dec.stream_state(S, cap, dev, torch.float32)
    want = [dec.step(x[:, t].contiguous(), eager) for t in range(8)]
    slot = x[:, 0].contiguous()
    dec.step(slot, held)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = dec.step(slot, held)
    for t in range(1, 8):
        slot.copy_(x[:, t])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want[t]), t


def test_network_with_the_stream_decoder_trains(dev):
    """CRNN with cfg.model.decoder = 'stream': the output's shape, every parameter gets a gradient. No frame's output
    depends on later decoder input (checked on the decoder)."""
    from types import SimpleNamespace as A
    from oracle import crnn as oc
    from oracle import synth
    from pseldnets_amd.loss.multi_accdoa import Losses
    from pseldnets_amd.models import multi_accdoa
    cfg = A(data=A(n_mels=64, sample_rate=24000, hoplen=240), model=A(decoder='stream', num_decoder_layers=1), adapt=A())
    net = multi_accdoa.CRNN(cfg, 3, 7, encoder='CNN12', pretrained_path=None, num_features=[8, 16, 16, 32, 32, 64])
    net.to(dev).train()
    x = oc.random_features(2, seed=1).to(dev)
    pred = net(x)
    ld = Losses('mse', 'loss_all')(pred, {'adpit_label': synth.formula_adpit_label(2, 100, 3).to(dev)})
    ld['loss_all'].backward()
    for name, p in net.named_parameters():
        assert p.grad is not None and bool(torch.isfinite(p.grad).all()), name
        if 'decoder' in name:
            assert p.grad.abs().max().item() > 0, name
    dec = net.dec_blocks
    a = torch.randn(30, 64, device=dev)
    b = a.clone()
    b[20:] = 0
    assert torch.equal(dec.forward(a, 1, 30)[0][:20], dec.forward(b, 1, 30)[0][:20])


def test_a_captured_pass_survives_other_shapes(dev):
    """The plans of chunk batches stay where a captured graph reads them, whatever shapes come between the replays."""
    dec, _, _ = make(dev, 64, 1)
    x = torch.randn(2 * 70, 64, generator=torch.Generator().manual_seed(4)).to(dev)
    want = dec.forward(x, 2, 70)[0]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = dec.forward(x, 2, 70)[0]
    first = dec._plans[(2, 70, x.device)]
    for B, T in ((1, 140), (4, 35), (140, 1)):
        dec.forward(x, B, T)
        junk = [torch.full((n,), 1 << 30, dtype=torch.int32, device=dev) for n in (8, 64, 512, 4096)]      # what a freed plan's memory would be given to
        y.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want) and len(junk) == 4
    assert dec._plans[(2, 70, x.device)] is first


def test_step_refuses_other_frames_and_leaves_the_streams_as_they_were(dev):
    from pseldnets_amd import _lib
    dec, _, _ = make(dev, 64, 1)
    state = dec.stream_state(2, 5, dev, torch.float32)
    x = torch.randn(2, 64, device=dev)
    for bad in (x[:1], torch.zeros(3, 64, device=dev), torch.zeros(2, 32, device=dev), x.bfloat16(), x.cpu()):
        with pytest.raises(_lib.PseldError):
            dec.step(bad, state)
    assert state.frames == 0 and state.plan.k_len.tolist() == [0, 0]
    assert torch.equal(dec.step(x, state), dec.step(x, dec.stream_state(2, 5, dev, torch.float32)))


def test_step_takes_a_frame_out_of_a_recording(dev):
    """x[:, t] of a [streams, T, D] tensor, whose rows lie apart: the same outputs and states as contiguous frames."""
    S, T, D = 3, 6, 64
    dec, _, _ = make(dev, D, 2)
    x = torch.randn(S, T, D, generator=torch.Generator().manual_seed(6)).to(dev)
    a, b = (dec.stream_state(S, T, dev, torch.float32) for _ in range(2))
    for t in range(T):
        assert torch.equal(dec.step(x[:, t], a), dec.step(x[:, t].contiguous(), b)), t
        assert a.frames == t + 1 and a.plan.k_len.tolist() == [t + 1] * S
    assert all(torch.equal(p, q) for p, q in zip(a.keys + a.values + a.states, b.keys + b.values + b.states))


def test_step_refuses_states_that_are_not_its_own(dev):
    """Another decoder's state, a type the kernels are not built for: refused before anything moves."""
    from pseldnets_amd import _lib
    dec, _, _ = make(dev, 64, 1)
    deeper, _, _ = make(dev, 64, 2)
    with pytest.raises(_lib.PseldError):
        dec.stream_state(2, 5, dev, torch.float16)
    x = torch.randn(2, 64, device=dev)
    state = deeper.stream_state(2, 5, dev, torch.float32)
    with pytest.raises(_lib.PseldError):
        dec.step(x, state)
    shallow = dec.stream_state(2, 5, dev, torch.float32)
    with pytest.raises(_lib.PseldError):
        deeper.step(x, shallow)
    for s in (state, shallow):
        assert s.frames == 0 and s.plan.k_len.tolist() == [0, 0]


def test_a_step_that_fails_half_way_leaves_the_streams_as_they_were(dev, monkeypatch):
    """An error in the second layer (memory that runs out, say): the frame can be given again."""
    from pseldnets_amd import ops
    S, T, D = 2, 4, 64
    dec, _, _ = make(dev, D, 2)
    x = torch.randn(S, T, D, generator=torch.Generator().manual_seed(7)).to(dev)
    a, b = (dec.stream_state(S, T, dev, torch.float32) for _ in range(2))
    real, calls = ops.linrec_fwd, []

    def failing(*args, **kw):
        calls.append(1)
        if len(calls) == 6:                                 # the third frame's second layer
            raise MemoryError
        return real(*args, **kw)
    for t in range(T):
        frame = x[:, t].contiguous()
        monkeypatch.setattr(ops, 'linrec_fwd', failing)
        try:
            y = dec.step(frame, a)
        except MemoryError:
            assert t == 2 and a.frames == 2 and a.plan.k_len.tolist() == [2, 2]
            y = dec.step(frame, a)
        monkeypatch.setattr(ops, 'linrec_fwd', real)
        assert torch.equal(y, dec.step(frame, b)), t
    assert len(calls) == 10 and all(torch.equal(p, q) for p, q in zip(a.states, b.states))


def test_replays_up_to_the_capacity_and_past_it(dev):
    """Counted replays: every frame that fits is right, the next is refused by advance(). Replays that nobody counted: frames past the capacity are NaN,
    from a replay as from an eager call, and so is every later one."""
    from pseldnets_amd import _lib
    S, D, cap = 2, 64, 6
    dec, _, _ = make(dev, D, 2)
    x = torch.randn(S, cap + 3, D, generator=torch.Generator().manual_seed(8)).to(dev)
    eager = dec.stream_state(S, cap, dev, torch.float32)
    want = [dec.step(x[:, t].contiguous(), eager) for t in range(cap)]
    for counted in (True, False):
        held = dec.stream_state(S, cap, dev, torch.float32)
        slot = x[:, 0].contiguous()
        assert torch.equal(dec.step(slot, held), want[0]) and held.frames == 1
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = dec.step(slot, held)
        assert held.frames == 1 and held.remaining() == cap - 1      # the capture itself ran nothing
        for t in range(1, cap):
            if counted:
                held.advance()
            slot.copy_(x[:, t])
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, want[t]), t
        assert held.plan.k_len.tolist() == [cap] * S
        if counted:
            assert held.remaining() == 0
            for call in (held.advance, lambda: held.advance(2), lambda: dec.step(slot, held)):
                with pytest.raises(_lib.PseldError):
                    call()
            assert held.frames == cap
        for t in range(cap, cap + 3):
            slot.copy_(x[:, t])
            graph.replay()
            torch.cuda.synchronize()
            assert bool(torch.isnan(y).all()), t
        if not counted:
            assert bool(torch.isnan(dec.step(slot, held)).all())


def test_einv2_network_with_the_stream_decoder_trains(dev):
    """EINV2: the parameters of all six decoders get a gradient."""
    from types import SimpleNamespace as A
    from oracle import crnn as oc
    from pseldnets_amd.models import einv2
    cfg = A(data=A(n_mels=64, sample_rate=24000, hoplen=240), model=A(decoder='stream', num_decoder_layers=1), adapt=A())
    net = einv2.CRNN(cfg, 3, 7, encoder='CNN12', pretrained_path=None, num_features=[8, 16, 16, 32, 32, 64])
    net.to(dev).train()
    pred = net(oc.random_features(2, seed=1).to(dev))
    (pred['sed'].float().square().mean() + pred['doa'].float().square().mean()).backward()
    seen = set()
    for name, p in net.named_parameters():
        assert p.grad is not None and bool(torch.isfinite(p.grad).all()), name
        if '.decoder.' in name:
            assert p.grad.abs().max().item() > 0, name
            seen.add(name.split('.')[0])
    assert len(seen) == 6
