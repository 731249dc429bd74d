"""Attention over packed recordings (csrc/packed_attn.hip) and its bucketed relative position bias against their definition in 64 bits.

Tolerances, elementwise. u = 2^-24, r = the output type's half step (2^-8 bf16, u f32), p = 2^-8 for bf16 operands (probabilities and score gradients are
rounded to bf16 before the second product), 0 for f32.
  probabilities: a score is a sum of D products in f32, off by at most (2 D + 32) u times the sum of its terms' sizes, the exponential and the row's sum of n
  terms add at most n u more: relative rho = u (2 D + 32 + n) (1 + max scale |q| |k| + |bias|).
  out: (p + rho) sum P |v| + r |out|.    lse: rho.
  delta: rho sum P |dP|, plus sum |dO| (error of out) where it comes from the stored out (f32 operands, or no table gradient wanted).
  dS: P (rho |dP - delta| + 2 D u sum |dO| |v| + error of delta) =: e;  dq: scale sum (e + p |dS|) |k| + r |dq|;  dk likewise with q over the group's heads;
  dv: (p + rho) sum P |dO| + r |dv|;  dtable: sum of e over the bucket's pairs + 64 u sum |dS|."""
import math

import pytest
import torch

U = 2.0 ** -24


def bucket_by_formula(rel, buckets, max_distance, bidirectional):
    """Bucket of key - query by comparing whole numbers, distance by distance (64-bit logarithms could miss a border)."""
    side = buckets // 2 if bidirectional else buckets
    base = side if bidirectional and rel > 0 else 0
    n = abs(rel) if bidirectional else max(0, -rel)
    e = side // 2
    if n < e:
        return base + n
    K = side - e
    return base + e + max(k for k in range(K) if k == 0 or n ** K * e ** k >= max_distance ** k * e ** K)


def reference(q, k, v, dout, q_lens, k_lens, k_starts, causal, scale, table=None, rel=None, stored_out=True):
    """Every output with its allowed error, float64 on the CPU: {name: (value, error without the output's own rounding)}."""
    p8 = 2.0 ** -8 if q.dtype == torch.bfloat16 else 0.0
    q, k, v = q.double().cpu(), k.double().cpu(), v.double().cpu()
    N, hq, D = q.shape
    hkv = k.shape[1]
    G = hq // hkv
    out, eout = torch.zeros_like(q), torch.zeros_like(q)
    lse, else_ = torch.full((N, hq), -math.inf, dtype=torch.float64), torch.zeros(N, hq, dtype=torch.float64)
    res = {}
    if dout is not None:
        dout = dout.double().cpu()
        dq, edq = torch.zeros_like(q), torch.zeros_like(q)
        dk, edk, dv, edv = (torch.zeros_like(k) for _ in range(4))
    if table is not None:
        table = table.double().cpu()
        dt, edt = torch.zeros_like(table), torch.zeros_like(table)
        span = max(list(q_lens) + list(k_lens)) + 1
        lut = torch.tensor([bucket_by_formula(r, *rel) for r in range(-span, span + 1)])
    row = 0
    for nq, nk, ks in zip(q_lens, k_lens, k_starts):
        a, b = slice(row, row + nq), slice(ks, ks + nk)
        row += nq
        if not nq or not nk:
            continue
        dist = torch.arange(nk)[None, :] - (torch.arange(nq)[:, None] + nk - nq)
        for h in range(hq):
            qq, kk, vv = q[a, h], k[b, h // G], v[b, h // G]
            s = scale * qq @ kk.t()
            size = scale * (qq.abs() @ kk.abs().t()).max().item()
            if table is not None:
                bias = table[lut[dist + span], h]
                s = s + bias
                size += bias.abs().max().item()
            live = dist <= 0 if causal else torch.ones_like(dist, dtype=torch.bool)
            s = s.masked_fill(~live, -math.inf)
            P = torch.nan_to_num(torch.softmax(s, -1), nan=0.0)
            rho = U * (2 * D + 32 + nk) * (1 + size)
            out[a, h] = P @ vv
            eout[a, h] = (p8 + rho) * (P @ vv.abs())
            lse[a, h] = torch.logsumexp(s, -1)
            else_[a, h] = rho * (1 + size)
            if dout is None:
                continue
            do = dout[a, h]
            dP = do @ vv.t()
            delta = (P * dP).sum(-1, keepdim=True)
            dS = P * (dP - delta)
            ed = rho * (P * dP.abs()).sum(-1, keepdim=True)
            if stored_out:
                r = 2.0 ** -8 if p8 else U
                ed = ed + (do.abs() * (eout[a, h] + r * out[a, h].abs())).sum(-1, keepdim=True) + 2 * D * U * (do.abs() * out[a, h].abs()).sum(-1, keepdim=True)
            e = P * (rho * (dP - delta).abs() + 2 * D * U * (do.abs() @ vv.abs().t()) + ed)
            eS = e + p8 * dS.abs()
            grow = 1 + U * (nq * G + nk)                      # the products' own f32 sums
            dq[a, h] = scale * dS @ kk
            edq[a, h] = grow * scale * eS @ kk.abs() + U * nk * scale * dS.abs() @ kk.abs()
            dk[b, h // G] += scale * dS.t() @ qq
            edk[b, h // G] += grow * scale * eS.t() @ qq.abs() + U * nq * G * scale * dS.abs().t() @ qq.abs()
            dv[b, h // G] += P.t() @ do
            edv[b, h // G] += (p8 + rho + U * nq * G) * P.t() @ do.abs()
            if table is not None:
                w = lut[dist + span].reshape(-1)
                dt[:, h].index_add_(0, w, dS.reshape(-1))
                edt[:, h].index_add_(0, w, (e + 64 * U * dS.abs()).reshape(-1))
    res = {'out': (out, eout), 'lse': (lse, else_)}
    if dout is not None:
        res.update(dq=(dq, edq), dk=(dk, edk), dv=(dv, edv))
        if table is not None:
            res['dtable'] = (dt, edt)
    return res


def compare(got, want):
    for name, t in got.items():
        ref, err = want[name]
        r = 2.0 ** -8 if t.dtype == torch.bfloat16 else U
        t = t.double().cpu()
        assert t.shape == ref.shape, name
        inf = torch.isinf(ref)
        assert torch.equal(inf, torch.isinf(t)) and not torch.isnan(t).any(), name
        d = torch.where(inf, torch.zeros_like(t), t - torch.where(inf, t, ref)).abs()
        over = d - (err + r * torch.where(inf, torch.zeros_like(ref), ref).abs() + 1e-30)
        worst = over.max().item() if over.numel() else 0.0
        print(f"{name}: max|d| = {d.max().item() if d.numel() else 0:.3e}, largest excess {worst:.3e}")
        assert worst <= 0, f"{name}: {int((over > 0).sum())} of {over.numel()} values off, by up to {worst:.3e} beyond the bound"


def rnd(shape, seed, dtype, dev, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype).to(dev)


def starts_of(lens):
    out, n = [], 0
    for x in lens:
        out.append(n)
        n += x
    return out


def case(dev, dtype, q_lens, hq, hkv, D, causal, bias=None, k_lens=None, cap=None, backward=True, seed=0, scale=None):
    """Runs one call through strided views of a projection (or of slabs with NaN behind every length) and checks every output."""
    from pseldnets_amd import ops
    plan = ops.packed_plan(q_lens, k_lens, k_cap=cap, device=dev)
    N, kl = sum(q_lens), k_lens if k_lens is not None else q_lens
    if k_lens is None:
        W = (hq + 2 * hkv) * D
        qkv = rnd((N, W), seed, dtype, dev)
        q, k, v = qkv[:, :hq * D].view(N, hq, D), qkv[:, hq * D:(hq + hkv) * D].view(N, hkv, D), qkv[:, (hq + hkv) * D:].view(N, hkv, D)
        dqkv = torch.full((N, W), float('nan'), dtype=dtype, device=dev)
        outs = dict(dq=dqkv[:, :hq * D].view(N, hq, D), dk=dqkv[:, hq * D:(hq + hkv) * D].view(N, hkv, D), dv=dqkv[:, (hq + hkv) * D:].view(N, hkv, D))
        ks = starts_of(q_lens)
    else:
        caps = [cap] * len(k_lens) if isinstance(cap, int) else cap if cap is not None else k_lens
        ks = starts_of(caps)
        q = rnd((N, hq, D), seed, dtype, dev)
        k, v = rnd((sum(caps), hkv, D), seed + 1, dtype, dev), rnd((sum(caps), hkv, D), seed + 2, dtype, dev)
        for s, (c, n) in enumerate(zip(caps, k_lens)):
            k[ks[s] + n:ks[s] + c] = float('nan')
            v[ks[s] + n:ks[s] + c] = float('nan')
        outs = {}
    table = rnd((bias[0], hq), seed + 3, torch.float32, dev, 0.7) if bias else None
    kw = dict(causal=causal, scale=scale)
    if bias:
        kw.update(bias_table=table, buckets=ops.relpos_buckets(*bias, device=dev))
    out, lse = ops.packed_attn_fwd(q, k, v, plan, **kw)
    got = {'out': out, 'lse': lse}
    dout = rnd((N, hq, D), seed + 4, dtype, dev) if backward else None
    if backward:
        if bias:
            got['dtable'] = torch.full_like(table, float('nan'))
            kw['dbias_table'] = got['dtable']
        got['dq'], got['dk'], got['dv'] = ops.packed_attn_bwd(dout, q, k, v, out, lse, plan, **outs, **kw)
    kc, vc = (torch.nan_to_num(x.double().cpu(), nan=0.0).to(dtype) for x in (k, v))
    want = reference(q, kc, vc, dout, q_lens, kl, ks, causal, scale if scale else D ** -0.5, table, bias, stored_out=not (bias and dtype == torch.bfloat16))
    compare(got, want)
    return got


DT = [torch.float32, torch.bfloat16]
RAGGED = [1, 0, 65, 129, 300, 31, 128, 7]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("hq,hkv,D", [(2, 2, 64), (4, 2, 128), (4, 1, 32), (3, 1, 24), (2, 2, 40), (6, 3, 96), (2, 1, 8)])
def test_whole_recordings(dev, dtype, causal, hq, hkv, D):
    case(dev, dtype, RAGGED, hq, hkv, D, causal)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("bias", [(32, 128, True), (32, 128, False), (8, 5, True), (2, 9, False), (320, 800, False), (64, 333, True), (512, 1024, True)])
@pytest.mark.parametrize("hq,hkv,D", [(4, 2, 64), (2, 1, 128)])
def test_position_bias(dev, dtype, causal, bias, hq, hkv, D):
    case(dev, dtype, [200, 1, 0, 333, 70], hq, hkv, D, causal, bias=bias)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("bias", [None, (32, 128, True), (16, 50, False)])
def test_distances_far_beyond_the_last_bucket(dev, dtype, bias):
    case(dev, dtype, [1100, 130], 2, 1, 64, bias is not None and not bias[2], bias=bias)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("causal", [False, True])
def test_keys_of_their_own_lengths(dev, dtype, causal):
    """Queries that are a recording's last frames, more queries than keys (rows without keys when causal), no keys, no queries; slabs whose rows
    behind the length are NaN."""
    case(dev, dtype, [40, 100, 33, 5, 0, 64], 4, 2, 64, causal, k_lens=[170, 60, 0, 5, 12, 64])
    case(dev, dtype, [40, 100, 33, 5, 0, 64], 4, 2, 64, causal, bias=(32, 128, True), k_lens=[170, 60, 0, 5, 12, 64], cap=[200, 64, 30, 5, 40, 300])
    case(dev, dtype, [64, 70], 2, 2, 32, causal, bias=(8, 20, False), k_lens=[500, 3], cap=512)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("hq,hkv,D,q_lens", [(8, 2, 64, [1, 1, 1, 1]), (16, 2, 128, [1, 0, 1, 1]), (4, 4, 32, [8, 3, 1, 0]), (32, 1, 64, [1] * 4),
                                             (3, 1, 24, [10, 2, 1, 1]), (6, 2, 96, [4, 1, 2, 3]), (2, 2, 8, [32, 1, 5, 31])])
@pytest.mark.parametrize("bias", [None, (32, 128, False), (64, 333, True)])
def test_few_rows(dev, dtype, hq, hkv, D, q_lens, bias):
    """The next frames of running streams: caches of one frame to several chunks, an empty one, the slab's tail NaN."""
    for causal in (True, False):
        case(dev, dtype, q_lens, hq, hkv, D, causal, bias=bias, k_lens=[700, 1, 0, 129], cap=768, backward=False)
        case(dev, dtype, q_lens, hq, hkv, D, causal, bias=bias, k_lens=[37, 256, 33, 32], cap=256, backward=False)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DT)
def test_few_rows_long_caches(dev, dtype):
    case(dev, dtype, [1, 1], 8, 2, 64, True, bias=(32, 128, False), k_lens=[20000, 9001], cap=20480, backward=False)
    case(dev, dtype, [2], 4, 1, 128, True, k_lens=[16385], cap=16400, backward=False)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DT)
def test_backward_of_few_rows(dev, dtype):
    """Recordings short enough for the few-rows forward still have their gradients."""
    case(dev, dtype, [2, 1, 0, 4], 4, 2, 64, True, bias=(32, 128, False))
    case(dev, dtype, [1], 1, 1, 32, False)


@pytest.mark.gpu
def test_large_scores_and_scale(dev):
    case(dev, torch.float32, [150, 20], 2, 1, 64, True, scale=2.0)
    case(dev, torch.bfloat16, [150, 20], 2, 1, 64, False, scale=3.0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DT)
def test_masking_by_the_table(dev, dtype):
    """A table whose far buckets are -inf (a learned window): rows keep their near keys, the probabilities beyond are exactly zero."""
    from pseldnets_amd import ops
    lens, hq, D = [300, 40], 2, 64
    plan = ops.packed_plan(lens, device=dev)
    buckets = ops.relpos_buckets(16, 64, bidirectional=False, device=dev)
    table = rnd((16, hq), 1, torch.float32, dev)
    table[12:] = -math.inf
    q, k, v = (rnd((sum(lens), hq, D), s, dtype, dev) for s in (2, 3, 4))
    out, lse = ops.packed_attn_fwd(q, k, v, plan, causal=True, bias_table=table, buckets=buckets)
    reach = [r for r in range(-64, 1) if buckets.host_lut[r + 64] < 12]
    for first, n in ((0, 300), (300, 40)):
        for i in (0, 5, n - 1):
            keys = [i + r for r in reach if i + r >= 0]
            for h in range(hq):
                s = D ** -0.5 * (k[first:first + n, h].double()[keys] @ q[first + i, h].double()).cpu() + \
                    torch.tensor([table[buckets.host_lut[j - i + 64], h].item() for j in keys], dtype=torch.float64)
                P = torch.softmax(s, 0)
                vv = v[first:first + n, h].double()[keys].cpu()
                bound = (2.0 ** -7 + 1e-4) * (P @ vv.abs()) if dtype == torch.bfloat16 else 1e-4 * (P @ vv.abs())
                assert bool(((out[first + i, h].double().cpu() - P @ vv).abs() <= bound).all())
                assert abs(lse[first + i, h].item() - torch.logsumexp(s, 0).item()) < 1e-4


@pytest.mark.gpu
def test_gradients_against_differences(dev):
    """Central differences of <out, dout> in f32. Every third derivative here stays below 8 (scores move by |k| scale e or by e, the softmax's
    derivatives are below one, 24 rows of unit gradients), so e = 2^-6 leaves e^2 / 6 * 8 = 3.3e-4; the value's rounding, 2^-24 * 200, over
    2 e adds 4e-4. 2e-3 is allowed."""
    from pseldnets_amd import ops
    lens, hq, hkv, D = [9, 15], 4, 2, 16
    plan = ops.packed_plan(lens, device=dev)
    buckets = ops.relpos_buckets(8, 12, True, device=dev)
    N = sum(lens)
    q, k, v = rnd((N, hq, D), 1, torch.float32, dev), rnd((N, hkv, D), 2, torch.float32, dev), rnd((N, hkv, D), 3, torch.float32, dev)
    table, dout = rnd((8, hq), 4, torch.float32, dev), rnd((N, hq, D), 5, torch.float32, dev)
    for causal in (False, True):
        kw = dict(causal=causal, buckets=buckets)
        out, lse = ops.packed_attn_fwd(q, k, v, plan, bias_table=table, **kw)
        dt = torch.empty_like(table)
        grads = ops.packed_attn_bwd(dout, q, k, v, out, lse, plan, bias_table=table, dbias_table=dt, **kw) + (dt,)

        def value(q, k, v, table):
            return (ops.packed_attn_fwd(q, k, v, plan, bias_table=table, **kw)[0].double() * dout.double()).sum().item()
        e = 2.0 ** -6
        for which, places in ((0, ((0, 0, 0), (20, 3, 7))), (1, ((0, 0, 0), (12, 1, 9))), (2, ((3, 0, 1), (23, 1, 15))), (3, ((0, 0), (1, 2), (3, 3)))):
            for at in places:
                args = [[q.clone(), k.clone(), v.clone(), table.clone()] for _ in range(2)]
                args[0][which][at] += e
                args[1][which][at] -= e
                diff = (value(*args[0]) - value(*args[1])) / (2 * e)
                assert abs(diff - grads[which][at].item()) < 2e-3, (causal, which, at)


@pytest.mark.gpu
def test_accumulated_table_gradient_and_repeatability(dev):
    from pseldnets_amd import ops
    lens, hq, hkv, D = [700, 130, 64], 4, 2, 64
    plan = ops.packed_plan(lens, device=dev)
    buckets = ops.relpos_buckets(device=dev)
    q, k, v, dout = (rnd((sum(lens), h, D), s, torch.bfloat16, dev) for s, h in ((1, hq), (2, hkv), (3, hkv), (4, hq)))
    table = rnd((32, hq), 5, torch.float32, dev)
    kw = dict(bias_table=table, buckets=buckets)

    def step(dt, accumulate=False):
        out, lse = ops.packed_attn_fwd(q, k, v, plan, **kw)
        return (out, lse) + ops.packed_attn_bwd(dout, q, k, v, out, lse, plan, dbias_table=dt, accumulate=accumulate, **kw)
    first = torch.empty_like(table)
    want = step(first)
    for _ in range(3):
        again = torch.empty_like(table)
        assert all(torch.equal(a, b) for a, b in zip(want, step(again))) and torch.equal(first, again)
    total = first.clone()
    step(total, accumulate=True)
    assert bool(((total - 2 * first).abs() <= 2 * U * (2 * first).abs()).all())       # one rounding of the sum


@pytest.mark.gpu
def test_a_recording_does_not_see_its_neighbours(dev):
    """The same recording alone and in a pack: the same bits forward."""
    from pseldnets_amd import ops
    lens, hq, hkv, D = [211, 500, 90], 4, 2, 64
    q, k, v = (rnd((sum(lens), h, D), s, torch.bfloat16, dev) for s, h in ((1, hq), (2, hkv), (3, hkv)))
    out, lse = ops.packed_attn_fwd(q, k, v, ops.packed_plan(lens, device=dev), causal=True)
    row = 0
    for n in lens:
        o, l = ops.packed_attn_fwd(q[row:row + n], k[row:row + n], v[row:row + n], ops.packed_plan([n], device=dev), causal=True)
        assert torch.equal(o, out[row:row + n]) and torch.equal(l, lse[row:row + n])
        row += n


@pytest.mark.gpu
def test_stream_steps_in_a_captured_graph(dev):
    """A cache that grows by one frame per replay: k_len is advanced and the new rows written inside the graph, every replay equals the eager call."""
    from pseldnets_amd import ops
    streams, cap, hq, hkv, D = 3, 600, 4, 2, 64
    lens = [5, 511, 0]
    plan = ops.packed_plan([1] * streams, lens, k_cap=cap, device=dev)
    buckets = ops.relpos_buckets(32, 128, False, device=dev)
    table = rnd((32, hq), 9, torch.float32, dev)
    k, v = (rnd((streams * cap, hkv, D), s, torch.bfloat16, dev) for s in (1, 2))
    q, nk, nv = rnd((streams, hq, D), 3, torch.bfloat16, dev), rnd((streams, hkv, D), 4, torch.bfloat16, dev), rnd((streams, hkv, D), 5, torch.bfloat16, dev)
    first = torch.arange(streams, device=dev) * cap

    def step():
        at = first + plan.k_len
        k.index_copy_(0, at, nk)
        v.index_copy_(0, at, nv)
        plan.k_len.add_(1)
        return ops.packed_attn_fwd(q, k, v, plan, causal=True, bias_table=table, buckets=buckets)
    k0, v0 = k.clone(), v.clone()
    step()                                                  # warm up (LDS attributes, allocator)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    k.copy_(k0); v.copy_(v0)
    plan.k_len.copy_(torch.tensor(lens, dtype=torch.int32))
    for t in range(4):
        q.copy_(rnd((streams, hq, D), 30 + t, torch.bfloat16, dev))
        nk.copy_(rnd((streams, hkv, D), 40 + t, torch.bfloat16, dev))
        graph.replay()
        now = [n + t + 1 for n in lens]
        assert plan.k_len.tolist() == now
        eager = ops.packed_attn_fwd(q, k, v, ops.packed_plan([1] * streams, now, k_cap=cap, device=dev), causal=True, bias_table=table, buckets=buckets)
        torch.cuda.synchronize()
        assert torch.equal(held[0], eager[0]) and torch.equal(held[1], eager[1])
    plan.k_len.fill_(10 ** 6)                               # a length past the slab is held to its capacity
    over = ops.packed_attn_fwd(q, k, v, plan, causal=True)
    full = ops.packed_attn_fwd(q, k, v, ops.packed_plan([1] * streams, [cap] * streams, k_cap=cap, device=dev), causal=True)
    assert torch.equal(over[0], full[0])


@pytest.mark.gpu
def test_training_step_in_a_captured_graph_and_on_another_stream(dev):
    from pseldnets_amd import ops
    lens, hq, hkv, D = [130, 70], 4, 1, 64
    plan = ops.packed_plan(lens, device=dev)
    buckets = ops.relpos_buckets(32, 128, True, device=dev)
    table, dt = rnd((32, hq), 9, torch.float32, dev), torch.empty(32, hq, device=dev)
    q, k, v, dout = (rnd((sum(lens), h, D), s, torch.bfloat16, dev) for s, h in ((1, hq), (2, hkv), (3, hkv), (4, hq)))

    def step():
        out, lse = ops.packed_attn_fwd(q, k, v, plan, bias_table=table, buckets=buckets)
        return (out, lse) + ops.packed_attn_bwd(dout, q, k, v, out, lse, plan, bias_table=table, buckets=buckets, dbias_table=dt) + (dt.clone(),)
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
    for t in range(3):
        q.copy_(rnd(q.shape, 20 + t, torch.bfloat16, dev))
        graph.replay()
        torch.cuda.synchronize()
        kept = [x.clone() for x in held]
        eager = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(kept, eager))


@pytest.mark.gpu
def test_decoder_step_of_both_operators(dev):
    """Attention with the bias, then the recurrence over its output, over one plan: a whole pass with its gradients against autograd in 64 bits."""
    from pseldnets_amd import ops
    lens, hq, hkv, D = [37, 64, 1], 4, 2, 32
    N, C = sum(lens), hq * D
    plan = ops.packed_plan(lens, device=dev)
    rel = (16, 40, False)
    buckets = ops.relpos_buckets(*rel, device=dev)
    q, k, v = rnd((N, hq, D), 1, torch.float32, dev), rnd((N, hkv, D), 2, torch.float32, dev), rnd((N, hkv, D), 3, torch.float32, dev)
    table, gate, dh = rnd((16, hq), 4, torch.float32, dev), rnd((N, C), 5, torch.float32, dev), rnd((N, C), 6, torch.float32, dev)
    kw = dict(causal=True, bias_table=table, buckets=buckets)
    out, lse = ops.packed_attn_fwd(q, k, v, plan, **kw)
    h, last, saved = ops.linrec_fwd(gate, out.view(N, C), plan)
    dgate, dn, _ = ops.linrec_bwd(dh, gate, out.view(N, C), saved, plan)
    dt = torch.empty_like(table)
    dq, dk, dv = ops.packed_attn_bwd(dn.view(N, hq, D), q, k, v, out, lse, plan, dbias_table=dt, **kw)
    leaves = [x.double().cpu().requires_grad_(True) for x in (q, k, v, table, gate)]
    Q, K, V, T, Gt = leaves
    row, hs = 0, []
    for n in lens:
        dist = torch.arange(n)[None, :] - torch.arange(n)[:, None]
        w = torch.tensor([[bucket_by_formula(r, *rel) for r in line] for line in dist.tolist()])
        o = []
        for head in range(hq):
            s = D ** -0.5 * Q[row:row + n, head] @ K[row:row + n, head // 2].t() + T[w, head]
            o.append(torch.softmax(s.masked_fill(dist > 0, -math.inf), -1) @ V[row:row + n, head // 2])
        o = torch.stack(o, 1).reshape(n, C)
        state = torch.zeros(C, dtype=torch.float64)
        for t in range(n):
            z = torch.sigmoid(Gt[row + t])
            state = z * state + (1 - z) * o[t]
            hs.append(state)
        row += n
    H = torch.stack(hs)
    (H * dh.double().cpu()).sum().backward()
    # f32 all the way: 64 frames of sums of at most 64 terms of order one, each step's relative error below 64 u, compounded over two operators: 1e-4 of the largest value
    for name, a, b in (('h', h, H.detach()), ('dq', dq, Q.grad), ('dk', dk, K.grad), ('dv', dv, V.grad), ('dtable', dt, T.grad), ('dgate', dgate, Gt.grad)):
        assert (a.double().cpu() - b).abs().max().item() <= 1e-4 * b.abs().max().item(), name


@pytest.mark.gpu
def test_refusals(dev):
    from pseldnets_amd import _lib, ops
    plan = ops.packed_plan([40, 3], device=dev)
    q, k = torch.zeros(43, 4, 64, device=dev), torch.zeros(43, 2, 64, device=dev)
    table, buckets = torch.zeros(32, 4, device=dev), ops.relpos_buckets(device=dev)
    f = ops.packed_attn_fwd
    out, lse = f(q, k, k, plan)
    bad = [lambda: f(q[:42], k, k, plan), lambda: f(q, k[:42], k[:42], plan), lambda: f(q, k, k[:, :1], plan), lambda: f(q, k[:, :, :32], k[:, :, :32], plan),
           lambda: f(q[:, :3].contiguous(), k, k, plan),                                       # 3 query heads, 2 key heads
           lambda: f(q, k.bfloat16(), k.bfloat16(), plan), lambda: f(q.half(), k.half(), k.half(), plan),
           lambda: f(q[:, :, :60].contiguous(), k[:, :, :60].contiguous(), k[:, :, :60].contiguous(), plan),
           lambda: f(torch.zeros(43, 4, 136, device=dev), torch.zeros(43, 2, 136, device=dev), torch.zeros(43, 2, 136, device=dev), plan),
           lambda: f(torch.zeros(43 * 256 + 1, device=dev)[1:].view(43, 4, 64), k, k, plan),   # off its 16-byte boundary
           lambda: f(torch.zeros(43, 4, 66, device=dev)[:, :, :64], k, k, plan),               # heads that are not whole 16-byte pieces apart
           lambda: f(torch.zeros(43, 64, 4, device=dev).transpose(1, 2), k, k, plan), lambda: f(q.cpu(), k.cpu(), k.cpu(), plan),
           lambda: f(q, k, k, plan, scale=0.0), lambda: f(q, k, k, plan, scale=-1.0), lambda: f(q, k, k, plan, scale=float('nan')),
           lambda: f(q, k, k, plan, bias_table=table), lambda: f(q, k, k, plan, buckets=buckets), lambda: f(q, k, k, plan, bias_table=table[:31], buckets=buckets),
           lambda: f(q, k, k, plan, bias_table=table.bfloat16(), buckets=buckets), lambda: f(q, k, k, plan, out=q[:, :2]),
           lambda: ops.packed_attn_bwd(q[:, :2], q, k, k, out, lse, plan), lambda: ops.packed_attn_bwd(q, q, k, k, out, lse[:, :2], plan),
           lambda: ops.packed_attn_bwd(q, q, k, k, out, lse, plan, dbias_table=table), lambda: ops.packed_attn_bwd(q, q, k, k, out, lse.double(), plan),
           lambda: ops.packed_attn_bwd(q, q, k, k, out, lse, plan, dk=k[:, :1])]
    for i, call in enumerate(bad):
        with pytest.raises(_lib.PseldError):
            call()
            print("not refused:", i)


def test_buckets_follow_the_formula():
    """Host side: every distance's bucket, at and around the borders, and past the last."""
    from pseldnets_amd import _lib, ops
    for n, m, both in ((32, 128, True), (32, 128, False), (16, 50, True), (64, 333, False), (320, 800, False), (512, 1024, True), (4, 2, True), (2, 9, False)):
        b = ops.RelposBuckets(n, m, both, 'cpu')
        assert len(b.host_lut) == 2 * m + 1
        assert b.host_lut == [bucket_by_formula(r, n, m, both) for r in range(-m, m + 1)]
        assert bucket_by_formula(-m - 5000, n, m, both) == b.host_lut[0] and bucket_by_formula(m + 5000, n, m, both) == b.host_lut[-1]
        assert 0 <= min(b.host_lut) and max(b.host_lut) < n
    for bad in ((1, 128, False), (33, 128, True), (514, 1024, True), (32, 8, True), (32, 1025, False), (2, 9, True)):
        with pytest.raises(_lib.PseldError):
            ops.RelposBuckets(*bad, 'cpu')


def test_c_entry_refuses_without_a_launch():
    """Argument checks come before anything touches a device: callable here without one."""
    import ctypes
    import os
    from pseldnets_amd import _lib
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip("libpseld_hip.so not built")
    L = _lib.lib()
    A = 4096                                                 # an address that is never followed
    plan = (ctypes.c_long * 18)(1, 40, 40, 40, 40, 1, 1, 1, 1, *[A] * 9)
    st = (ctypes.c_long * 16)(*[256, 64] * 8)

    def fwd(dtype=0, q=A, k=A, st=st, plan=plan, hq=4, hkv=4, D=64, scale=1.0, table=None, lut=None, nb=0, md=0):
        return L.pseld_packed_attn_fwd(dtype, q, k, A, A, A, st, plan, hq, hkv, D, 0, scale, table, lut, nb, md, None, 0, None)
    odd = (ctypes.c_long * 16)(*[257, 64] * 8)
    far = (ctypes.c_long * 16)(*[1 << 24, 64] * 8)
    few = (ctypes.c_long * 18)(1, 1, 1, 100000, 100000, 1, 782, 782, 782, *[A] * 9)
    for bad in (dict(dtype=3), dict(q=None), dict(k=None), dict(q=A + 8), dict(st=odd), dict(st=far), dict(st=None), dict(plan=None), dict(hq=5, hkv=2), dict(hkv=0),
                dict(D=60), dict(D=136), dict(D=0), dict(scale=0.0), dict(scale=float('inf')), dict(table=A), dict(table=A, lut=A, nb=513, md=128),
                dict(table=A, lut=A, nb=32, md=1025), dict(plan=few)):
        assert fwd(**bad) == -1, bad
    assert b"workspace" in L.pseld_last_error()
    assert L.pseld_packed_attn_bwd(0, A, A, A, A, A, A, A, A, A, st, plan, 4, 4, 64, 0, 1.0, None, None, 0, 0, A, 0, A, 1 << 30, None) == -1
    assert L.pseld_packed_attn_bwd(0, A, A, A, A, A, A, A, A, A, st, plan, 4, 4, 64, 0, 1.0, None, None, 0, 0, None, 0, A, 16, None) == -1


def test_c_entry_refuses_overlapping_results_and_too_many_rows():
    import ctypes
    import os
    from pseldnets_amd import _lib
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip("libpseld_hip.so not built")
    L = _lib.lib()
    A = [4096 * i for i in range(1, 12)]                     # addresses that are never followed

    def plan(rows=40, k_rows=40):
        return (ctypes.c_long * 18)(1, rows, min(rows, 40), k_rows, min(k_rows, 40), 1, 1, 1, 1, *[4096] * 9)

    def fwd(out=A[3], so=(256, 64), p=plan()):
        return L.pseld_packed_attn_fwd(0, A[0], A[1], A[2], out, A[9], (ctypes.c_long * 8)(*[256, 64] * 3, *so), p, 4, 4, 64, 0, 1.0, None, None, 0, 0, None, 0, None)

    def bwd(dq=A[5], dk=A[6], dv=A[7], sdq=(256, 64), sdk=(256, 64)):
        return L.pseld_packed_attn_bwd(0, A[4], A[0], A[1], A[2], A[3], A[9], dq, dk, dv, (ctypes.c_long * 16)(*[256, 64] * 5, *sdq, *sdk, 256, 64), plan(), 4, 4, 64,
                                       0, 1.0, None, None, 0, 0, None, 0, A[10], 1 << 30, None)
    for bad in (dict(out=A[0]), dict(out=A[1]), dict(out=A[2]), dict(so=(0, 64)), dict(so=(192, 64)), dict(so=(256, 0)), dict(so=(64, 64)), dict(so=(64, 2496)),
                dict(p=plan(rows=(1 << 30) + 1)), dict(p=plan(k_rows=(1 << 30) + 1))):
        assert fwd(**bad) == -1, bad
    for bad in (dict(dq=A[0]), dict(dk=A[1]), dict(dv=A[2]), dict(dq=A[4]), dict(dq=A[3]), dict(dk=A[5]), dict(dv=A[6]), dict(dv=A[5]), dict(sdq=(0, 64)), dict(sdk=(128, 32))):
        assert bwd(**bad) == -1, bad


def test_chunks_of_the_longest_caches_stay_joinable():
    """The joining launch keeps one weight per chunk of a recording's keys in LDS: 64 KB at most."""
    import ctypes
    import os
    from pseldnets_amd import _lib
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip("libpseld_hip.so not built")
    for keys in (1000, 100_000, 131_072, 50_000_000, 400_000_000, 1 << 30):
        for hkv in (1, 16):
            plan = (ctypes.c_long * 18)(1, 1, 1, keys, keys, 1, (keys + 127) // 128, 1, 1, *[4096] * 9)
            chunks = _lib.lib().pseld_packed_attn_fwd_workspace(plan, hkv, hkv, 64, 0) // (hkv * 68 * 4)
            assert 1 <= chunks <= 16384


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("q_lens,k_lens,row", [([70, 200], None, 130), ([1, 1, 1], [9, 600, 300], 1), ([1, 1], [4000, 90], 0)])
def test_a_nan_query_shows_in_its_own_row_alone(dev, dtype, q_lens, k_lens, row):
    """Whole recordings, few rows in one chunk and in many: out, lse and dq of the (row, head) are NaN, every other row's are not."""
    from pseldnets_amd import ops
    plan = ops.packed_plan(q_lens, k_lens, device=dev)
    q, dout = rnd((plan.rows, 4, 64), 1, dtype, dev), rnd((plan.rows, 4, 64), 2, dtype, dev)
    k, v = rnd((plan.k_rows, 2, 64), 3, dtype, dev), rnd((plan.k_rows, 2, 64), 4, dtype, dev)
    q[row, 1, 5] = float('nan')
    out, lse = ops.packed_attn_fwd(q, k, v, plan, causal=True)
    dq, _, _ = ops.packed_attn_bwd(dout, q, k, v, out, lse, plan, causal=True)
    want = torch.zeros(plan.rows, 4, dtype=torch.bool, device=dev)
    want[row, 1] = True
    assert torch.equal(torch.isnan(lse), want) and not torch.isinf(lse).any()
    for t in (out, dq):
        assert torch.equal(torch.isnan(t).all(-1), want) and torch.equal(torch.isnan(t).any(-1), want)


def _plan_array(q, cap):
    """The host array of a plan with these lengths (addresses that are never followed), and its key lists."""
    import ctypes
    import numpy as np
    from pseldnets_amd import ops
    (qf, _), keys, work = ops._packed_work(np.array(q), np.array(cap))
    return (ctypes.c_long * 18)(len(q), sum(q), max(q), sum(cap), max(cap), len(qf), len(keys[0]), *work, *[4096] * 9), keys, work


def test_backward_workspace_follows_the_work():
    """Packs of long and short recordings: what the parts of dk and dv take is bounded by the number of parts that the work is cut into (at most 700, twice that
    with the tiles' ends), 128 x 2 x 128 floats each, whatever the longest recording times the number of tiles would be. It was 1.7 and 3.3 GB."""
    import os
    from pseldnets_amd import _lib
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip("libpseld_hip.so not built")
    for q, hq, hkv in (([6000] + [500] * 60, 8, 1), ([12000] + [2000] * 100, 16, 2), ([8191], 16, 2), ([1] * 1000 + [30000], 4, 4)):
        plan, _, _ = _plan_array(q, q)
        for dtype, parts in ((0, 700), (1, 400)):
            for causal in (0, 1):
                size = _lib.lib().pseld_packed_attn_bwd_workspace(dtype, plan, hq, hkv, 128, causal, 0)
                assert size <= 2 * parts * 2 * 128 * 128 * 4 + 4 * sum(q) * hq + 64, (q[0], dtype, causal)


def test_parts_of_dk_and_dv_have_places_of_their_own():
    """What the dk/dv kernel writes and its joining launch reads, computed here from the lists: over every kind of pack, and with caches that are shorter than their
    capacity when the call is made, the places of two key tiles' parts never meet and all lie inside the workspace."""
    import os
    import random
    from pseldnets_amd import _lib
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip("libpseld_hip.so not built")
    rng, cut = random.Random(3), 0
    for case_ in range(150):
        n = rng.randint(1, 12)
        q = [rng.choice([0, 1, rng.randint(0, 500), rng.randint(0, 9000)]) for _ in range(n)]
        cap = list(q) if case_ % 3 == 0 else [max(0, x + rng.randint(-300, 900)) if rng.random() < 0.7 else rng.randint(0, 9000) for x in q]
        hkv = rng.choice([1, 2, 4])
        G = rng.choice([1, 2, 8])
        D = rng.choice([32, 64, 128])
        pad = 32 if D <= 32 else 64 if D <= 64 else 128
        plan, keys, work = _plan_array(q, cap)
        for causal in (0, 1):
            for dtype in (0, 1):
                parts, least = (700, 1) if dtype == 0 else (400 if D > 64 else 600, 4)
                steps = work[causal] * hkv * G
                chunk = max(least, min(1 << 20, -(-steps // parts)))
                longest = -(-max(q) // 64) * G
                most = -(-longest // chunk) if longest > chunk else 1
                size = _lib.lib().pseld_packed_attn_bwd_workspace(dtype, plan, hkv * G, hkv, D, causal, 0) - 4 * ((sum(q) * hkv * G + 3) // 4 * 4) - 16
                assert size % (hkv * 2 * 128 * pad * 4) == 0
                slots = size // (hkv * 2 * 128 * pad * 4)
                for k_len in (cap, [rng.randint(0, c) for c in cap]):
                    end = 0
                    for t, (s, first, _, q_len, _, k_cap, low, high) in enumerate(keys[causal].tolist()):
                        start = q_len if first >= k_len[s] else max(0, first - (k_len[s] - q_len)) // 64 * 64 if causal else 0
                        total = (-(-(q_len - start) // 64) if start < q_len else 0) * G
                        ns = max(1, min(most, -(-total // chunk)))
                        if ns == 1:
                            continue
                        cut += 1
                        place = (low + (high << 32)) * G // chunk + t
                        assert place >= end and place + ns <= slots
                        end = place + ns
    assert cut > 1000


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("D", [64, 128])
def test_a_long_recording_among_short_ones(dev, dtype, D):
    """Some key tiles are cut into many parts, some into a few, most into none."""
    lens = [40, 1500, 7, 300, 130, 1, 0, 65, 129] + [50] * 6
    case(dev, dtype, lens, 4, 1, D, True)
    case(dev, dtype, lens, 4, 2, D, False, bias=(32, 128, True))
    case(dev, dtype, [700, 3, 90, 0], 4, 1, D, True, bias=(16, 50, False), k_lens=[1100, 64, 0, 12], cap=[1400, 64, 300, 700])


def test_chunks_of_unequal_caches_have_places_of_their_own():
    """Few rows over caches of different capacities: what the chunks take follows the rows of all caches together (it was the longest cache's chunks for every
    recording, more than the caches themselves: 448 MB beside 257), and no two recordings' chunks meet, with empty caches among them and behind."""
    import os
    import random
    from pseldnets_amd import _lib
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip("libpseld_hip.so not built")
    size = _lib.lib().pseld_packed_attn_fwd_workspace
    for caps, q, hq, hkv, D, most in (([131072] + [600] * 200, 8, 16, 4, 64, 12e6), ([1 << 20] + [512] * 999, 1, 32, 8, 128, 21e6)):
        assert size(_plan_array([q] * len(caps), caps)[0], hq, hkv, D, 0) <= most
    rng, cut = random.Random(5), 0
    for _ in range(200):
        n, hkv, D = rng.randint(1, 20), rng.choice([1, 2, 8]), rng.choice([8, 64, 128])
        caps = [rng.choice([0, 1, 256 * rng.randint(0, 40), rng.randint(0, 30000)]) for _ in range(n)]
        total = sum(caps)
        need = size(_plan_array([1] * n, caps)[0], hkv, hkv, D, 0)
        chunk = 512 if max(caps) <= 512 else max(256, min(8192, -(-((total * hkv + 511) // 512) // 128) * 128))      # keys per chunk
        if max(caps) <= chunk:
            assert need == 0
            continue
        slots, rest = divmod(need, hkv * (D + 4) * 4)
        assert rest == 0
        first, end = 0, 0
        for s, cap in enumerate(caps):
            place = first // chunk + s
            assert place >= end
            end = place + max(1, -(-cap // chunk))
            assert end <= slots
            first += cap
            cut += cap > chunk
    assert cut > 300


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DT)
def test_few_rows_over_unequal_caches(dev, dtype):
    """Recordings cut into many chunks beside empty ones, an empty one last behind whole chunks."""
    case(dev, dtype, [1, 2, 1, 3], 8, 2, 64, True, bias=(32, 128, False), k_lens=[5000, 0, 700, 0], cap=[5120, 0, 768, 0], backward=False)
    case(dev, dtype, [1, 1, 0, 1, 1], 4, 4, 128, False, k_lens=[1, 3000, 40, 0, 513], cap=[300, 3333, 600, 0, 600], backward=False)


def test_c_entry_refuses_a_workspace_off_its_boundary():
    """Both directions read their workspaces in 16-byte pieces."""
    import ctypes
    import os
    from pseldnets_amd import _lib
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip("libpseld_hip.so not built")
    L = _lib.lib()
    A = [4096 * i for i in range(1, 12)]                     # addresses that are never followed
    plan, st = _plan_array([1], [100000])[0], (ctypes.c_long * 16)(*[256, 64] * 8)
    assert L.pseld_packed_attn_fwd_workspace(plan, 4, 4, 64, 0) > 0
    for off in (4, 8):
        assert L.pseld_packed_attn_fwd(0, A[0], A[1], A[2], A[3], A[9], st, plan, 4, 4, 64, 0, 1.0, None, None, 0, 0, A[10] + off, 1 << 40, None) == -1
        assert b"boundary" in L.pseld_last_error()
        assert L.pseld_packed_attn_bwd(0, A[4], A[0], A[1], A[2], A[3], A[9], A[5], A[6], A[7], st, plan, 4, 4, 64, 0, 1.0, None, None, 0, 0, None, 0,
                                       A[10] + off, 1 << 40, None) == -1
        assert b"boundary" in L.pseld_last_error()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("q_lens,k_lens", [([70, 1, 130], None), ([2, 1, 1], [600, 9, 1300])])
def test_head_major_operands_and_results_of_the_caller(dev, dtype, q_lens, k_lens):
    """Heads outside rows, for operands and for every result that a caller may pass (out=, dq=, dk=, dv=); whole recordings and few rows."""
    from pseldnets_amd import ops
    hq, hkv, D = 4, 2, 64
    plan = ops.packed_plan(q_lens, k_lens, device=dev)
    heads_out = lambda rows, heads, seed: rnd((heads, rows, D), seed, dtype, dev).transpose(0, 1)      # noqa: E731
    q, k, v, dout = heads_out(plan.rows, hq, 1), heads_out(plan.k_rows, hkv, 2), heads_out(plan.k_rows, hkv, 3), heads_out(plan.rows, hq, 4)
    kept, dq, dk, dv = (torch.full_like(t, float('nan')) for t in (q, q, k, v))
    assert kept.stride() == (D, plan.rows * D, 1)
    out, lse = ops.packed_attn_fwd(q, k, v, plan, causal=True, out=kept)
    grads = ops.packed_attn_bwd(dout, q, k, v, out, lse, plan, causal=True, dq=dq, dk=dk, dv=dv)
    assert out is kept and all(a is b for a, b in zip(grads, (dq, dk, dv)))
    kl = k_lens if k_lens is not None else q_lens
    want = reference(q, k, v, dout, q_lens, kl, starts_of(kl), True, D ** -0.5)
    compare(dict(out=out, lse=lse, dq=dq, dk=dk, dv=dv), want)
    rows_out = torch.full((plan.rows, 3, hq, D), float('nan'), dtype=dtype, device=dev)      # heads inside rows, rows apart
    again, lse2 = ops.packed_attn_fwd(q.contiguous(), k.contiguous(), v.contiguous(), plan, causal=True, out=rows_out[:, 1])
    assert torch.equal(again, out) and torch.equal(lse2, lse) and bool(torch.isnan(rows_out[:, 0::2]).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DT)
def test_one_frame_of_heads_or_buckets_past_the_few_rows_kernel(dev, dtype):
    """More than 32 query heads a key head, more table entries than the few-rows kernel holds: the query-tiled kernel answers for single frames too."""
    case(dev, dtype, [1, 3, 1], 64, 1, 64, True, k_lens=[300, 40, 0], cap=320)
    case(dev, dtype, [1, 1], 40, 1, 32, False, bias=(32, 128, True), k_lens=[900, 33], cap=1000, backward=False)
    case(dev, dtype, [1, 1], 16, 1, 64, True, bias=(320, 800, False), k_lens=[900, 33], cap=1000, backward=False)
