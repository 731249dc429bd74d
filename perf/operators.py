"""Measurement cases of the sequence operators: attention over packed recordings (whole recordings, training, one frame of a running
stream), its learned relative position bias by buckets, and the gated linear recurrence.

Each case is one call a program makes: a forward pass over recordings of different lengths, a training step's forward and backward
pass, or the next frame of streams that run in parallel. `run` computes it either in plain torch (32 bits, elementary operations,
recordings padded to a rectangle) or, with `own` set, through pseldnets_amd.ops.
"""
import math
import random

import numpy as np
import torch

own = False

_DT = {"bf16": torch.bfloat16, "f32": torch.float32}


# ---- cases -------------------------------------------------------------------------------------------------------------------------
def _attn(name, kind, dtype, seqs, lo, hi, hq, hkv, d, causal, buckets=0, max_distance=0, cap=0, lens_seed=1):
    return dict(name=name, kind=kind, dtype=dtype, seqs=seqs, len_lo=lo, len_hi=hi, hq=hq, hkv=hkv, d=d, causal=causal,
                buckets=buckets, max_distance=max_distance, cap=cap, lens_seed=lens_seed)


def _rec(name, kind, dtype, seqs, lo, hi, c, reverse=False, lens_seed=1):
    return dict(name=name, kind=kind, dtype=dtype, seqs=seqs, len_lo=lo, len_hi=hi, c=c, reverse=reverse, lens_seed=lens_seed)


def listed():
    return [
        # the next frame of one live stream a few seconds after its start: nothing but latency
        _attn("attn_step_one", "attn_step", "bf16", 1, 37, 37, 8, 2, 64, True, 32, 128, cap=256),
        # 48 live microphones whose caches hold between some seconds and some minutes
        _attn("attn_step_streams", "attn_step", "bf16", 48, 100, 4096, 16, 2, 128, True, cap=4096),
        # three day-long monitoring streams: long caches, few rows
        _attn("attn_step_long", "attn_step", "bf16", 3, 60001, 131072, 16, 4, 64, True, 32, 128, cap=131072),
        # validation in the f32 parity mode: a few short recordings, both directions
        _attn("attn_fwd_short_f32", "attn_fwd", "f32", 4, 25, 125, 8, 8, 32, False, 32, 128),
        # inference over a pack of recordings of all lengths with a wide learned bias
        _attn("attn_fwd_packed", "attn_fwd", "bf16", 24, 57, 1999, 16, 4, 64, True, 320, 800),
        # one 20-minute recording at 10 frames a second, causal
        _attn("attn_fwd_long", "attn_fwd", "bf16", 1, 12289, 12289, 16, 2, 128, True),
        # a training step of the causal decoder on recordings of different lengths
        _attn("attn_train_packed", "attn_train", "bf16", 12, 100, 1200, 16, 4, 64, True, 32, 128),
        # a training step on one long recording with strongly grouped heads
        _attn("attn_train_long", "attn_train", "bf16", 1, 8191, 8191, 16, 2, 128, True),
        # a training step in the f32 parity mode, both directions
        _attn("attn_train_f32", "attn_train", "f32", 6, 30, 600, 8, 8, 64, False, 32, 128),
        # the recurrence's next frame of 32 live streams
        _rec("rec_step", "rec_step", "bf16", 32, 1, 1, 512),
        # a training batch of recordings
        _rec("rec_train_batch", "rec_train", "bf16", 32, 200, 1000, 1024),
        # two long recordings, backwards in time, in the f32 parity mode
        _rec("rec_train_long_f32", "rec_train", "f32", 2, 50001, 60000, 512, reverse=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["attn_step", "attn_step", "attn_fwd", "attn_fwd", "attn_train", "attn_train", "rec_step", "rec_train", "rec_train"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    lens_seed = rng.randrange(1 << 20)
    if kind.startswith("rec"):
        c = 8 * _log_int(rng, 4, 256)
        if kind == "rec_step":
            return _rec(None, kind, dtype, _log_int(rng, 1, 256), 1, 1, c, rng.random() < 0.3, lens_seed) | {"name": ""}
        seqs = _log_int(rng, 1, 64)
        hi = min(_log_int(rng, 2, 60000), max(2, 60_000_000 // (c * seqs)))
        return _rec(None, kind, dtype, seqs, rng.choice([0, 1, max(1, hi // 3), hi]), hi, c, rng.random() < 0.5, lens_seed) | {"name": ""}
    hkv = rng.choice([1, 2, 3, 4, 8])
    hq = hkv * rng.choice([g for g in (1, 2, 3, 4, 8) if hkv * g <= 16])
    d = rng.choice([32, 64, 128, 24, 40, 96])
    causal = rng.random() < 0.6
    buckets, max_distance = rng.choice([(0, 0), (32, 128), (16, 50), (64, 333), (320, 800)])
    if kind == "attn_step":
        cap = _log_int(rng, 16, 131072)
        seqs = max(1, min(_log_int(rng, 1, 128), 300_000 // cap))
        return _attn(None, kind, dtype, seqs, rng.choice([0, 1, max(1, cap // 5), cap]), cap, hq, hkv, d, True, buckets, max_distance, cap, lens_seed) | {"name": ""}
    most = 60_000_000 if kind == "attn_fwd" else 16_000_000         # pairs of the padded rectangle
    if dtype == "f32" or (kind == "attn_train" and buckets == 320):
        most //= 4
    seqs = _log_int(rng, 1, 32)
    hi = min(_log_int(rng, 8, 6000), int(math.sqrt(most / seqs)))
    return _attn(None, kind, dtype, seqs, rng.choice([0, 1, max(1, hi // 4), hi]), hi, hq, hkv, d, causal, buckets, max_distance, 0, lens_seed) | {"name": ""}


def _lens(case):
    r = random.Random(case["lens_seed"])
    got = [r.randint(case["len_lo"], case["len_hi"]) for _ in range(case["seqs"])]
    got[0] = case["len_hi"]
    return got


def _pairs(case):
    """(query, key) pairs that the mask leaves, summed over the recordings."""
    if case["kind"] == "attn_step":
        return sum(_lens(case))
    return sum(n * (n + 1) // 2 if case["causal"] else n * n for n in _lens(case))


def work(case):
    e = 2 if case["dtype"] == "bf16" else 4
    lens = _lens(case)
    n = sum(lens)
    if case["kind"].startswith("rec"):
        c, state = case["c"], 4 * case["seqs"] * case["c"]
        if case["kind"] == "rec_train":      # gates, candidates and the output's gradient in; states and two gradients out; h0, h_last and their gradients
            return {"bytes": 6 * n * c * e + 4 * state, "flops": 20 * n * c}
        return {"bytes": 3 * n * c * e + 2 * state, "flops": 8 * n * c}
    nq = case["seqs"] if case["kind"] == "attn_step" else n
    q, kv = nq * case["hq"] * case["d"] * e, n * case["hkv"] * case["d"] * e
    table = 4 * case["buckets"] * case["hq"]
    flops = 4 * case["d"] * _pairs(case) * case["hq"]
    if case["kind"] == "attn_train":         # + the gradients of the output in, of queries, keys, values and the table out; five products more
        return {"bytes": 4 * q + 4 * kv + 2 * table, "flops": 7 * flops // 2}
    return {"bytes": 2 * q + 2 * kv + table + 4 * nq * case["hq"], "flops": flops}


# ---- the relative position's bucket ------------------------------------------------------------------------------------------------
def _thresholds(n_side, max_distance):
    """Distances at which the next bucket of one side begins: n_side/2 buckets of one distance each, then logarithmic ones up to
    max_distance. Exact: distance n is in log bucket k or above where (n / e)^K >= (max_distance / e)^k."""
    e = n_side // 2
    k_all = n_side - e
    starts = list(range(1, e + 1))
    n = e
    for k in range(1, k_all):
        while n ** k_all * e ** k < max_distance ** k * e ** k_all:
            n += 1
        starts.append(n)
    return starts


def _bucket(rel, starts, buckets, causal):
    """Bucket of key position - query position (an integer tensor): the number of thresholds at or below the distance."""
    n_side = buckets if causal else buckets // 2
    dist = torch.clamp(-rel, min=0) if causal else rel.abs()
    b = torch.bucketize(dist, starts, right=True)
    return b if causal else b + n_side * (rel > 0)


# ---- inputs ------------------------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    dev = torch.device("cuda:0")
    g = torch.Generator(device=dev).manual_seed(seed * 7919 + 13)
    dt = _DT[case["dtype"]]
    lens = _lens(case)
    n = sum(lens)

    def randn(*shape, dtype=dt, scale=1.0, shift=0.0):
        return (torch.randn(*shape, generator=g, device=dev) * scale + shift).to(dtype)

    s = {"case": dict(case)}
    if case["kind"].startswith("rec"):
        c = case["c"]
        s["gates"] = randn(n, 2 * c)                         # one projection's output: update gates | candidates
        s["gates"][:, :c] += 2.0                             # gates that keep most of the state
        s["h0"] = randn(case["seqs"], c, dtype=torch.float32)
        if case["kind"] == "rec_train":
            s["dh"] = randn(n, c)
            s["dlast"] = randn(case["seqs"], c, dtype=torch.float32)
        q_lens, k_lens, cap = lens, None, None
    else:
        hq, hkv, d = case["hq"], case["hkv"], case["d"]
        if case["buckets"]:
            s["table"] = randn(case["buckets"], hq, dtype=torch.float32, scale=0.7)
        if case["kind"] == "attn_step":
            q_lens, k_lens, cap = [1] * case["seqs"], lens, case["cap"]
            s["q"] = randn(case["seqs"], hq, d)
            s["k"] = randn(case["seqs"], cap, hkv, d)        # caches; rows past a stream's length hold what was there before
            s["v"] = randn(case["seqs"], cap, hkv, d)
        else:
            q_lens, k_lens, cap = lens, None, None
            s["qkv"] = randn(n, (hq + 2 * hkv) * d)          # one projection's output: queries | keys | values
            if case["kind"] == "attn_train":
                s["dout"] = randn(n, hq, d)
    if own:
        from pseldnets_amd import ops
        s["plan"] = ops.packed_plan(q_lens, k_lens, k_cap=cap, device=dev)
        if case.get("buckets"):
            s["buckets"] = ops.relpos_buckets(case["buckets"], case["max_distance"], bidirectional=not case["causal"], device=dev)
        return s
    # plain form: recordings padded to a rectangle; row of (recording, position), and which positions exist
    mq = max(1, max(q_lens))
    ql = torch.tensor(q_lens, device=dev)
    starts = torch.cumsum(ql, 0) - ql
    t = torch.arange(mq, device=dev)
    s["q_live"] = t[None, :] < ql[:, None]
    at = (ql[:, None] - 1 - t[None, :]) if case.get("reverse") else t[None, :].expand(len(q_lens), mq)
    s["q_rows"] = torch.where(s["q_live"], starts[:, None] + at, 0)
    s["q_lens"] = ql
    if case.get("buckets"):
        s["starts"] = torch.tensor(_thresholds(case["buckets"] // (1 if case["causal"] else 2), case["max_distance"]), device=dev)
    s["k_lens"] = torch.tensor(k_lens, device=dev) if k_lens is not None else ql
    return s


# ---- plain forms -------------------------------------------------------------------------------------------------------------------
def _pad(x, s):
    """Packed rows [N, ...] -> [recordings, longest, ...] in 32 bits, zeros past the end."""
    live = s["q_live"].reshape(*s["q_live"].shape, *([1] * (x.dim() - 1)))
    if not x.shape[0]:
        return torch.zeros(*s["q_live"].shape, *x.shape[1:], device=x.device)
    return torch.where(live, x[s["q_rows"]].float(), 0.0)


def _unpad(x, s, dtype):
    """The inverse of _pad, rounded once."""
    out = torch.empty(int(s["n"]), *x.shape[2:], dtype=dtype, device=x.device)
    out[s["q_rows"][s["q_live"]]] = x[s["q_live"]].to(dtype)
    return out


def _plain_scores(q, k, s):
    """Probabilities [B, Hkv, G, Mq, Mk] and their log-sum-exp; q [B, Mq, Hq, D], k [B, Mk, Hkv, D] in 32 bits."""
    case = s["case"]
    B, mq, hq, d = q.shape
    mk, hkv = k.shape[1], k.shape[2]
    grp = hq // hkv
    qh = q.reshape(B, mq, hkv, grp, d).permute(0, 2, 3, 1, 4).reshape(B, hkv, grp * mq, d).contiguous()
    kh = k.permute(0, 2, 3, 1).contiguous()                                        # [B, Hkv, D, Mk]
    sc = torch.matmul(qh, kh).reshape(B, hkv, grp, mq, mk) * (1.0 / math.sqrt(d))
    kpos = torch.arange(mk, device=q.device)
    qpos = torch.arange(mq, device=q.device)[None, :] + (s["k_lens"] - s["q_lens"])[:, None]      # [B, Mq]
    rel = kpos[None, None, :] - qpos[:, :, None]
    live = (kpos[None, None, :] < s["k_lens"][:, None, None]) & s["q_live"][:, :, None]
    if case["causal"]:
        live = live & (rel <= 0)
    bucket = None
    if case["buckets"]:
        bucket = _bucket(rel, s["starts"], case["buckets"], case["causal"])
        sc = sc + s["table"][bucket].reshape(B, mq, mk, hkv, grp).permute(0, 3, 4, 1, 2)
    sc = sc.masked_fill(~live[:, None, None], -math.inf)
    mx = sc.amax(-1, keepdim=True)
    mx = torch.where(torch.isinf(mx), 0.0, mx)
    p = torch.exp(sc - mx)
    total = p.sum(-1, keepdim=True)
    lse = (mx + torch.log(total)).squeeze(-1)
    p = torch.where(total > 0, p / total, 0.0)
    return p, lse, bucket


def _heads_out(x):
    """[B, Hkv, G, Mq, D] -> [B, Mq, Hq, D]"""
    B, hkv, grp, mq, d = x.shape
    return x.permute(0, 3, 1, 2, 4).reshape(B, mq, hkv * grp, d)


def _plain_attn(s):
    case = s["case"]
    dt = _DT[case["dtype"]]
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    grp = hq // hkv
    if case["kind"] == "attn_step":
        s["n"] = case["seqs"]
        q = s["q"].float()[:, None]
        past = torch.arange(case["cap"], device=q.device)[None, :, None, None] >= s["k_lens"][:, None, None, None]
        k, v = (x.float().masked_fill(past, 0.0) for x in (s["k"], s["v"]))
    else:
        n = s["n"] = s["qkv"].shape[0]
        q, k, v = (_pad(x, s) for x in (s["qkv"][:, :hq * d].reshape(n, hq, d), s["qkv"][:, hq * d:(hq + hkv) * d].reshape(n, hkv, d),
                                        s["qkv"][:, (hq + hkv) * d:].reshape(n, hkv, d)))
    B, mq, mk = q.shape[0], q.shape[1], k.shape[1]
    p, lse, bucket = _plain_scores(q, k, s)
    vh = v.permute(0, 2, 1, 3).contiguous()                                        # [B, Hkv, Mk, D]
    o = torch.matmul(p.reshape(B, hkv, grp * mq, mk), vh).reshape(B, hkv, grp, mq, d)
    out = _unpad(_heads_out(o), s, dt)
    if case["kind"] != "attn_train":
        return out, _unpad(lse.permute(0, 3, 1, 2).reshape(B, mq, hq), s, torch.float32)
    do = _pad(s["dout"], s).reshape(B, mq, hkv, grp, d).permute(0, 2, 3, 1, 4)     # [B, Hkv, G, Mq, D]
    dor = do.reshape(B, hkv, grp * mq, d).contiguous()
    pr = p.reshape(B, hkv, grp * mq, mk)
    dv = torch.matmul(pr.transpose(2, 3).contiguous(), dor)
    dp = torch.matmul(dor, vh.transpose(2, 3).contiguous()).reshape(p.shape)
    ds = p * (dp - (p * dp).sum(-1, keepdim=True))
    scale = 1.0 / math.sqrt(d)
    dsr = ds.reshape(B, hkv, grp * mq, mk)
    qr = q.reshape(B, mq, hkv, grp, d).permute(0, 2, 3, 1, 4).reshape(B, hkv, grp * mq, d).contiguous()
    kr = k.permute(0, 2, 1, 3).contiguous()
    dq = torch.matmul(dsr, kr).reshape(B, hkv, grp, mq, d) * scale
    dk = torch.matmul(dsr.transpose(2, 3).contiguous(), qr) * scale
    res = [out, _unpad(_heads_out(dq), s, dt), _unpad(dk.permute(0, 2, 1, 3), s, dt), _unpad(dv.permute(0, 2, 1, 3), s, dt)]
    if case["buckets"]:                                      # long sums that nearly cancel: in 64 bits
        which = (bucket.reshape(B * mq, 1, mk) == torch.arange(case["buckets"], device=q.device)[:, None]).double()
        res.append(torch.matmul(which, ds.permute(0, 3, 4, 1, 2).reshape(B * mq, mk, hq).double()).sum(0).float())
    return tuple(res)


def _scan(a, b):
    """h[:, t] = a[:, t] h[:, t - 1] + b[:, t] from h = 0, by doubling the distance that a step spans."""
    d = 1
    while d < a.shape[1]:
        b = torch.cat((b[:, :d], b[:, d:] + a[:, d:] * b[:, :-d]), 1)
        a = torch.cat((a[:, :d], a[:, d:] * a[:, :-d]), 1)
        d *= 2
    return b


def _plain_rec(s):
    case = s["case"]
    dt, c = _DT[case["dtype"]], case["c"]
    s["n"] = s["gates"].shape[0]
    gate, cand = _pad(s["gates"][:, :c], s), _pad(s["gates"][:, c:], s)
    z, y = torch.sigmoid(gate), torch.sigmoid(-gate)         # y = 1 - z without the cancellation
    b = y * cand
    b[:, 0] += z[:, 0] * s["h0"]
    h = _scan(z, b)
    some = (s["q_lens"] > 0)[:, None]
    end = torch.clamp(s["q_lens"] - 1, min=0)[:, None, None].expand(-1, 1, c)
    last = torch.where(some, h.gather(1, end)[:, 0], s["h0"])
    out = _unpad(h, s, dt)
    if case["kind"] != "rec_train":
        return out, last
    dh = _pad(s["dh"], s).scatter_add(1, end, torch.where(some, s["dlast"], 0.0)[:, None])
    nxt = torch.cat((z[:, 1:], torch.zeros_like(z[:, :1])), 1)
    nxt = torch.where(torch.cat((s["q_live"][:, 1:], torch.zeros_like(s["q_live"][:, :1])), 1)[:, :, None], nxt, 0.0)
    lam = _scan(nxt.flip(1), dh.flip(1)).flip(1)
    prev = torch.cat((s["h0"][:, None], h[:, :-1]), 1)
    dgate = lam * (prev - cand) * z * y
    dh0 = torch.where(some, z[:, 0] * lam[:, 0], s["dlast"])
    return out, last, _unpad(dgate, s, dt), _unpad(lam * y, s, dt), dh0


# ---- one pass ----------------------------------------------------------------------------------------------------------------------
def run(s):
    if not own:
        return _plain_rec(s) if s["case"]["kind"].startswith("rec") else _plain_attn(s)
    from pseldnets_amd import ops
    case, plan = s["case"], s["plan"]
    if case["kind"].startswith("rec"):
        c = case["c"]
        gate, cand = s["gates"][:, :c], s["gates"][:, c:]
        h, last, saved = ops.linrec_fwd(gate, cand, plan, h0=s["h0"], reverse=case["reverse"], need_saved=case["kind"] == "rec_train")
        if case["kind"] != "rec_train":
            return h, last
        dgate, dcand, dh0 = ops.linrec_bwd(s["dh"], gate, cand, saved, plan, dh_last=s["dlast"], h0=s["h0"], reverse=case["reverse"])
        return h, last, dgate, dcand, dh0
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    bias = dict(bias_table=s["table"], buckets=s["buckets"]) if case["buckets"] else {}
    if case["kind"] == "attn_step":
        return ops.packed_attn_fwd(s["q"], s["k"].view(-1, hkv, d), s["v"].view(-1, hkv, d), plan, causal=True, **bias)
    n = s["qkv"].shape[0]
    q = s["qkv"][:, :hq * d].view(n, hq, d)
    k = s["qkv"][:, hq * d:(hq + hkv) * d].view(n, hkv, d)
    v = s["qkv"][:, (hq + hkv) * d:].view(n, hkv, d)
    out, lse = ops.packed_attn_fwd(q, k, v, plan, causal=case["causal"], **bias)
    if case["kind"] != "attn_train":
        return out, lse
    if not case["buckets"]:
        return (out,) + ops.packed_attn_bwd(s["dout"], q, k, v, out, lse, plan, causal=case["causal"])
    dtable = torch.empty_like(s["table"])
    return (out,) + ops.packed_attn_bwd(s["dout"], q, k, v, out, lse, plan, causal=case["causal"], dbias_table=dtable, **bias) + (dtable,)


# ---- the definition in 64 bits -----------------------------------------------------------------------------------------------------
def _bucket_of(rel, buckets, max_distance, causal):
    """Bucket of one relative position (key - query), straight from the formula: the largest log bucket k with
    (n / e)^K >= (m / e)^k, found by comparing whole numbers."""
    side = buckets if causal else buckets // 2
    base = side if (not causal and rel > 0) else 0
    n = max(0, -rel) if causal else abs(rel)
    e = side // 2
    if n < e:
        return base + n
    top = side - e
    k = 0
    while k + 1 < top and n ** top * e ** (k + 1) >= max_distance ** (k + 1) * e ** top:
        k += 1
    return base + e + k


def _exact_attn(case, s, lens):
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    step, train = case["kind"] == "attn_step", case["kind"] == "attn_train"
    n = case["seqs"] if step else sum(lens)
    dev = (s["q"] if step else s["qkv"]).device
    out = torch.zeros(n, hq, d, dtype=torch.float64, device=dev)
    lse = torch.full((n, hq), -math.inf, dtype=torch.float64, device=dev)
    if not step:
        q_all, k_all, v_all = s["qkv"].double().split([hq * d, hkv * d, hkv * d], 1)
        dq, dk, dv = (torch.zeros(n, h, d, dtype=torch.float64, device=dev) for h in (hq, hkv, hkv))
    table = s["table"].double().requires_grad_(train) if case["buckets"] else None
    if case["buckets"]:
        m = max(lens) + 1
        far = min(m, case["max_distance"])
        lut = torch.tensor([_bucket_of(r, case["buckets"], case["max_distance"], case["causal"]) for r in range(-far, far + 1)], device=dev)
    row = 0
    for b, ln in enumerate(lens):
        nq = 1 if step else ln
        rows = slice(row, row + nq)
        row += nq
        if not ln or not nq:
            continue
        if step:
            q, k, v = s["q"][rows].double(), s["k"][b, :ln].double(), s["v"][b, :ln].double()
        else:
            q, k, v = q_all[rows].reshape(nq, hq, d), k_all[rows].reshape(ln, hkv, d), v_all[rows].reshape(ln, hkv, d)
        if case["buckets"] or case["causal"]:
            rel = torch.arange(ln, device=dev)[None, :] - (torch.arange(nq, device=dev)[:, None] + ln - nq)
        for kv in range(hkv):                                # one shared head and the query heads that read it
            hs = slice(kv * (hq // hkv), (kv + 1) * (hq // hkv))
            qq, kk, vv = (x.clone().requires_grad_(train) for x in (q[:, hs].transpose(0, 1), k[:, kv], v[:, kv]))
            sc = torch.matmul(qq, kk.t()) / math.sqrt(d)
            if case["buckets"]:
                sc = sc + table[:, hs].t()[:, lut[rel.clamp(-far, far) + far]]
            if case["causal"]:
                sc = sc.masked_fill(rel > 0, -math.inf)
            o = torch.matmul(torch.softmax(sc, -1), vv)
            out[rows, hs] = o.detach().transpose(0, 1)
            lse[rows, hs] = torch.logsumexp(sc.detach(), -1).t()
            if train:
                o.backward(s["dout"][rows, hs].double().transpose(0, 1))
                dq[rows, hs], dk[rows, kv], dv[rows, kv] = qq.grad.transpose(0, 1), kk.grad, vv.grad
            del sc, o
    if not train:
        return out, lse
    if not case["buckets"]:
        return out, dq, dk, dv
    return out, dq, dk, dv, table.grad if table.grad is not None else torch.zeros_like(table)


def _exact_rec(case, s, lens):
    c, reverse, train = case["c"], case["reverse"], case["kind"] == "rec_train"
    gate, cand = s["gates"].double().split(c, 1)
    z = 1 / (1 + torch.exp(-gate))
    h, lam = torch.zeros_like(z), torch.zeros_like(z)
    last, dh0 = s["h0"].double(), torch.zeros_like(s["h0"], dtype=torch.float64)
    prev = torch.zeros_like(z)
    order = np.argsort([-x for x in lens], kind="stable")    # longest first: the streams still running are a prefix
    first = np.cumsum([0] + list(lens))[:-1]
    idx = [int(i) for i in order]
    start = torch.tensor([int(first[i]) for i in idx], device=z.device)
    length = torch.tensor([int(lens[i]) for i in idx], device=z.device)
    state = last[idx].clone()

    def rows_at(t):
        live = sum(1 for i in idx if lens[i] > t)
        at = start[:live] + (length[:live] - 1 - t if reverse else t)
        return live, at

    longest = max(lens)
    steps = [rows_at(t) for t in range(longest)]
    for live, at in steps:
        prev[at] = state[:live]
        state[:live] = z[at] * state[:live] + (1 - z[at]) * cand[at]
        h[at] = state[:live]
    last = last.clone()
    last[idx] = state
    if not train:
        return h, last
    grad = s["dlast"].double()[idx].clone()
    dh = s["dh"].double()
    for live, at in reversed(steps):
        grad[:live] += dh[at]
        lam[at] = grad[:live]
        grad[:live] *= z[at]
    dh0[idx] = grad
    return h, last, lam * (prev - cand) * z * (1 - z), lam * (1 - z), dh0


def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    lens = _lens(case)
    return _exact_rec(case, s, lens) if case["kind"].startswith("rec") else _exact_attn(case, s, lens)
