"""Causal decoder of the CRNN networks for whole recordings and running streams - forward AND hand-written backward.

The decoders of `Decoder` (reference models/components/model_utilities.py:245-263: Conformer, GRU, nn.TransformerEncoder) look at both
sides of a frame and at chunks of one length. This one (`cfg.model.decoder` = 'stream') looks back only and takes recordings of any lengths laid
back to back, and its step() carries a batch of live streams forward by one frame with the same weights. Per layer, pre-norm:
x = x + out_proj(attention(norm1(x))); x = x + linear2(recurrence(linear1(norm2(x)))). The attention is causal with grouped heads and a learned
relative position bias by buckets (ops.packed_attn_*); linear1 gives the update gates | candidates of the gated linear recurrence
(ops.linrec_*: nn.GRU's update rule without the recurrent product).
"""
import math

import torch

from ... import _lib, ops


class StreamState:
    """What step() carries from frame to frame: per layer the key and value slabs [streams * capacity, key heads, head size] and the recurrence's
    state f32 [streams, D]; plan.k_len holds the frames each stream has seen. All streams of a state begin together. `frames` is what the host has
    counted: step() adds one where it runs, advance() what replays of a captured step() are about to add."""

    def __init__(self, plan, first, keys, values, states, capacity):
        self.plan, self.first, self.keys, self.values, self.states, self.capacity, self.frames = plan, first, keys, values, states, capacity, 0

    def remaining(self):
        """Frames that the caches still have room for, by the host's count."""
        return self.capacity - self.frames

    def advance(self, n=1):
        """To be called before n replays of a captured step(), which the host does not see otherwise: counts them, or refuses where the caches
        would overflow. (Replays past the capacity that nobody counted answer with NaN.)"""
        if n < 0 or n > self.remaining():
            raise _lib.PseldError(f"stream decoder: the streams' caches hold {self.capacity} frames, {self.frames} are taken: no room for {n} more")
        self.frames += n


class StreamDecoder:
    """num_layers blocks of width dim; head size 64 where dim allows it, four query heads share a key head."""

    def __init__(self, arena, prefix, dim, num_layers, num_buckets=32, max_distance=128):
        if dim % 8:
            raise ValueError("stream decoder: the width must be a multiple of 8")
        self.arena, self.prefix, self.D, self.L = arena, prefix, dim, num_layers
        self.hd = next(h for h in (64, 32, 16, 8) if dim % h == 0)
        self.heads = dim // self.hd
        self.kv_heads = self.heads // 4 if self.heads % 4 == 0 else self.heads
        self.W = (self.heads + 2 * self.kv_heads) * self.hd
        self.num_buckets, self.max_distance = num_buckets, max_distance
        self._buckets, self._plans = {}, {}      # never dropped: a captured graph goes on reading them
        for li in range(num_layers):
            b = f'{prefix}layers.{li}.'
            arena.add(b + 'norm1.weight', (dim,)); arena.add(b + 'norm1.bias', (dim,))
            arena.add(b + 'self_attn.in_proj_weight', (self.W, dim)); arena.add(b + 'self_attn.in_proj_bias', (self.W,))
            arena.add(b + 'self_attn.relative_position_bias_table', (num_buckets, self.heads))
            arena.add(b + 'self_attn.out_proj.weight', (dim, dim)); arena.add(b + 'self_attn.out_proj.bias', (dim,))
            arena.add(b + 'norm2.weight', (dim,)); arena.add(b + 'norm2.bias', (dim,))
            arena.add(b + 'linear1.weight', (2 * dim, dim)); arena.add(b + 'linear1.bias', (2 * dim,))
            arena.add(b + 'linear2.weight', (dim, dim)); arena.add(b + 'linear2.bias', (dim,))

    def static_buffers(self):
        return {}

    def _relpos(self, device):
        if device not in self._buckets:
            self._buckets[device] = ops.relpos_buckets(self.num_buckets, self.max_distance, bidirectional=False, device=device)
        return self._buckets[device]

    def _heads(self, qkv):
        n, hq, hk, d = qkv.shape[0], self.heads, self.kv_heads, self.hd
        return (qkv[:, :hq * d].view(n, hq, d), qkv[:, hq * d:(hq + hk) * d].view(n, hk, d), qkv[:, (hq + hk) * d:].view(n, hk, d))

    # -- recordings ------------------------------------------------------------------------------------------------------
    def forward(self, x, B, T, training=None, buffers=None):
        """x [B*T, D], B chunks of T frames -> [B*T, D]."""
        key = (B, T, x.device)
        if key not in self._plans:
            self._plans[key] = ops.packed_plan([T] * B, device=x.device)
        return self.forward_packed(x, self._plans[key])

    def forward_packed(self, x, plan):
        """x [rows, D]: the plan's recordings back to back -> [rows, D]."""
        a, dt, D = self.arena, x.dtype, self.D
        buckets, saved = self._relpos(x.device), []
        for li in range(self.L):
            b = f'{self.prefix}layers.{li}.'
            y1 = ops.layernorm_fwd(x, a.p(b + 'norm1.weight'), a.p(b + 'norm1.bias'))
            qkv = ops.linear_fwd(y1, a.w(b + 'self_attn.in_proj_weight', dt), a.p(b + 'self_attn.in_proj_bias'))
            ctx, lse = ops.packed_attn_fwd(*self._heads(qkv), plan, causal=True, bias_table=a.p(b + 'self_attn.relative_position_bias_table'), buckets=buckets)
            x1 = ops.linear_fwd(ctx.view(-1, D), a.w(b + 'self_attn.out_proj.weight', dt), a.p(b + 'self_attn.out_proj.bias'), resid=x)
            y2 = ops.layernorm_fwd(x1, a.p(b + 'norm2.weight'), a.p(b + 'norm2.bias'))
            u = ops.linear_fwd(y2, a.w(b + 'linear1.weight', dt), a.p(b + 'linear1.bias'))
            h, _, states = ops.linrec_fwd(u[:, :D], u[:, D:], plan)
            x2 = ops.linear_fwd(h, a.w(b + 'linear2.weight', dt), a.p(b + 'linear2.bias'), resid=x1)
            saved.append(dict(x=x, y1=y1, qkv=qkv, ctx=ctx, lse=lse, x1=x1, y2=y2, u=u, states=states, h=h))
            x = x2
        return x, dict(layers=saved, plan=plan)

    def backward(self, dx, saved, B=None):
        """dx [rows, D] -> the input's gradient; parameter gradients land in the arena."""
        a, dt, D, plan = self.arena, dx.dtype, self.D, saved['plan']
        buckets = self._relpos(dx.device)
        for li in reversed(range(self.L)):
            b = f'{self.prefix}layers.{li}.'
            s = saved['layers'][li]
            ops.linear_wgrad(dx, s['h'], a.g(b + 'linear2.weight'), dbias=a.g(b + 'linear2.bias'))
            dh = ops.linear_dgrad(dx, a.w(b + 'linear2.weight', dt), wt=a.wt(b + 'linear2.weight', dt))
            u, du = s['u'], torch.empty_like(s['u'])
            ops.linrec_bwd(dh, u[:, :D], u[:, D:], s['states'], plan, dg=du[:, :D], dn=du[:, D:])
            ops.linear_wgrad(du, s['y2'], a.g(b + 'linear1.weight'), dbias=a.g(b + 'linear1.bias'))
            dy2 = ops.linear_dgrad(du, a.w(b + 'linear1.weight', dt), wt=a.wt(b + 'linear1.weight', dt))
            dx1 = ops.layernorm_bwd(dy2, s['x1'], a.p(b + 'norm2.weight'), a.g(b + 'norm2.weight'), a.g(b + 'norm2.bias'), dres=dx)
            ops.linear_wgrad(dx1, s['ctx'].view(-1, D), a.g(b + 'self_attn.out_proj.weight'), dbias=a.g(b + 'self_attn.out_proj.bias'))
            dctx = ops.linear_dgrad(dx1, a.w(b + 'self_attn.out_proj.weight', dt), wt=a.wt(b + 'self_attn.out_proj.weight', dt))
            dqkv = torch.empty_like(s['qkv'])
            dq, dk, dv = self._heads(dqkv)
            table = b + 'self_attn.relative_position_bias_table'
            ops.packed_attn_bwd(dctx.view(-1, self.heads, self.hd), *self._heads(s['qkv']), s['ctx'], s['lse'], plan, causal=True, bias_table=a.p(table),
                                buckets=buckets, dbias_table=a.g(table), dq=dq, dk=dk, dv=dv)
            ops.linear_wgrad(dqkv, s['y1'], a.g(b + 'self_attn.in_proj_weight'), dbias=a.g(b + 'self_attn.in_proj_bias'))
            dy1 = ops.linear_dgrad(dqkv, a.w(b + 'self_attn.in_proj_weight', dt), wt=a.wt(b + 'self_attn.in_proj_weight', dt))
            dx = ops.layernorm_bwd(dy1, s['x'], a.p(b + 'norm1.weight'), a.g(b + 'norm1.weight'), a.g(b + 'norm1.bias'), dres=dx1)
        return dx

    # -- running streams -------------------------------------------------------------------------------------------------
    def stream_state(self, streams, capacity, device, dtype):
        """Empty caches for `streams` live streams of at most `capacity` frames."""
        if dtype not in (torch.float32, torch.bfloat16):
            raise _lib.PseldError(f"stream decoder: streams run in float32 or bfloat16, not {dtype}")
        plan = ops.packed_plan([1] * streams, [0] * streams, k_cap=capacity, device=device)
        slab = lambda: torch.zeros((streams * capacity, self.kv_heads, self.hd), dtype=dtype, device=plan.device)      # noqa: E731
        return StreamState(plan, torch.arange(streams, device=plan.device) * capacity, [slab() for _ in range(self.L)], [slab() for _ in range(self.L)],
                           [torch.zeros((streams, self.D), dtype=torch.float32, device=plan.device) for _ in range(self.L)], capacity)

    def step(self, x, state):
        """x [streams, D]: the next frame of every stream (any row stride) -> [streams, D], what forward_packed gives for that frame of the whole
        recording. The caches and states move on in place, or not at all where the call raises. It can be captured into a graph (after one eager
        step): state.advance() before a replay refuses the frame that no longer fits, as an eager call does by itself. A stream whose cache is full
        all the same, by replays that were not counted, gets NaN: its caches and its state are no longer those of its frames."""
        plan, D = state.plan, self.D
        ops._on_plan("stream decoder", plan)
        if len(state.keys) != self.L or state.keys[0].shape[1:] != (self.kv_heads, self.hd) or state.states[0].shape[1] != D:
            raise _lib.PseldError("stream decoder: the state was made by a decoder of another shape")
        if x.shape != (plan.seqs, D) or x.dtype != state.keys[0].dtype or x.device != plan.device:
            raise _lib.PseldError(f"stream decoder: a frame of these streams is {state.keys[0].dtype} [{plan.seqs}, {D}] on {plan.device}")
        capturing = torch.cuda.is_current_stream_capturing()      # nothing runs then: the replays count
        if state.remaining() < 1:
            raise _lib.PseldError(f"stream decoder: the streams' caches hold {state.capacity} frames and are full")
        x = x.contiguous()
        at = state.first + plan.k_len.clamp(0, state.capacity - 1)      # a replay past the capacity stays inside the slabs
        plan.k_len.add_(1)
        try:
            x, states = self._step(x, state, at)
            x.masked_fill_((plan.k_len > state.capacity)[:, None], math.nan)
        except BaseException:
            if not capturing:
                plan.k_len.sub_(1)
            raise
        for kept, last in zip(state.states, states):
            kept.copy_(last)
        if not capturing:
            state.advance()
        return x

    def _step(self, x, state, at):
        """The layers of step(): writes the new keys and values at the rows `at` (past what the plan's lengths counted so far), returns the output and
        the recurrences' new states."""
        a, dt, D, plan, states = self.arena, x.dtype, self.D, state.plan, []
        buckets = self._relpos(x.device)
        for li in range(self.L):
            b = f'{self.prefix}layers.{li}.'
            y1 = ops.layernorm_fwd(x, a.p(b + 'norm1.weight'), a.p(b + 'norm1.bias'))
            qkv = ops.linear_fwd(y1, a.w(b + 'self_attn.in_proj_weight', dt), a.p(b + 'self_attn.in_proj_bias'))
            q, k, v = self._heads(qkv)
            state.keys[li].index_copy_(0, at, k)
            state.values[li].index_copy_(0, at, v)
            ctx, _ = ops.packed_attn_fwd(q, state.keys[li], state.values[li], plan, causal=True,
                                         bias_table=a.p(b + 'self_attn.relative_position_bias_table'), buckets=buckets)
            x1 = ops.linear_fwd(ctx.view(-1, D), a.w(b + 'self_attn.out_proj.weight', dt), a.p(b + 'self_attn.out_proj.bias'), resid=x)
            y2 = ops.layernorm_fwd(x1, a.p(b + 'norm2.weight'), a.p(b + 'norm2.bias'))
            u = ops.linear_fwd(y2, a.w(b + 'linear1.weight', dt), a.p(b + 'linear1.bias'))
            h, last, _ = ops.linrec_fwd(u[:, :D], u[:, D:], plan, h0=state.states[li], need_saved=False)
            states.append(last)
            x = ops.linear_fwd(h, a.w(b + 'linear2.weight', dt), a.p(b + 'linear2.bias'), resid=x1)
        return x, states
