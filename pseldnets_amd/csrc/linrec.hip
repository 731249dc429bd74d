// Gated linear recurrence over packed recordings, forward and backward, gfx950.
//
//   z = sigmoid(g),  h_t = z_t h_{t-1} + (1 - z_t) n_t          (the update rule of nn.GRU with its recurrent product taken out)
//   backward with lambda_t = dL/dh_t in full and mu_t = z_t lambda_t (what reaches h_{t-1}):
//   lambda_t = dh_t + mu_{t+1},  dn_t = lambda_t (1 - z_t),  dg_t = lambda_t (h_{t-1} - n_t) z_t (1 - z_t),  dh0 = mu_0
//
// Both directions are first-order linear recurrences x -> A x + B, which compose: (A2, B2) o (A1, B1) = (A2 A1, A2 B1 + B2). A workgroup
// owns 64 channels (one whole cache line of bf16 per row) of one segment of one recording and walks it in tiles of 64 frames: a thread
// holds 4 consecutive frames of 4 channels in registers, composes them, the four thread groups of a wave compose by shuffles and the four
// waves through 4 KB of LDS (one barrier per tile, images alternate), then every thread replays its 4 frames from its exact starting state.
// The next tile's rows are requested before the current one is worked on. Composition order is fixed by the sizes alone: results do not
// depend on timing.
//
// What bounds it: HBM. The forward reads g and n and writes h once; the backward reads g, n, dh and writes dg, dn - h is recomputed from the f32
// states that the forward leaves at every tile start (1/32 of h's bytes in bf16), so the gradient does not see h's rounding either.
// Few recordings with few channels leave CUs idle, so a long recording is cut into segments: one more launch composes every segment
// to (A, B) first, and each segment's workgroup folds the segments before its own into its starting state. That reads the operands twice, so the
// segment length is the shortest that still gives about SEG_WGS workgroups, and one segment (one launch) where the batch fills the chip.
// States, sums and compositions are f32; h, dg, dn are rounded once to the operands' type on their way out.
#include "common.h"

namespace {

constexpr int TILE = 64;         // frames per tile: 16 thread groups x 4 frames
constexpr int R = 4;             // frames per thread (8, twice the bytes in flight: 32 x 200-1000 x 1024 bf16, forward + backward, 93 us against 90)
constexpr int SLAB = 64;         // channels per workgroup: 16 lanes x 4
constexpr int SEG_WGS = 1024;    // four workgroups per CU (2 x 60000 x 512 f32, forward + backward: 512 606 us, 1024 601, 2048 607)

struct LinrecArgs {
    const void* g; const void* n; const void* dh;
    void* h; void* dg; void* dn;
    long ldg, ldn, lddh, ldh, lddg, lddn;      // row strides in elements
    const float* h0;          // [seqs, C] or null (zeros)
    const float* dlast;       // [seqs, C] or null
    float* h_last;            // [seqs, C]
    float* dh0;               // [seqs, C] or null
    float* states;            // [rows / TILE + seqs + 1, C] state before each tile's first frame; null: not wanted (forward)
    float* agg;               // [rows / seg_len + seqs + 1, 2, C]
    const int* start; const int* len;
    int seqs, C, slabs, nseg, seg_len, reverse;
    int descending;           // workgroups take the segments last to first
};

template <typename T> struct Quad;
template <> struct Quad<bf16_t> {
    bf16x4 v;
    __device__ __forceinline__ float get(int i) const { return (float)v[i]; }
};
template <> struct Quad<float> {
    f32x4 v;
    __device__ __forceinline__ float get(int i) const { return v[i]; }
};
template <typename T> __device__ __forceinline__ void put_quad(T* p, const float (&x)[4]) {
    Quad<T> q;
#pragma unroll
    for (int i = 0; i < 4; ++i) q.v[i] = (T)x[i];
    *(decltype(q.v)*)p = q.v;
}
// z = sigmoid(g) = 1 / (1 + e) and 1 - z = e / (1 + e) with e = exp(-g): neither by cancellation. e is held below 2^115, so that e / (1 + e) stays 1
// where exp(-g) would overflow (a NaN stays one)
__device__ __forceinline__ void gate_of(float g, float& z, float& y) {
    float x = g * -1.4426950408889634f;
    x = x > 115.f ? 115.f : x;
    const float e = __builtin_amdgcn_exp2f(x);
    z = __builtin_amdgcn_rcpf(1.f + e);
    y = e * z;
}

struct Place {       // which recording, segment and channels a workgroup owns, and which frames and channels a thread does
    int seq, seg, len, t_end, t0, c, tg, tgl, wave;
    long row0;
    bool live;       // the thread's channels exist
};
__device__ __forceinline__ Place place_of(const LinrecArgs& a) {
    Place p;
    const int slab = blockIdx.x % a.slabs, at = blockIdx.x / a.slabs, rest = a.descending ? a.seqs * a.nseg - 1 - at : at;
    p.seg = rest % a.nseg;
    p.seq = rest / a.nseg;
    p.len = a.len[p.seq];
    p.row0 = a.start[p.seq];
    p.t0 = p.seg * a.seg_len;
    p.t_end = min(p.len, p.t0 + a.seg_len);
    const int lane = threadIdx.x & 63;
    p.wave = threadIdx.x >> 6;
    p.tgl = lane >> 4;
    p.tg = p.wave * 4 + p.tgl;
    p.c = slab * SLAB + (lane & 15) * 4;
    p.live = p.c < a.C;
    return p;
}
// An operand's rows of one tile: a uniform base (the tile's lowest row in memory) and 32-bit offsets per lane that are the same for every tile. Rows
// step up with time, down when reverse. Loads are unconditional - rows past the segment repeat its last one, channels past C the last four, and
// the values are dropped later - so that nothing has to merge behind a request and wait for it.
template <typename T> struct Rows {
    char* base;                // row0 of the recording
    long ld;                   // bytes per row
    unsigned first, chan;      // bytes from a tile's lowest row to the thread's first frame; of its channels
    int step;                  // bytes from one frame's row to the next
    __device__ __forceinline__ Rows(const void* p0, long ld_, const LinrecArgs& a, const Place& p) {
        ld = ld_ * (long)sizeof(T);
        base = (char*)p0 + p.row0 * ld;
        first = (a.reverse ? TILE - 1 - p.tg * R : p.tg * R) * (unsigned)ld;
        chan = min(p.c, a.C - 4) * (unsigned)sizeof(T);
        step = a.reverse ? -(int)ld : (int)ld;
    }
    __device__ __forceinline__ char* tile(const LinrecArgs& a, const Place& p, int t0) const {
        return base + (long)(a.reverse ? p.len - t0 - TILE : t0) * ld;
    }
    __device__ __forceinline__ char* row(char* tile_base, int i) const { return tile_base + (first + (unsigned)(i * step) + chan); }
    __device__ __forceinline__ void fetch(Quad<T> (&q)[R], const LinrecArgs& a, const Place& p, int t0) const {
        char* b = tile(a, p, t0);
        const int live = min(TILE, p.t_end - t0);          // frames of the tile that exist
        const unsigned lo = a.reverse ? (unsigned)(TILE - live) * (unsigned)ld : 0u, hi = a.reverse ? (TILE - 1) * (unsigned)ld : (unsigned)(live - 1) * (unsigned)ld;
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const unsigned o = max(lo, min(hi, first + (unsigned)(i * step)));
            q[i].v = *(const decltype(q[i].v)*)(b + (o + chan));
        }
    }
};

// lanes `from` lanes below / above hold the neighbouring thread groups of the same channels
__device__ __forceinline__ float from_lane(float v, int lane) { return __shfl(v, lane, 64); }

// ---- forward. AGG: only the segment's composition (A, B) is wanted -----------------------------------------------------------------
template <typename T, bool AGG>
__global__ __launch_bounds__(256) void linrec_fwd_kernel(LinrecArgs a) {
    __shared__ f32x4 xa[2][4][16], xb[2][4][16];
    const Place p = place_of(a);
    const int cl = threadIdx.x & 15, lane = threadIdx.x & 63;
    if (p.t0 >= p.len) {
        if (!AGG && p.len == 0 && p.seg == 0 && p.live && p.tg == 0)
            *(f32x4*)(a.h_last + (long)p.seq * a.C + p.c) = a.h0 ? *(const f32x4*)(a.h0 + (long)p.seq * a.C + p.c) : f32x4{0.f, 0.f, 0.f, 0.f};
        return;
    }
    if (AGG && p.t_end == p.len) return;                 // nobody starts from the last segment's end
    float carry[4] = {0.f, 0.f, 0.f, 0.f}, prod[4] = {1.f, 1.f, 1.f, 1.f};
    const long seg0 = p.row0 / a.seg_len + p.seq;
    if (!AGG && p.live) {
        if (a.h0) {
            const f32x4 v = *(const f32x4*)(a.h0 + (long)p.seq * a.C + p.c);
#pragma unroll
            for (int i = 0; i < 4; ++i) carry[i] = v[i];
        }
#pragma unroll 4
        for (int j = 0; j < p.seg; ++j) {                // the segments before this one, in order
            const float* s = a.agg + (seg0 + j) * 2 * a.C + p.c;
            const f32x4 A = *(const f32x4*)s, B = *(const f32x4*)(s + a.C);
#pragma unroll
            for (int i = 0; i < 4; ++i) carry[i] = fmaf(A[i], carry[i], B[i]);
        }
    }
    const Rows<T> rg(a.g, a.ldg, a, p), rn(a.n, a.ldn, a, p), rh(a.h, a.ldh, a, p);
    Quad<T> qg[R], qn[R];
    rg.fetch(qg, a, p, p.t0);
    rn.fetch(qn, a, p, p.t0);
    const int last = p.t0 + (p.t_end - 1 - p.t0) / TILE * TILE;
    int par = 0;
    for (int t0 = p.t0; t0 < p.t_end; t0 += TILE, par ^= 1) {
        const int t = t0 + p.tg * R;
        const bool whole = t0 + TILE <= p.t_end;
        float z[R][4], b[R][4], A[4], B[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) { A[c] = 1.f; B[c] = 0.f; }
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                float y;
                gate_of(qg[i].get(c), z[i][c], y);
                b[i][c] = y * qn[i].get(c);
            }
        if (!whole)
#pragma unroll
            for (int i = 0; i < R; ++i)
                if (t + i >= p.t_end)
#pragma unroll
                    for (int c = 0; c < 4; ++c) { z[i][c] = 1.f; b[i][c] = 0.f; }
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                A[c] *= z[i][c];
                B[c] = fmaf(z[i][c], B[c], b[i][c]);
            }
        rg.fetch(qg, a, p, min(t0 + TILE, last));
        rn.fetch(qn, a, p, min(t0 + TILE, last));
        // inclusive composition over the wave's four thread groups
#pragma unroll
        for (int o = 16; o <= 32; o <<= 1)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const float pa = from_lane(A[c], lane - o), pb = from_lane(B[c], lane - o);
                if (lane >= o) { B[c] = fmaf(A[c], pb, B[c]); A[c] *= pa; }
            }
        if (p.tgl == 3) { xa[par][p.wave][cl] = f32x4{A[0], A[1], A[2], A[3]}; xb[par][p.wave][cl] = f32x4{B[0], B[1], B[2], B[3]}; }
        __syncthreads();
        float in[4] = {carry[0], carry[1], carry[2], carry[3]};      // state before the wave's first frame
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const f32x4 wa = xa[par][w][cl], wb = xb[par][w][cl];
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                if (w == p.wave) in[c] = carry[c];
                carry[c] = fmaf(wa[c], carry[c], wb[c]);
                if (AGG) prod[c] *= wa[c];
            }
        }
        if constexpr (!AGG) {
            if (a.states && p.tg == 0 && p.live)
                *(f32x4*)(a.states + (p.row0 / TILE + p.seq + t0 / TILE) * a.C + p.c) = f32x4{in[0], in[1], in[2], in[3]};
            float x[4];
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const float ea = from_lane(A[c], lane - 16), eb = from_lane(B[c], lane - 16);
                x[c] = p.tgl ? fmaf(ea, in[c], eb) : in[c];
            }
            char* hb = rh.tile(a, p, t0);
#pragma unroll
            for (int i = 0; i < R; ++i) {
#pragma unroll
                for (int c = 0; c < 4; ++c) x[c] = fmaf(z[i][c], x[c], b[i][c]);
                if (p.live && (whole || t + i < p.t_end)) put_quad<T>((T*)rh.row(hb, i), x);
            }
            // frames past the end leave the state alone: the last thread's is the recording's
            if (t0 + TILE >= p.len && p.live && p.tg == 15) *(f32x4*)(a.h_last + (long)p.seq * a.C + p.c) = f32x4{x[0], x[1], x[2], x[3]};
        }
    }
    if (AGG && p.tg == 0 && p.live) {
        float* s = a.agg + (seg0 + p.seg) * 2 * a.C + p.c;
        *(f32x4*)s = f32x4{prod[0], prod[1], prod[2], prod[3]};
        *(f32x4*)(s + a.C) = f32x4{carry[0], carry[1], carry[2], carry[3]};
    }
}

// ---- backward: the tiles of a segment last to first. AGG: only mu's composition over the segment ------------------------------------
template <typename T, bool AGG>
__global__ __launch_bounds__(256) void linrec_bwd_kernel(LinrecArgs a) {
    __shared__ f32x4 xa[2][4][16], xb[2][4][16], xm[2][4][16];
    const Place p = place_of(a);
    const int cl = threadIdx.x & 15, lane = threadIdx.x & 63;
    const long sc = (long)p.seq * a.C + p.c;
    if (p.t0 >= p.len) {
        if (!AGG && p.len == 0 && p.seg == 0 && p.live && p.tg == 0 && a.dh0)
            *(f32x4*)(a.dh0 + sc) = a.dlast ? *(const f32x4*)(a.dlast + sc) : f32x4{0.f, 0.f, 0.f, 0.f};
        return;
    }
    if (AGG && p.seg == 0) return;                       // nobody takes over from the first segment's start
    float carry[4] = {0.f, 0.f, 0.f, 0.f}, prod[4] = {1.f, 1.f, 1.f, 1.f};      // mu of the frame behind the tile
    const long seg0 = p.row0 / a.seg_len + p.seq;
    if (!AGG && p.live) {
        if (a.dlast) {
            const f32x4 v = *(const f32x4*)(a.dlast + sc);
#pragma unroll
            for (int i = 0; i < 4; ++i) carry[i] = v[i];
        }
#pragma unroll 4
        for (int j = (p.len - 1) / a.seg_len; j > p.seg; --j) {
            const float* s = a.agg + (seg0 + j) * 2 * a.C + p.c;
            const f32x4 A = *(const f32x4*)s, B = *(const f32x4*)(s + a.C);
#pragma unroll
            for (int i = 0; i < 4; ++i) carry[i] = fmaf(A[i], carry[i], B[i]);
        }
    }
    Quad<T> qg[R], qn[R], qd[R];
    const int last = p.t0 + (p.t_end - 1 - p.t0) / TILE * TILE;
    const Rows<T> rg(a.g, a.ldg, a, p), rn(a.n, a.ldn, a, p), rd(a.dh, a.lddh, a, p), og(a.dg, a.lddg, a, p), on(a.dn, a.lddn, a, p);
    rg.fetch(qg, a, p, last);
    if constexpr (!AGG) rn.fetch(qn, a, p, last);
    rd.fetch(qd, a, p, last);
    const float* states = AGG ? nullptr : a.states + (p.row0 / TILE + p.seq) * a.C + min(p.c, a.C - 4);
    f32x4 nst = {0.f, 0.f, 0.f, 0.f};
    if constexpr (!AGG) nst = *(const f32x4*)(states + (long)(last / TILE) * a.C);
    int par = 0;
    for (int t0 = last; t0 >= p.t0; t0 -= TILE, par ^= 1) {
        const int t = t0 + p.tg * R;
        const bool whole = t0 + TILE <= p.t_end;
        float z[R][4], y[R][4], n[R][4], d[R][4], A[4], B[4], M[4];
        const f32x4 st = nst;                             // the state before the tile
#pragma unroll
        for (int c = 0; c < 4; ++c) { A[c] = 1.f; B[c] = 0.f; M[c] = 0.f; }
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                gate_of(qg[i].get(c), z[i][c], y[i][c]);
                d[i][c] = qd[i].get(c);
                if constexpr (!AGG) n[i][c] = qn[i].get(c);
            }
        if (!whole)
#pragma unroll
            for (int i = 0; i < R; ++i)
                if (t + i >= p.t_end)
#pragma unroll
                    for (int c = 0; c < 4; ++c) { z[i][c] = 1.f; y[i][c] = 0.f; d[i][c] = 0.f; }
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                A[c] *= z[i][c];
                if constexpr (!AGG) B[c] = fmaf(z[i][c], B[c], y[i][c] * n[i][c]);
            }
#pragma unroll
        for (int i = R - 1; i >= 0; --i)
#pragma unroll
            for (int c = 0; c < 4; ++c) M[c] = z[i][c] * (d[i][c] + M[c]);
        const int next = max(t0 - TILE, p.t0);
        rg.fetch(qg, a, p, next);
        if constexpr (!AGG) rn.fetch(qn, a, p, next);
        rd.fetch(qd, a, p, next);
        if constexpr (!AGG) nst = *(const f32x4*)(states + (long)(next / TILE) * a.C);
        // inclusive compositions over the wave's thread groups: the states from the first group on, mu from the last group back
        float S[4] = {A[0], A[1], A[2], A[3]};           // product from this group to the wave's last
#pragma unroll
        for (int o = 16; o <= 32; o <<= 1)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                if constexpr (!AGG) {
                    const float pa = from_lane(A[c], lane - o), pb = from_lane(B[c], lane - o);
                    if (lane >= o) { B[c] = fmaf(A[c], pb, B[c]); A[c] *= pa; }
                }
                const float na = from_lane(S[c], lane + o), nm = from_lane(M[c], lane + o);
                if (lane + o < 64) { M[c] = fmaf(S[c], nm, M[c]); S[c] *= na; }
            }
        if (p.tgl == 3 && !AGG) xb[par][p.wave][cl] = f32x4{B[0], B[1], B[2], B[3]};
        if (p.tgl == 0) { xa[par][p.wave][cl] = f32x4{S[0], S[1], S[2], S[3]}; xm[par][p.wave][cl] = f32x4{M[0], M[1], M[2], M[3]}; }
        __syncthreads();
        float mu[4] = {0.f, 0.f, 0.f, 0.f}, in[4] = {st[0], st[1], st[2], st[3]};      // mu behind the wave's last frame, state before its first
#pragma unroll
        for (int w = 3; w >= 0; --w) {
            const f32x4 wa = xa[par][w][cl], wm = xm[par][w][cl];
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                if (w == p.wave) mu[c] = carry[c];
                carry[c] = fmaf(wa[c], carry[c], wm[c]);
                if (AGG) prod[c] *= wa[c];
            }
        }
        if constexpr (!AGG) {
#pragma unroll
            for (int w = 0; w < 3; ++w) {
                const f32x4 wa = xa[par][w][cl], wb = xb[par][w][cl];
                if (w < p.wave)
#pragma unroll
                    for (int c = 0; c < 4; ++c) in[c] = fmaf(wa[c], in[c], wb[c]);
            }
            float x[4], m[4];
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const float ea = from_lane(A[c], lane - 16), eb = from_lane(B[c], lane - 16);
                const float na = from_lane(S[c], lane + 16), nm = from_lane(M[c], lane + 16);
                x[c] = p.tgl ? fmaf(ea, in[c], eb) : in[c];
                m[c] = p.tgl < 3 ? fmaf(na, mu[c], nm) : mu[c];
            }
            float hp[R][4];                              // h_{t-1}
#pragma unroll
            for (int i = 0; i < R; ++i)
#pragma unroll
                for (int c = 0; c < 4; ++c) { hp[i][c] = x[c]; x[c] = fmaf(z[i][c], x[c], y[i][c] * n[i][c]); }
            char *gb = og.tile(a, p, t0), *nb = on.tile(a, p, t0);
#pragma unroll
            for (int i = R - 1; i >= 0; --i) {
                float vg[4], vn[4];
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const float lam = d[i][c] + m[c];
                    vn[c] = lam * y[i][c];
                    vg[c] = vn[c] * z[i][c] * (hp[i][c] - n[i][c]);
                    m[c] = z[i][c] * lam;
                }
                if (p.live && (whole || t + i < p.t_end)) {
                    put_quad<T>((T*)og.row(gb, i), vg);
                    put_quad<T>((T*)on.row(nb, i), vn);
                }
            }
        }
    }
    if (p.tg == 0 && p.live) {
        if constexpr (AGG) {
            float* s = a.agg + (seg0 + p.seg) * 2 * a.C + p.c;
            *(f32x4*)s = f32x4{prod[0], prod[1], prod[2], prod[3]};
            *(f32x4*)(s + a.C) = f32x4{carry[0], carry[1], carry[2], carry[3]};
        } else if (p.seg == 0 && a.dh0) {
            *(f32x4*)(a.dh0 + sc) = f32x4{carry[0], carry[1], carry[2], carry[3]};
        }
    }
}

// Frames per segment. Cutting costs a second read of the operands, so a batch whose longest recording is at most twice an even share of the rows over
// two workgroups per CU stays whole (32 x 200-1000 x 1024 bf16, forward + backward: whole 103 us, cut 158); otherwise about SEG_WGS segments
// of at least four tiles.
int seg_len_of(long rows, int max_len, int C) {
    const long slabs = (C + SLAB - 1) / SLAB, whole = max_len > 0 ? ((long)max_len + TILE - 1) / TILE * TILE : TILE;
    if (max_len <= 2 * (rows * slabs) / 512) return (int)whole;
    long s = ((rows * slabs + SEG_WGS - 1) / SEG_WGS + TILE - 1) / TILE * TILE;
    if (s < 4 * TILE) s = 4 * TILE;
    return (int)(s < whole ? s : whole);
}
long agg_bytes_of(long rows, int seqs, int max_len, int C) {
    const int s = seg_len_of(rows, max_len, C);
    return s >= max_len ? 0 : (rows / s + seqs + 1) * 2 * (long)C * (long)sizeof(float);
}

template <typename T>
void launch(LinrecArgs a, int backward, hipStream_t s) {
    const dim3 grid((unsigned)((long)a.slabs * a.nseg * a.seqs));
    if (!backward) {
        if (a.nseg > 1) hipLaunchKernelGGL((linrec_fwd_kernel<T, true>), grid, dim3(256), 0, s, a);
        a.descending = a.nseg > 1;                         // what the first launch read last is still in the caches
        hipLaunchKernelGGL((linrec_fwd_kernel<T, false>), grid, dim3(256), 0, s, a);
    } else {
        if (a.nseg > 1) hipLaunchKernelGGL((linrec_bwd_kernel<T, true>), grid, dim3(256), 0, s, a);
        a.descending = a.nseg > 1;
        hipLaunchKernelGGL((linrec_bwd_kernel<T, false>), grid, dim3(256), 0, s, a);
    }
}

int go(const char* name, int dtype, LinrecArgs& a, long rows, int max_len, const float* ws, long ws_bytes, int backward, void* stream) {
    PSELD_CHECK_ARG(dtype == PSELD_F32 || dtype == PSELD_BF16, "%s: unknown dtype", name);
    PSELD_CHECK_ARG(a.start && a.len && a.seqs > 0 && rows >= 0 && rows <= (1l << 30) && max_len >= 0 && max_len <= rows, "%s: bad recordings", name);
    PSELD_CHECK_ARG(a.C > 0 && a.C % 8 == 0, "%s: channels must be a positive multiple of 8", name);
    const long need = agg_bytes_of(rows, a.seqs, max_len, a.C);
    PSELD_CHECK_ARG(need == 0 || (ws && ws_bytes >= need), "%s: workspace too small", name);
    const void* const results[] = {a.h, a.dg, a.dn};
    for (const void* r : results) PSELD_CHECK_ARG(!r || (r != a.g && r != a.n && r != a.dh), "%s: a result must not be an operand", name);
    PSELD_CHECK_ARG(!a.dg || a.dg != a.dn, "%s: dg and dn must not be the same memory", name);
    a.slabs = (a.C + SLAB - 1) / SLAB;
    a.seg_len = seg_len_of(rows, max_len, a.C);
    a.nseg = max_len > a.seg_len ? (max_len + a.seg_len - 1) / a.seg_len : 1;
    PSELD_CHECK_ARG((long)a.slabs * a.nseg * a.seqs < (1l << 31), "%s: too many recordings x segments for one launch", name);
    if (dtype == PSELD_BF16) launch<bf16_t>(a, backward, (hipStream_t)stream);
    else launch<float>(a, backward, (hipStream_t)stream);
    PSELD_LAUNCH_CHECK(name);
    return PSELD_OK;
}
// rows of a result must not overlap
bool apart(long ld, long rows, int C) { return rows <= 1 || ld >= C; }
bool quads(const void* p, long ld, int dtype) { return ((uintptr_t)p & (dtype == PSELD_BF16 ? 7 : 15)) == 0 && (ld & 3) == 0 && ld >= 0 && ld < (1l << 23); }

}  // namespace

extern "C" long pseld_linrec_workspace(long rows, int seqs, int max_len, int C) {
    return rows > 0 && seqs > 0 && C > 0 ? agg_bytes_of(rows, seqs, max_len, C) : 0;
}
extern "C" long pseld_linrec_states(long rows, int seqs) { return rows / TILE + seqs + 1; }

extern "C" int pseld_linrec_fwd(int dtype, const void* g, long ldg, const void* n, long ldn, const float* h0, void* h, long ldh, float* h_last,
                                float* states, const int* start, const int* len, int seqs, long rows, int max_len, int C, int reverse,
                                float* workspace, long workspace_bytes, void* stream) {
    PSELD_CHECK_ARG(h_last && (rows == 0 || (g && n && h)), "linrec_fwd: null pointer");
    PSELD_CHECK_ARG(quads(g, ldg, dtype) && quads(n, ldn, dtype) && quads(h, ldh, dtype), "linrec_fwd: rows must start on 4-element boundaries, less than 2^23 elements apart");
    PSELD_CHECK_ARG(apart(ldh, rows, C), "linrec_fwd: the rows of h overlap");
    LinrecArgs a{};
    a.g = g; a.ldg = ldg; a.n = n; a.ldn = ldn; a.h0 = h0; a.h = h; a.ldh = ldh; a.h_last = h_last; a.states = states; a.agg = workspace;
    a.start = start; a.len = len; a.seqs = seqs; a.C = C; a.reverse = reverse;
    return go("linrec_fwd", dtype, a, rows, max_len, workspace, workspace_bytes, 0, stream);
}

extern "C" int pseld_linrec_bwd(int dtype, const void* dh, long lddh, const void* g, long ldg, const void* n, long ldn, const float* states,
                                const float* dh_last, void* dg, long lddg, void* dn, long lddn, float* dh0, const int* start, const int* len,
                                int seqs, long rows, int max_len, int C, int reverse, float* workspace, long workspace_bytes, void* stream) {
    PSELD_CHECK_ARG(rows == 0 || (dh && g && n && dg && dn && states), "linrec_bwd: null pointer");
    PSELD_CHECK_ARG(quads(dh, lddh, dtype) && quads(g, ldg, dtype) && quads(n, ldn, dtype) && quads(dg, lddg, dtype) && quads(dn, lddn, dtype),
                    "linrec_bwd: rows must start on 4-element boundaries, less than 2^23 elements apart");
    PSELD_CHECK_ARG(apart(lddg, rows, C) && apart(lddn, rows, C), "linrec_bwd: the rows of dg or dn overlap");
    LinrecArgs a{};
    a.dh = dh; a.lddh = lddh; a.g = g; a.ldg = ldg; a.n = n; a.ldn = ldn; a.states = const_cast<float*>(states); a.dlast = dh_last;
    a.dg = dg; a.lddg = lddg; a.dn = dn; a.lddn = lddn; a.dh0 = dh0; a.agg = workspace;
    a.start = start; a.len = len; a.seqs = seqs; a.C = C; a.reverse = reverse;
    return go("linrec_bwd", dtype, a, rows, max_len, workspace, workspace_bytes, 1, stream);
}
