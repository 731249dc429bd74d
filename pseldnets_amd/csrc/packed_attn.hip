// Attention over packed recordings, forward and backward, gfx950: recordings of different lengths back to back, causal or full, query heads that
// share key heads, a learned relative position bias by buckets, head sizes that are multiples of 8 up to 128, bf16 and f32.
//
//   S = scale q k^T + bias[bucket(key position - query position)],  P = softmax over the keys the mask leaves,  out = P v,  lse = log sum exp S
//   (a row that the mask leaves nothing: out 0, lse -inf).  Backward: delta = sum_j P dP (= sum_d dO O), dP = dO v^T, dS = P (dP - delta),
//   dq = scale dS k, dk = scale dS^T q (over the query heads that share the key head), dv = P^T dO, dtable[b] = sum of dS over the pairs of bucket b.
//
// No score matrix exists in HBM. Scores are computed TRANSPOSED in the forward and dq kernels (accumulator rows = keys, lanes = queries), so a
// query's maximum and sum are lane-local but for one exchange of the wave's halves, and the probabilities are the B operand of the second
// product as they stand; the dk/dv kernel has lanes = keys for the same reason. K / V (Q / dO) tiles of 64 rows reach LDS by LDS-DMA, into two
// buffers with one barrier per tile (dq with the table's gradient for heads above 32: one buffer, two barriers, dq_buffers); rows are lane-linear with their 16-byte pieces XOR-swizzled on the source address (image_swizzle),
// which leaves both the row reads and the transposed reads free of bank conflicts without padding. Rows past a recording's end are never
// addressed: the DMA repeats the last row and the mask drops it, so what a cache holds behind its length does not matter.
//
// bias: the table column of the workgroup's head is laid out by DISTANCE in LDS once (dist_fill); a tile whose distances are all at or past the
// last bucket adds one constant instead (it goes into the exponent's offset for free), the others read their diagonal's values.
// Its gradient: every wave sums its dS along the diagonals of a tile and adds them to LDS sums by distance, a copy per wave (add_diagonals): no two
// lanes of an instruction meet and the order of additions is fixed; sums per workgroup are folded to buckets, and a last launch adds the workgroups
// in order, in 64 bits.
// With bf16 operands O comes from rounded probabilities, so delta = dO O would be off by 2^-9 of itself - too coarse for the table's f32
// gradient, whose sums cancel. There delta = sum_j P dP is computed in its own pass over the keys (DELTA mode) from f32 P and dP.
#include "common.h"
#include "mma_frag.h"
#include <type_traits>

namespace {

constexpr int KT = 64;          // rows of a streamed tile
constexpr int WR = 32;          // rows of a wave's own tile
constexpr int TILE = 128;       // rows of a workgroup's own tile (four waves)
constexpr int NEAR_PAD = 96;    // a tile that touches a distance below max_distance has none past max_distance + KT + WR - 2
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

struct Strides { long rs, hs; };        // bytes between rows and between heads

struct PAttnArgs {
    const char *q, *k, *v, *dout, *o;
    char *out, *dq, *dk, *dv;
    Strides sq, sk, sv, so, sdo, sdq, sdk, sdv;
    float* lse;                 // [rows, hq]
    float* delta;               // [rows, hq]
    const int *q_start, *q_len, *k_start, *k_cap, *k_len, *tiles;
    int seqs, hq, hkv, D, causal;
    int nsplit, chunk;          // parts of a recording's keys and keys per part (few rows); of a key tile's query tiles and tiles per part (dk, dv)
    float scale, c;             // c = scale * log2(e)
    const float* table; const int* lut; const int* ranges;      // [buckets, hq]; bucket of distance -max .. max; [buckets, 2] first and last distance
    int buckets, maxd;
    float* part;                // dtable: [tiles, hq, buckets]; split dk/dv: [hkv, slots, 2, TILE, DP]; few rows: see there
    long slots;                 // dk, dv: parts reserved per key head; few rows: chunks
    int max_rows;               // few rows: rows reserved per key head
    int bias_heads;             // dk, dv: heads whose bias LDS has room for
};

// Two waves per SIMD where 256 registers hold a wave's accumulators and operands: the compiler then keeps the accumulators in vector registers
// (with more, it moves them to accumulation registers and back around every softmax). f32 operands of heads above 64 take the whole file.
template <typename T, int DP> constexpr int waves_per_simd() { return sizeof(T) == 2 || DP <= 64 ? 2 : 1; }

// ---- LDS images: rows of DP elements, lane-linear, 16-byte pieces swizzled inside the row ------------------------------------------
// What the XOR has to do (64 banks of 4 bytes): 16 rows that are read one 16-byte piece each (row_frag) must hit all 64 banks once, and so must 4 rows
// that are read 64 bytes each (half a wave of col_frag). With only 8 rows and 32 bytes apart every read took half as long again.
template <int RB, int E> __device__ __forceinline__ int image_swizzle(int row) {
    if constexpr (RB == 64) return (row >> 2) & 3;                                             // four rows span the banks
    else if constexpr (RB == 128) return (((row >> 1) & 1) << 2) | ((row >> 2) & 3);           // two
    else if constexpr (E == 2) return ((row & 3) << 2) | ((row >> 2) & 3);
    else return (((row >> 2) & 1) << 3) | ((row & 3) << 1) | ((row >> 3) & 1);                 // f32 columns: rows 4 apart, 128 bytes each
}
typedef __attribute__((address_space(3))) const char* lds_cptr;
// A lane's reads of an image. The swizzle only XORs bits inside a row, so a lane keeps three offsets for the tile at hand and reaches every piece by
// XOR with a constant and the instruction's immediate. move<true> hides the offsets from loop-invariant motion: where the accumulators fill the
// register file, the hoisted XORs spill (60 registers in the dk/dv kernel for 128); elsewhere hoisting them is faster (forward for 128: 10 %).
template <typename T, int DP> struct Image {
    static constexpr int RB = DP * (int)sizeof(T);
    using M = AMma<T>;
    using Frag = typename M::Frag;
    struct Lane { unsigned row, lo, hi; };
    static __device__ __forceinline__ Lane lane_offsets(int lane) {
        const int r = lane & 31, h2 = lane >> 5;
        Lane l;
        if constexpr (sizeof(T) == 2) {
            const int ra = 4 * h2 + ((lane & 15) >> 2), rb = ra + 8, p = lane & 3, ch = 2 * ((lane >> 4) & 1) + (p >> 1);
            l.row = r * RB + ((h2 ^ image_swizzle<RB, (int)sizeof(T)>(r)) << 4);
            l.lo = ra * RB + ((ch ^ image_swizzle<RB, (int)sizeof(T)>(ra)) << 4) + (p & 1) * 8;
            l.hi = rb * RB + ((ch ^ image_swizzle<RB, (int)sizeof(T)>(rb)) << 4) + (p & 1) * 8;
        } else {
            l.row = r * RB + (((2 * h2) ^ image_swizzle<RB, (int)sizeof(T)>(r)) << 4);
            l.lo = l.hi = 0;
        }
        return l;
    }
    template <bool HIDE> static __device__ __forceinline__ void move(Lane& l, unsigned by) {
        l.row += by;
        l.lo += by;
        if constexpr (sizeof(T) == 2) l.hi += by;
        if constexpr (HIDE) asm volatile("" : "+v"(l.row), "+v"(l.lo));
        if constexpr (HIDE && sizeof(T) == 2) asm volatile("" : "+v"(l.hi));
    }
    static __device__ __forceinline__ Lane at(Lane l, unsigned tile) { move<false>(l, tile); return l; }
    // elements 16 kk + 8 h2 .. + 7 of image row 32 t + (lane & 31); off: bytes from the tile that l stands for (a multiple of 1024)
    static __device__ __forceinline__ Frag row_frag(const Lane& l, int t, int kk, int off = 0) {
        if constexpr (sizeof(T) == 2) return *(const __attribute__((address_space(3))) bf16x8*)(lds_cptr)(uintptr_t)((l.row ^ (kk << 5)) + t * 32 * RB + off);
        else {
            const f32x4 a = *(const __attribute__((address_space(3))) f32x4*)(lds_cptr)(uintptr_t)((l.row ^ (kk << 6)) + t * 32 * RB + off);
            const f32x4 b = *(const __attribute__((address_space(3))) f32x4*)(lds_cptr)(uintptr_t)((l.row ^ (kk << 6) ^ 16) + t * 32 * RB + off);
            Frag x;
#pragma unroll
            for (int j = 0; j < 4; ++j) { x.v[j] = a[j]; x.v[4 + j] = b[j]; }
            return x;
        }
    }
    // element j = M[row0 + 8 (j >> 2) + 4 h2 + (j & 3)][32 dt + (lane & 31)], the k order of an accumulator operand; row0 a multiple of 16
    static __device__ __forceinline__ Frag col_frag(const Lane& l, int row0, int dt, int lane, int off = 0) {
        if constexpr (sizeof(T) == 2) {
            const short4v lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4_ptr)(lds_cptr)(uintptr_t)((l.lo ^ (dt << 6)) + row0 * RB + off));
            const short4v hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4_ptr)(lds_cptr)(uintptr_t)((l.hi ^ (dt << 6)) + row0 * RB + off));
            short8v s;
            s[0] = lo[0]; s[1] = lo[1]; s[2] = lo[2]; s[3] = lo[3];
            s[4] = hi[0]; s[5] = hi[1]; s[6] = hi[2]; s[7] = hi[3];
            return __builtin_bit_cast(bf16x8, s);
        } else {
            const int col = 32 * dt + (lane & 31), h2 = lane >> 5;
            Frag x;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int row = row0 + 8 * (j >> 2) + 4 * h2 + (j & 3);
                x.v[j] = *(const __attribute__((address_space(3))) float*)(lds_cptr)(uintptr_t)(l.lo + row * RB + (((col >> 2) ^ image_swizzle<RB, (int)sizeof(T)>(row)) << 4) + (col & 3) * 4 + off);
            }
            return x;
        }
    }
};
// the wave's operand rows straight from global memory: 8 elements at 16 kk + 8 h2 of the lane's row, zeros past the head's size
template <typename T, int DP>
__device__ __forceinline__ typename AMma<T>::Frag global_frag(const char* row, int kk, int h2, int D) {
    typename AMma<T>::Frag f;
    const int d = 16 * kk + 8 * h2;
    if constexpr (sizeof(T) == 2) {
        f32x4 v = {0.f, 0.f, 0.f, 0.f};
        if (d < D) v = *(const f32x4*)(row + d * 2);
        f = __builtin_bit_cast(bf16x8, v);
    } else {
        f32x4 x = {0.f, 0.f, 0.f, 0.f}, y = x;
        if (d < D) { x = *(const f32x4*)(row + d * 4); y = *(const f32x4*)(row + d * 4 + 16); }
#pragma unroll
        for (int j = 0; j < 4; ++j) { f.v[j] = x[j]; f.v[4 + j] = y[j]; }
    }
    return f;
}

// one LDS-DMA wave-instruction: 64 lanes x 16 B from (uniform base + per-lane 32-bit offset) to 1 KiB of LDS at a uniform address.
// Inline asm, its waits counted by hand: the compiler would drain it in front of every fragment read.
__device__ __forceinline__ void pa_dma(unsigned lds_dst, const void* sbase, unsigned voff) {
    unsigned keep;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %3\n\ts_mov_b32 m0, %0"
                 : "=&s"(keep) : "v"(voff), "s"(lds_dst), "s"(sbase) : "memory");
}
__device__ __forceinline__ const char* uniform_ptr(const char* p) {
    const unsigned long long v = (unsigned long long)p;
    const unsigned lo = __builtin_amdgcn_readfirstlane((unsigned)v), hi = __builtin_amdgcn_readfirstlane((unsigned)(v >> 32));
    return (const char*)(((unsigned long long)hi << 32) | lo);
}
__device__ __forceinline__ unsigned lds_addr(const void* p) { return (unsigned)(unsigned long long)(__attribute__((address_space(3))) const char*)p; }

// Every ordinary load has landed, as a wait that the compiler's own bookkeeping sees (gfx9 encoding: vmcnt 0, expcnt 7, lgkmcnt 15). In front of each loop
// that keeps DMAs in flight: without it the compiler waits for the operands loaded before the loop INSIDE it, at every turn, and drains the next
// tile's DMA right after its request.
#define PA_LOADS_DONE() __builtin_amdgcn_s_waitcnt(0x0F70)
#define PA_SYNC_TILE()                                                  \
    do {                                                                \
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");     \
        __builtin_amdgcn_sched_barrier(0);                              \
        __builtin_amdgcn_s_barrier();                                   \
        __builtin_amdgcn_sched_barrier(0);                              \
        asm volatile("" ::: "memory");                                  \
    } while (0)

// A stream of ROWS-row tiles of one operand into LDS by NW waves. The swizzle repeats after NP instructions, so NP lane offsets serve a whole
// tile and the rest is added to the uniform base. A tile that ends inside takes its rows past the end from the last one. LAZY: the offsets are
// computed anew for every tile (where registers are short: spilled, each one's reload waits behind the DMAs already in flight).
template <typename T, int DP, int ROWS, int NW, bool LAZY = false> struct Stream {
    static constexpr int RB = DP * (int)sizeof(T);
    static constexpr int NI = ROWS * RB / 1024 / NW;       // wave-instructions per wave
    static constexpr int RPI = 1024 / RB;                  // rows per instruction
    static constexpr int NP = 16 / RPI;                    // the swizzle repeats after 16 rows
    static_assert(NI >= NP && NI % NP == 0 && NI * NW * 1024 == ROWS * RB, "whole swizzle periods per wave");
    unsigned voff[LAZY ? 1 : NP];
    unsigned rs;
    int wave, pieces;
    __device__ __forceinline__ unsigned offset(int lane, int row0, int limit) const {
        const int row = row0 + lane * 16 / RB;
        return (unsigned)min(row, limit) * rs + (unsigned)min(((lane * 16 % RB) >> 4) ^ image_swizzle<RB, (int)sizeof(T)>(row), pieces - 1) * 16;
    }
    __device__ __forceinline__ void init(long row_bytes, int D, int w) {
        wave = w; rs = (unsigned)row_bytes; pieces = D * (int)sizeof(T) / 16;
        if constexpr (!LAZY)
#pragma unroll
            for (int j = 0; j < NP; ++j) voff[j] = offset(threadIdx.x & 63, j * RPI, ROWS);
    }
    // base: first row of the tile (uniform); rows: rows that exist from there on (> 0)
    __device__ __forceinline__ void load(const char* base, int rows, unsigned lds) const {
        const unsigned dst = __builtin_amdgcn_readfirstlane(lds + wave * NI * 1024);
        int lane = threadIdx.x & 63;
        if constexpr (LAZY) asm volatile("" : "+v"(lane));
        if (rows >= ROWS) {
            const char* b = uniform_ptr(base + (long)(wave * NI * RPI) * rs);
#pragma unroll
            for (int j = 0; j < NI; ++j) pa_dma(dst + j * 1024, b + (long)(j / NP * NP * RPI) * rs, LAZY ? offset(lane, j % NP * RPI, ROWS) : voff[LAZY ? 0 : j % NP]);
        } else {
            const char* b = uniform_ptr(base);
#pragma unroll
            for (int j = 0; j < NI; ++j) pa_dma(dst + j * 1024, b, offset(lane, (wave * NI + j) * RPI, rows - 1));
        }
    }
};

// ---- relative position bias by distance ---------------------------------------------------------------------------------------------
__device__ __forceinline__ int dist_count(int maxd) { return 2 * (maxd + NEAR_PAD) + 1; }
__device__ __forceinline__ float bias_at(const PAttnArgs& a, int rel, int head) {
    const int r = max(-a.maxd, min(a.maxd, rel));
    return a.table[(long)a.lut[r + a.maxd] * a.hq + head];
}
// The bias of one head by distance, laid out in LDS: dist[i] = bias of distance i - maxd - NEAR_PAD over the scale, in units of the raw products, whose
// accumulators start from it. ask / look / put are the three steps of a chain of dependent reads (lut, table, LDS), so that a kernel can put
// its other requests between them: ask needs nothing but the arguments. The first 512 distances go that way, the rest in a loop.
struct Dist {
    int n, b[2], b_lo, b_hi;
    float v[2], lo, hi;
    __device__ __forceinline__ void ask(const PAttnArgs& a) {
        n = dist_count(a.maxd);
#pragma unroll
        for (int j = 0; j < 2; ++j) b[j] = a.lut[max(0, min(2 * a.maxd, (int)threadIdx.x + 256 * j - NEAR_PAD))];
        b_lo = a.lut[0];
        b_hi = a.lut[2 * a.maxd];
    }
    __device__ __forceinline__ void look(const PAttnArgs& a, int head) {
#pragma unroll
        for (int j = 0; j < 2; ++j) v[j] = a.table[(long)b[j] * a.hq + head];
        lo = a.table[(long)b_lo * a.hq + head];
        hi = a.table[(long)b_hi * a.hq + head];
    }
    __device__ __forceinline__ void put(float* dist, const PAttnArgs& a, int head) const {
        const float inv = 1.f / a.scale;
#pragma unroll
        for (int j = 0; j < 2; ++j) if ((int)threadIdx.x + 256 * j < n) dist[threadIdx.x + 256 * j] = v[j] * inv;
        for (int i = threadIdx.x + 512; i < n; i += 256) dist[i] = bias_at(a, i - a.maxd - NEAR_PAD, head) * inv;
    }
    // the first and the last bucket's bias in log2 units, in scalar registers
    __device__ __forceinline__ float far(float x) const { return __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, x * LOG2E))); }
};

// the whole layout in one loop: where a head changes amid a kernel's tiles
__device__ __forceinline__ void dist_fill(float* dist, const PAttnArgs& a, int head) {
    const int n = dist_count(a.maxd);
    const float inv = 1.f / a.scale;
    for (int i = threadIdx.x; i < n; i += 256) dist[i] = bias_at(a, i - a.maxd - NEAR_PAD, head) * inv;
}

// Keeps the scheduler from requesting a whole product's operands at once where the accumulators leave no registers for them
template <bool TIGHT> __device__ __forceinline__ void pace() {
    if constexpr (TIGHT) __builtin_amdgcn_sched_barrier(0);
}
template <int N> __device__ __forceinline__ void zero_acc(f32x16 (&z)[N]) {
#pragma unroll
    for (int t = 0; t < N; ++t)
#pragma unroll
        for (int e = 0; e < 16; ++e) z[t][e] = 0.f;
}
__device__ __forceinline__ float half_swap_max(float v) { return fmaxf(v, __shfl_xor(v, 32, 64)); }

// a transposed result z (rows = d in registers, lane & 31 = row of the output) x mul -> global rows. bf16: the halves trade 4-element pieces so that
// a lane stores 16 bytes
template <typename T, int DP>
__device__ __forceinline__ void store_rows(char* row, bool live, const f32x16 (&z)[DP / 32], float mul, int D, int h2) {
#pragma unroll
    for (int dt = 0; dt < DP / 32; ++dt) {
        if constexpr (sizeof(T) == 2) {
#pragma unroll
            for (int g = 0; g < 4; g += 2) {
                unsigned pc[2][2];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    bf16x2 lo, hi;
                    lo[0] = (bf16_t)(z[dt][4 * (g + i)] * mul); lo[1] = (bf16_t)(z[dt][4 * (g + i) + 1] * mul);
                    hi[0] = (bf16_t)(z[dt][4 * (g + i) + 2] * mul); hi[1] = (bf16_t)(z[dt][4 * (g + i) + 3] * mul);
                    pc[i][0] = __builtin_bit_cast(unsigned, lo); pc[i][1] = __builtin_bit_cast(unsigned, hi);
                }
                // half 0 keeps its piece g and takes the other half's piece g, half 1 its piece g + 1 and half 0's piece g + 1
                const auto a = __builtin_amdgcn_permlane32_swap(pc[0][0], pc[1][0], false, false);
                const auto b = __builtin_amdgcn_permlane32_swap(pc[0][1], pc[1][1], false, false);
                const int d = dt * 32 + 8 * (g + h2);
                typedef __attribute__((ext_vector_type(4))) unsigned u32x4;
                if (live && d < D) *(u32x4*)(row + d * 2) = u32x4{a[0], b[0], a[1], b[1]};
            }
        } else {
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int d = dt * 32 + 8 * g + 4 * h2;
                if (live && d < D) *(f32x4*)(row + d * 4) = f32x4{z[dt][4 * g] * mul, z[dt][4 * g + 1] * mul, z[dt][4 * g + 2] * mul, z[dt][4 * g + 3] * mul};
            }
        }
    }
}

// z (rows = d) += M[tile rows][d]^T x, x = accumulator tiles whose rows are the image's rows 32 t0 ..
template <typename T, int DP, int NT, bool TIGHT = false>
__device__ __forceinline__ void acc_product(f32x16 (&z)[DP / 32], const f32x16 (&x)[NT], const typename Image<T, DP>::Lane& l, int t0, int lane, int off) {
    using I = Image<T, DP>;
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const typename I::Frag fx = I::M::from_acc(x[t], s);
#pragma unroll
            for (int dt = 0; dt < DP / 32; ++dt) I::M::mma(I::col_frag(l, (t0 + t) * 32 + 16 * s, dt, lane, off), fx, z[dt]);
            pace<TIGHT>();
        }
}

// The running maximum, sum and output of a wave's 32 queries (lane & 31), keys in accumulator rows.
template <int DP> struct Softmax {
    f32x16 ot[DP / 32];
    float m, l;                 // log2 units; l holds the lane half's own keys
    __device__ __forceinline__ void init() { zero_acc(ot); m = -__builtin_inff(); l = 0.f; }
    // x: raw products; score = x * c + off. The maximum may lag by up to 2^8 (the sums are f32, the probabilities keep their relative
    // rounding), so most tiles do not touch the output accumulators.
    template <int NT> __device__ __forceinline__ void step(f32x16 (&x)[NT], float c, float off) {
        float mx = -__builtin_inff();
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int e = 0; e < 16; ++e) mx = fmaxf(mx, x[t][e]);
        mx = half_swap_max(mx);
        mx = fmaf(mx, c, off);
        if (__any(mx > m + 8.f)) {
            const float mn = fmaxf(m, mx);
            const float alpha = mn == m ? 1.f : __builtin_amdgcn_exp2f(m - mn);
            m = mn;
            l *= alpha;
#pragma unroll
            for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
                for (int e = 0; e < 16; ++e) ot[dt][e] *= alpha;
        }
        const float sub = off - (m == -__builtin_inff() ? 0.f : m);
        float ps = 0.f;
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const float p = __builtin_amdgcn_exp2f(fmaf(x[t][e], c, sub));
                x[t][e] = p;
                ps += p;
            }
        l += ps;
    }
};

// A row's sum is 0 only where it has no keys (or -inf scores alone); a NaN goes on into out and lse
__device__ __forceinline__ float inverse(float l) { return l == 0.f ? 0.f : 1.f / l; }
__device__ __forceinline__ float lse_of(float m, float l) { return l == 0.f ? -__builtin_inff() : (m + __log2f(l)) * LN2; }

// Where a tile's scores start: from their diagonals' bias; d points at the entry of (accumulator row 0, this lane's column)
template <int NT, int SIGN> __device__ __forceinline__ void start_near(f32x16 (&x)[NT], const float* d) {
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 16; ++e) x[t][e] = d[SIGN * (t * 32 + (e & 3) + 8 * (e >> 2))];
}
// A tile's distances lo .. hi: all at or past -maxd / maxd (one bias for the whole tile), or near
enum { FAR_LO = -1, NEAR = 0, FAR_HI = 1 };
__device__ __forceinline__ int place_of(int lo, int hi, int maxd) { return hi <= -maxd ? FAR_LO : lo >= maxd ? FAR_HI : NEAR; }
// keeps rows <= lim (rows counted from the tile's first, lim already less 4 * (lane >> 5))
template <int NT> __device__ __forceinline__ void mask_rows(f32x16 (&x)[NT], int lim, float with) {
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 16; ++e) x[t][e] = (t * 32 + (e & 3) + 8 * (e >> 2)) <= lim ? x[t][e] : with;
}

// which recording, rows and head a workgroup of the query-tiled kernels owns. Heads fastest, the query heads of one key head a multiple of
// hkv apart: with hkv a multiple of the eight XCDs every key head's tiles stay on one XCD's L2
// f32 (the parity mode): an f32 matrix instruction takes 64 cycles and short recordings leave few waves, so the four waves are two groups of 32
// rows x two halves of every key tile, joined through LDS at the end: half the rows per workgroup, half the time per tile (6 recordings of 30-600,
// 8 heads of 64: forward 63 -> 43 us). bf16 tiles are too short for it (12 x 100-1200, 16 heads of 64, causal: forward 34 -> 40 us)
template <typename T> constexpr int key_split() { return sizeof(T) == 4 ? 2 : 1; }
struct QTile {
    int seq, q0, q_len, k_len, off, head, kvh, nk;
    long q_row, k_row;
};
template <int KS> __device__ __forceinline__ QTile q_tile_of(const PAttnArgs& a) {
    QTile t;
    const int p = blockIdx.x % a.hq, ti = blockIdx.x / a.hq / KS;
    t.kvh = p % a.hkv;
    t.head = t.kvh * (a.hq / a.hkv) + p / a.hkv;
    const int* rec = a.tiles + 8 * (long)ti;               // one load for all that is fixed: the chain to the first key row is two loads long
    t.seq = rec[0];
    t.q0 = rec[1] + blockIdx.x / a.hq % KS * (TILE / KS);
    t.q_row = rec[2];
    t.q_len = rec[3];
    t.k_row = rec[4];
    t.k_len = max(0, min(a.k_len[t.seq], rec[5]));
    t.off = t.k_len - t.q_len;
    t.nk = t.q0 >= t.q_len ? 0 : a.causal ? max(0, min(t.k_len, t.q0 + TILE / KS + t.off)) : t.k_len;
    return t;
}

// ---- forward: 128 queries of one (recording, head), a wave 32 --------------------------------------------------------------------------
template <typename T, int DP, bool BIAS>
__global__ __launch_bounds__(256, (waves_per_simd<T, DP>())) void packed_attn_fwd_kernel(PAttnArgs a) {
    using I = Image<T, DP>;
    constexpr int TB = KT * I::RB, KS = key_split<T>(), KW = KT / KS, NT = 2 / KS;
    extern __shared__ __attribute__((aligned(1024))) char smem[];      // 2 x (K tile | V tile) | bias by distance
    float* dist = (float*)(smem + 4 * TB);
    Dist bias;
    if constexpr (BIAS) bias.ask(a);
    const QTile w = q_tile_of<KS>(a);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 31, h2 = lane >> 5;
    const int rg = wave % (4 / KS), kh = wave / (4 / KS);       // the wave's rows and its part of every key tile
    const int qi = w.q0 + rg * WR + r;
    const bool live = qi < w.q_len;
    const long qrow = w.q_row + min(qi, w.q_len - 1);
    const char* kb = a.k + w.k_row * a.sk.rs + (long)w.kvh * a.sk.hs;
    const char* vb = a.v + w.k_row * a.sv.rs + (long)w.kvh * a.sv.hs;
    Stream<T, DP, KT, 4> ks, vs;
    ks.init(a.sk.rs, a.D, wave);
    vs.init(a.sv.rs, a.D, wave);
    const unsigned lds0 = lds_addr(smem);
    const typename I::Lane im0 = I::lane_offsets(lane);
    const int nt = (w.nk + KT - 1) / KT;
    if constexpr (BIAS) bias.look(a, w.head);
    if (nt) { ks.load(kb, w.k_len, lds0); vs.load(vb, w.k_len, lds0 + TB); }
    typename I::Frag fq[DP / 16];
    {
        const char* row = a.q + qrow * a.sq.rs + (long)w.head * a.sq.hs;
#pragma unroll
        for (int kk = 0; kk < DP / 16; ++kk) fq[kk] = global_frag<T, DP>(row, kk, h2, a.D);
    }
    const int qpos = qi + w.off, qw0 = w.q0 + rg * WR + w.off;        // the lane's and the wave's first query position
    const int klim = a.causal ? min(w.k_len - 1, qpos) : w.k_len - 1;
    const int wlim0 = a.causal ? min(w.k_len - 1, qw0) : w.k_len - 1;   // every query of the wave sees keys up to here,
    const int wlim1 = w.q0 + rg * WR >= w.q_len ? -1 : a.causal ? min(w.k_len - 1, qw0 + WR - 1) : w.k_len - 1;     // none sees one past here
    float far_lo = 0.f, far_hi = 0.f;
    if constexpr (BIAS) { bias.put(dist, a, w.head); far_lo = bias.far(bias.lo); far_hi = bias.far(bias.hi); }
    Softmax<DP> sm;
    sm.init();
    PA_LOADS_DONE();
    for (int i = 0; i < nt; ++i) {
        const int k0 = i * KT;
        PA_SYNC_TILE();
        if (i + 1 < nt) {
            const unsigned dst = lds0 + ((i + 1) & 1) * 2 * TB;
            ks.load(kb + (long)(k0 + KT) * a.sk.rs, w.k_len - k0 - KT, dst);
            vs.load(vb + (long)(k0 + KT) * a.sv.rs, w.k_len - k0 - KT, dst + TB);
        }
        const int kt0 = k0 + kh * KW;                      // the wave's first key of the tile
        if (kt0 > wlim1) continue;
        const typename I::Lane im = I::at(im0, lds0 + kh * KW * I::RB + (i & 1) * 2 * TB);
        f32x16 st[NT];
        zero_acc(st);
        float off = 0.f;
        if constexpr (BIAS) {
            const int place = place_of(kt0 - (qw0 + WR - 1), kt0 + KW - 1 - qw0, a.maxd);
            if (place == NEAR) start_near<NT, 1>(st, dist + (kt0 + 4 * h2 - qpos + a.maxd + NEAR_PAD));
            else off = place < 0 ? far_lo : far_hi;
        }
#pragma unroll
        for (int kk = 0; kk < DP / 16; ++kk)
#pragma unroll
            for (int t = 0; t < NT; ++t) I::M::mma(I::row_frag(im, t, kk), fq[kk], st[t]);
        if constexpr (DP == 128 && sizeof(T) == 2) {       // four reads ahead of the products: two waves per SIMD do not cover an LDS read (668 -> 601 us)
            __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
#pragma unroll
            for (int kk = 0; kk < DP / 8; ++kk) {
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
            }
        }
        if (kt0 + KW - 1 > wlim0) mask_rows<NT>(st, klim - kt0 - 4 * h2, -__builtin_inff());
        sm.template step<NT>(st, a.c, off);
        acc_product<T, DP, NT>(sm.ot, st, im, 0, lane, TB);
    }
    if constexpr (KS > 1) {                                // the second half's waves hand over their maxima, sums and outputs, a register per row of 64 lanes
        float* x = (float*)smem + rg * (DP / 2 + 2) * 64 + lane;
        __syncthreads();
        if (kh) {
#pragma unroll
            for (int e = 0; e < DP / 2; ++e) x[e * 64] = sm.ot[e >> 4][e & 15];
            x[DP / 2 * 64] = sm.m;
            x[(DP / 2 + 1) * 64] = sm.l;
        }
        __syncthreads();
        if (kh) return;
        const float m2 = x[DP / 2 * 64], mn = fmaxf(sm.m, m2);
        const float f1 = sm.m == mn ? 1.f : __builtin_amdgcn_exp2f(sm.m - mn), f2 = m2 == mn ? 1.f : __builtin_amdgcn_exp2f(m2 - mn);
#pragma unroll
        for (int e = 0; e < DP / 2; ++e) sm.ot[e >> 4][e & 15] = fmaf(sm.ot[e >> 4][e & 15], f1, x[e * 64] * f2);
        sm.l = sm.l * f1 + x[(DP / 2 + 1) * 64] * f2;
        sm.m = mn;
    }
    const float l = sm.l + __shfl_xor(sm.l, 32, 64);
    store_rows<T, DP>(a.out + qrow * a.so.rs + (long)w.head * a.so.hs, live, sm.ot, inverse(l), a.D, h2);
    if (live && h2 == 0) a.lse[qrow * a.hq + w.head] = lse_of(sm.m, l);
}

// ---- few rows: a step of running streams ------------------------------------------------------------------------------------------------
// A recording's q_len x (hq / hkv) rows of one key head fit one 32-row operand. A workgroup takes `chunk` keys of one (recording, key head), its
// waves 32-key blocks in turn; a wave streams its own blocks through its own LDS (no barrier in the loop) and the waves' maxima, sums
// and outputs are joined through LDS. More than one chunk per recording: f32 partials and a joining launch, both in a fixed order. HBM
// bound: K and V are read once for all rows that share them.
// The place of a recording's first chunk: slabs lie one behind the other, so those before this one, of k_start rows together, take the sum of ceil(capacity / chunk)
// places, which floor(k_start / chunk) + their number is never less than.
__device__ __forceinline__ long few_slot(const PAttnArgs& a, int seq, int kvh) { return kvh * a.slots + (unsigned)a.k_start[seq] / (unsigned)a.chunk + seq; }
template <typename T, int DP, int NW, bool BIAS>
__global__ __launch_bounds__(64 * NW) void packed_attn_few_kernel(PAttnArgs a) {
    using I = Image<T, DP>;
    constexpr int BB = WR * I::RB;                         // one block of K or V
    extern __shared__ __attribute__((aligned(1024))) char smem[];      // waves x 2 x (K | V) | (waves + 1) x 32 x (m, l) | table | lut
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 31, h2 = lane >> 5;
    const int kvh = blockIdx.x % a.hkv, rest = blockIdx.x / a.hkv, split = rest % a.nsplit, seq = rest / a.nsplit;
    const int G = a.hq / a.hkv, q_len = a.q_len[seq];
    const int k_len = max(0, min(a.k_len[seq], a.k_cap[seq])), rows = q_len * G;
    const int kbeg = split * a.chunk, kend = min(k_len, kbeg + a.chunk);
    if (rows == 0 || (kbeg >= k_len && split)) return;     // chunk 0 answers for a recording without keys
    float* ml = (float*)(smem + NW * 4 * BB);
    float* all = ml + NW * 64;                             // the waves' joined (m, l)
    float* tab = all + 64;
    unsigned short* lut = (unsigned short*)(tab + a.buckets * G);
    const char* kb = a.k + (long)a.k_start[seq] * a.sk.rs + (long)kvh * a.sk.hs;
    const char* vb = a.v + (long)a.k_start[seq] * a.sv.rs + (long)kvh * a.sv.hs;
    Stream<T, DP, WR, 1> ks, vs;
    ks.init(a.sk.rs, a.D, 0);
    vs.init(a.sv.rs, a.D, 0);
    char* mine = smem + wave * 4 * BB;
    const unsigned lds0 = lds_addr(mine);
    const typename I::Lane im0 = I::lane_offsets(lane);
    const int first = kbeg + wave * WR;                    // the first block is on its way before anything else is read
    if (first < kend) { ks.load(kb + (long)first * a.sk.rs, k_len - first, lds0); vs.load(vb + (long)first * a.sv.rs, k_len - first, lds0 + BB); }
    const int off = k_len - q_len;
    const int rr = min(r, rows - 1), qi = rr / G, g = rr - qi * G;
    const long qrow = (long)a.q_start[seq] + qi;
    typename I::Frag fq[DP / 16];
    {
        const char* row = a.q + qrow * a.sq.rs + (long)(kvh * G + g) * a.sq.hs;
#pragma unroll
        for (int kk = 0; kk < DP / 16; ++kk) fq[kk] = global_frag<T, DP>(row, kk, h2, a.D);
    }
    if constexpr (BIAS) {
        if (kend - 1 - off > -a.maxd) {                    // some key is near some query
            for (int i = threadIdx.x; i < a.buckets * G; i += 64 * NW) tab[i] = a.table[(long)(i / G) * a.hq + kvh * G + i % G] / a.scale;
            for (int i = threadIdx.x; i <= 2 * a.maxd; i += 64 * NW) lut[i] = (unsigned short)a.lut[i];
        }
        __syncthreads();
    }
    const int qpos = qi + off, klim = a.causal ? min(k_len - 1, qpos) : k_len - 1;
    float far_lo = 0.f, far_hi = 0.f;
    if constexpr (BIAS) { far_lo = bias_at(a, -a.maxd, kvh * G + g) * LOG2E; far_hi = bias_at(a, a.maxd, kvh * G + g) * LOG2E; }
    Softmax<DP> sm;
    sm.init();
    PA_LOADS_DONE();
    int par = 0;
    for (int k0 = first; k0 < kend; k0 += NW * WR, par ^= 1) {
        const int nx = k0 + NW * WR;
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); // the last block's reads are done with the buffer that is filled next
        if (nx < kend) {
            const unsigned dst = lds0 + (par ^ 1) * 2 * BB;
            ks.load(kb + (long)nx * a.sk.rs, k_len - nx, dst);
            vs.load(vb + (long)nx * a.sv.rs, k_len - nx, dst + BB);
            asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * Stream<T, DP, WR, 1>::NI) : "memory");      // all but the block just requested
        } else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
        const typename I::Lane im = I::at(im0, lds0 + par * 2 * BB);
        f32x16 st[1];
        zero_acc(st);
        float o = 0.f;
        if constexpr (BIAS) {
            const int place = place_of(k0 - (k_len - 1), min(k0 + WR, kend) - 1 - off, a.maxd);      // over every query of the recording
            if (place == NEAR) {
                const int base = k0 + 4 * h2 - qpos + a.maxd;
#pragma unroll
                for (int e = 0; e < 16; ++e) st[0][e] = tab[lut[max(0, min(2 * a.maxd, base + (e & 3) + 8 * (e >> 2)))] * G + g];
            } else o = place < 0 ? far_lo : far_hi;
        }
#pragma unroll
        for (int kk = 0; kk < DP / 16; ++kk) I::M::mma(I::row_frag(im, 0, kk), fq[kk], st[0]);
        if (a.causal ? k0 + WR - 1 > min(k_len - 1, off) || k0 + WR > kend : k0 + WR > kend) mask_rows<1>(st, min(klim, kend - 1) - k0 - 4 * h2, -__builtin_inff());
        sm.template step<1>(st, a.c, o);
        acc_product<T, DP, 1>(sm.ot, st, im, 0, lane, BB);
    }
    // join the waves
    const float l = sm.l + __shfl_xor(sm.l, 32, 64);
    if (h2 == 0) { ml[wave * 64 + r] = sm.m; ml[wave * 64 + 32 + r] = l; }
    __syncthreads();
    float mt = -__builtin_inff(), lt = 0.f;
#pragma unroll
    for (int x = 0; x < NW; ++x) mt = fmaxf(mt, ml[x * 64 + r]);
#pragma unroll
    for (int x = 0; x < NW; ++x) { const float mx = ml[x * 64 + r]; lt += ml[x * 64 + 32 + r] * (mx == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(mx - mt)); }
    const float f = sm.m == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(sm.m - mt);
    constexpr int PITCH = DP + 4;                          // floats per row of a wave's output image: 32 rows of 4-float pieces fall in different banks
    static_assert(32 * PITCH * 4 <= 4 * BB, "the output image fits the wave's buffers");
    float* oi = (float*)mine;
#pragma unroll
    for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
        for (int gg = 0; gg < 4; ++gg)
            *(f32x4*)(oi + r * PITCH + dt * 32 + 8 * gg + 4 * h2) = f32x4{sm.ot[dt][4 * gg] * f, sm.ot[dt][4 * gg + 1] * f, sm.ot[dt][4 * gg + 2] * f, sm.ot[dt][4 * gg + 3] * f};
    if (wave == 0 && h2 == 0) { all[r] = mt; all[32 + r] = lt; }
    __syncthreads();
    const long pslot = (few_slot(a, seq, kvh) + split) * a.max_rows;
    for (int i = threadIdx.x; i < rows * (a.D / 4); i += 64 * NW) {
        const int row = i / (a.D / 4), d = (i - row * (a.D / 4)) * 4;
        f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int x = 0; x < NW; ++x) s += *(const f32x4*)((const float*)(smem + x * 4 * BB) + row * PITCH + d);
        const float m = all[row], lr = all[32 + row];
        if (a.nsplit > 1) {
            float* p = a.part + (pslot + row) * (a.D + 4);
            *(f32x4*)(p + 4 + d) = s;
            if (d == 0) { p[0] = m; p[1] = lr; }
        } else {
            const int qj = row / G, head = kvh * G + row - qj * G;
            const long qr = (long)a.q_start[seq] + qj;
            const float inv = inverse(lr);
            store4<T>(a.out + qr * a.so.rs + (long)head * a.so.hs + d * (int)sizeof(T), s[0] * inv, s[1] * inv, s[2] * inv, s[3] * inv);
            if (d == 0) a.lse[qr * a.hq + head] = lse_of(m, lr);
        }
    }
}
// one wave joins the chunks of one (row, head): weights from the chunks' maxima and sums, then a weighted sum in chunk order
template <typename T>
__global__ __launch_bounds__(64) void packed_attn_join_kernel(PAttnArgs a) {
    extern __shared__ float wgt[];
    const int G = a.hq / a.hkv, lane = threadIdx.x;
    const int row = blockIdx.x % a.max_rows, rest = blockIdx.x / a.max_rows, kvh = rest % a.hkv, seq = rest / a.hkv;
    if (row >= a.q_len[seq] * G) return;
    const int k_len = max(0, min(a.k_len[seq], a.k_cap[seq]));
    const int n = max(1, (k_len + a.chunk - 1) / a.chunk);
    const float* p = a.part + (few_slot(a, seq, kvh) * a.max_rows + row) * (a.D + 4);
    const long step = (long)a.max_rows * (a.D + 4);
    float m = -__builtin_inff();
    for (int i = lane; i < n; i += 64) m = fmaxf(m, p[i * step]);
    m = wave_max(m);
    float l = 0.f;
    for (int i = lane; i < n; i += 64) {
        const float mi = p[i * step], w = mi == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(mi - m);
        wgt[i] = w;
        l += w * p[i * step + 1];
    }
    l = wave_sum(l);
    __syncthreads();
    const float inv = inverse(l);
    const int qj = row / G, head = kvh * G + row - qj * G;
    const long qr = (long)a.q_start[seq] + qj;
    // 16-lane groups take the chunks in turn, 8 elements a lane; the four groups' sums meet by shuffles
    const int dl = (lane & 15) * 8, grp = lane >> 4;
    float s[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (dl < a.D) {
#pragma unroll 4
        for (int i = grp; i < n; i += 4) {
            float x[8];
            load8<float>(p + i * step + 4 + dl, x);
            const float w = wgt[i];
#pragma unroll
            for (int j = 0; j < 8; ++j) s[j] = fmaf(w, x[j], s[j]);
        }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        s[j] += __shfl_xor(s[j], 16, 64);
        s[j] += __shfl_xor(s[j], 32, 64);
        s[j] *= inv;
    }
    if (grp == 0 && dl < a.D) store8<T>((T*)(a.out + qr * a.so.rs + (long)head * a.so.hs) + dl, s);
    if (lane == 0) a.lse[qr * a.hq + head] = lse_of(m, l);
}

// ---- backward ------------------------------------------------------------------------------------------------------------------------------
// delta[row, head] = sum_d dO O; 16 lanes per (row, head)
template <typename T>
__global__ __launch_bounds__(256) void packed_attn_delta_kernel(PAttnArgs a, long n) {
    const long i = (long)blockIdx.x * 16 + (threadIdx.x >> 4);
    const int d = (threadIdx.x & 15) * 8;
    float s = 0.f;
    if (i < n && d < a.D) {
        const long row = i / a.hq;
        const int head = (int)(i - row * a.hq);
        float x[8], y[8];
        load8<T>((const T*)(a.o + row * a.so.rs + (long)head * a.so.hs) + d, x);
        load8<T>((const T*)(a.dout + row * a.sdo.rs + (long)head * a.sdo.hs) + d, y);
#pragma unroll
        for (int j = 0; j < 8; ++j) s = fmaf(x[j], y[j], s);
    }
    s = group_sum<16>(s);
    if (i < n && d == 0) a.delta[i] = s;
}

enum { DQ = 0, DQ_TABLE = 1, DELTA = 2 };

// Adds a wave's 32 x (32 NT) dS (lanes = queries) to its sums by distance; h points at the entry of distance (tile's first key - wave's first query).
// The tile goes through LDS as [query][key]. 64 keys: in step q lane l reads key (q + l - 31) mod 64 of query q, so over the 32 steps every element
// is read once, and what a lane sees is one diagonal key - query = l - 31 while q + l >= 31 and one diagonal l + 33 before. 32 keys: the same
// modulo 32 by half waves, one for queries 0..15 and one for 16..31, whose sums then meet: 16 steps. (One LDS float atomic per element
// instead took 67 cycles each: 200 us of the dq kernel for 12 recordings of 100-1200 frames, 16 heads of 64.)
template <int NT> constexpr int diag_pitch() { return 32 * NT + 4; }      // floats; 16-byte pieces of eight rows fall in different banks
template <int NT> constexpr int diag_floats() { return 32 * diag_pitch<NT>(); }
typedef __attribute__((address_space(3))) float* lds_fptr;
typedef __attribute__((address_space(3))) f32x4* lds_f4ptr;
template <int NT> __device__ __forceinline__ void add_diagonals(unsigned m, unsigned h, const f32x16 (&x)[NT], int lane) {
    constexpr int P = diag_pitch<NT>(), S = 16 * NT;
    const int r = lane & 31, h2 = lane >> 5;
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int g = 0; g < 4; ++g)
            *(lds_f4ptr)(uintptr_t)(m + (r * P + 4 * h2) * 4 + (t * 32 + 8 * g) * 4) = f32x4{x[t][4 * g], x[t][4 * g + 1], x[t][4 * g + 2], x[t][4 * g + 3]};
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");      // a wave's LDS operations run in order; this keeps the compiler's order too
    float all = 0.f, before = 0.f;
    const int l = NT == 2 ? lane : r, q0 = NT == 2 ? 0 : 16 * h2;
    const unsigned mq = m + q0 * P * 4;
#pragma unroll
    for (int s = 0; s < S; ++s) {
        const float v = *(lds_fptr)(uintptr_t)(mq + (((l + q0 + s + 32 * NT - 31) & (32 * NT - 1)) << 2) + s * P * 4);
        all += v;
        if (NT == 1 || s < 31) before += l < 31 - q0 - s ? v : 0.f;
        if ((s & 7) == 7) pace<true>();
    }
    if constexpr (NT == 2) {
        const unsigned a = h + (lane - 31) * 4;
        *(lds_fptr)(uintptr_t)a = *(lds_fptr)(uintptr_t)a + (all - before);
        asm volatile("" ::: "memory");
        if (lane < 31) *(lds_fptr)(uintptr_t)(a + 64 * 4) = *(lds_fptr)(uintptr_t)(a + 64 * 4) + before;
    } else {
        all += __shfl_xor(all, 32, 64);
        before += __shfl_xor(before, 32, 64);
        const unsigned a = h + (h2 ? l + 1 : l - 31) * 4;
        *(lds_fptr)(uintptr_t)a = *(lds_fptr)(uintptr_t)a + (h2 ? before : all - before);      // (h2, l = 31: nothing, + 0)
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
}

// Keys of a wave's step in 32s, LDS buffers and waves per SIMD. With the table's gradient LDS holds its sums too: for heads above 32 one buffer and 32 keys at
// a time let three (64) or two (f32, 128) workgroups share a CU, whose others cover a wait for the tile (bf16, 12 x 100-1200, 16 heads of 64,
// forward + backward: two buffers and 64 keys 197 us, one and 32 186; f32, 6 x 30-600, 8 heads of 64, this kernel alone: 70 -> 59).
template <typename T, int DP, int MODE> constexpr int dq_step() { return sizeof(T) == 4 || MODE == DQ_TABLE || (DP <= 64 && MODE == DQ) ? 1 : 2; }
template <typename T, int DP, int MODE> constexpr int dq_buffers() { return DP >= 64 && MODE == DQ_TABLE ? 1 : 2; }
template <typename T, int DP, int MODE> constexpr int dq_waves() { return sizeof(T) == 2 && DP == 64 && MODE != DELTA ? 3 : waves_per_simd<T, DP>(); }
// dq (and the table's gradient), tiled like the forward; DELTA: only delta = sum_j P dP
template <typename T, int DP, bool BIAS, int MODE>
__global__ __launch_bounds__(256, (dq_waves<T, DP, MODE>())) void packed_attn_dq_kernel(PAttnArgs a) {
    using I = Image<T, DP>;
    constexpr int TB = KT * I::RB, NB = dq_buffers<T, DP, MODE>(), KS = key_split<T>(), KW = KT / KS, NT = 2 / KS, N = dq_step<T, DP, MODE>();
    constexpr bool TIGHT = DP == 128;
    extern __shared__ __attribute__((aligned(1024))) char smem[];      // NB x (K | V) | bias by distance | then (DQ_TABLE) sums by distance, a copy per wave | 8 floats | 4 x diag_floats
    float* dist = (float*)(smem + NB * 2 * TB);
    const int ndist = BIAS ? dist_count(a.maxd) : 0;
    float* hist = dist + ndist;
    float* far = hist + 4 * ndist;
    const unsigned diag = (lds_addr(far + 8) + 15) & ~15u;
    Dist bias;
    if constexpr (BIAS) bias.ask(a);
    const QTile w = q_tile_of<KS>(a);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 31, h2 = lane >> 5;
    const int rg = wave % (4 / KS), kh = wave / (4 / KS);       // the wave's rows and its part of every key tile
    const int qi = w.q0 + rg * WR + r;
    const bool live = qi < w.q_len;
    const long qrow = w.q_row + min(qi, w.q_len - 1);
    const char* kb = a.k + w.k_row * a.sk.rs + (long)w.kvh * a.sk.hs;
    const char* vb = a.v + w.k_row * a.sv.rs + (long)w.kvh * a.sv.hs;
    Stream<T, DP, KT, 4> ks, vs;
    ks.init(a.sk.rs, a.D, wave);
    vs.init(a.sv.rs, a.D, wave);
    const unsigned lds0 = lds_addr(smem);
    const typename I::Lane im0 = I::lane_offsets(lane);
    const int nt = (w.nk + KT - 1) / KT;
    if constexpr (BIAS) bias.look(a, w.head);
    if (nt) { ks.load(kb, w.k_len, lds0); vs.load(vb, w.k_len, lds0 + TB); }
    if constexpr (MODE == DQ_TABLE)
        for (int i = threadIdx.x; i < 4 * ndist; i += 256) hist[i] = 0.f;
    typename I::Frag fq[DP / 16], fo[DP / 16];
    {
        const char* row = a.q + qrow * a.sq.rs + (long)w.head * a.sq.hs;
        const char* dor = a.dout + qrow * a.sdo.rs + (long)w.head * a.sdo.hs;
#pragma unroll
        for (int kk = 0; kk < DP / 16; ++kk) { fq[kk] = global_frag<T, DP>(row, kk, h2, a.D); fo[kk] = global_frag<T, DP>(dor, kk, h2, a.D); }
    }
    const long si = qrow * a.hq + w.head;
    const float lse = a.lse[si];
    const float lse2 = live && lse != -__builtin_inff() ? lse * LOG2E : __builtin_inff();      // +inf: every probability of the row is 0 (a NaN stays one)
    float dl = 0.f;
    if constexpr (MODE != DELTA) dl = a.delta[si];
    const int qpos = qi + w.off, qw0 = w.q0 + rg * WR + w.off;
    const int klim = a.causal ? min(w.k_len - 1, qpos) : w.k_len - 1;
    const int wlim0 = a.causal ? min(w.k_len - 1, qw0) : w.k_len - 1;
    const int wlim1 = w.q0 + rg * WR >= w.q_len ? -1 : a.causal ? min(w.k_len - 1, qw0 + WR - 1) : w.k_len - 1;
    float far_lo = 0.f, far_hi = 0.f, sum_lo = 0.f, sum_hi = 0.f;
    if constexpr (BIAS) { bias.put(dist, a, w.head); far_lo = bias.far(bias.lo); far_hi = bias.far(bias.hi); }
    f32x16 dq[DP / 32], start;
    zero_acc(dq);
#pragma unroll
    for (int e = 0; e < 16; ++e) start[e] = MODE == DELTA ? 0.f : -dl;
    PA_LOADS_DONE();
    for (int i = 0; i < nt; ++i) {
        const int k0 = i * KT;
        PA_SYNC_TILE();
        if (NB == 1 && i) {
            ks.load(kb + (long)k0 * a.sk.rs, w.k_len - k0, lds0);
            vs.load(vb + (long)k0 * a.sv.rs, w.k_len - k0, lds0 + TB);
            PA_SYNC_TILE();
        }
        if (NB == 2 && i + 1 < nt) {
            const unsigned dst = lds0 + ((i + 1) & 1) * 2 * TB;
            ks.load(kb + (long)(k0 + KT) * a.sk.rs, w.k_len - k0 - KT, dst);
            vs.load(vb + (long)(k0 + KT) * a.sv.rs, w.k_len - k0 - KT, dst + TB);
        }
        const int kt0 = k0 + kh * KW;                      // the wave's first key of the tile
        if (kt0 > wlim1) continue;
        const typename I::Lane im = I::at(im0, lds0 + kh * KW * I::RB + (NB == 2 ? i & 1 : 0) * 2 * TB);
#pragma unroll
        for (int t0 = 0; t0 < NT; t0 += N) {
            const int kt = kt0 + 32 * t0;
            if (t0 && kt > wlim1) continue;
            f32x16 st[N], dp[N];
            zero_acc(st);
            float off = 0.f;
            int place = NEAR;
            if constexpr (BIAS) {
                place = place_of(kt - (qw0 + WR - 1), kt + 32 * N - 1 - qw0, a.maxd);
                if (place == NEAR) start_near<N, 1>(st, dist + (kt + 4 * h2 - qpos + a.maxd + NEAR_PAD));
                else off = place < 0 ? far_lo : far_hi;
            }
#pragma unroll
            for (int t = 0; t < N; ++t) dp[t] = start;          // dP - delta: the product starts from -delta of the lane's query
#pragma unroll
            for (int kk = 0; kk < DP / 16; ++kk)
#pragma unroll
                for (int t = 0; t < N; ++t) {
                    I::M::mma(I::row_frag(im, t0 + t, kk), fq[kk], st[t]);
                    I::M::mma(I::row_frag(im, t0 + t, kk, TB), fo[kk], dp[t]);
                    if (t == N - 1) pace<TIGHT>();
                }
            if (kt + 32 * N - 1 > wlim0) mask_rows<N>(st, klim - kt - 4 * h2, -__builtin_inff());
            const float sub = off - lse2;
#pragma unroll
            for (int t = 0; t < N; ++t)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const float p = __builtin_amdgcn_exp2f(fmaf(st[t][e], a.c, sub));
                    if constexpr (MODE == DELTA) dl = fmaf(p, dp[t][e], dl);
                    else st[t][e] = p * dp[t][e];
                }
            if constexpr (MODE == DQ_TABLE) {
                if (place == NEAR) {
                    add_diagonals<N>(diag + wave * diag_floats<N>() * 4, lds_addr(hist) + (wave * ndist + kt - qw0 + a.maxd + NEAR_PAD) * 4, st, lane);
                } else {
                    float s = 0.f;
#pragma unroll
                    for (int t = 0; t < N; ++t)
#pragma unroll
                        for (int e = 0; e < 16; ++e) s += st[t][e];
                    if (place < 0) sum_lo += s; else sum_hi += s;
                }
            }
            if constexpr (MODE != DELTA) acc_product<T, DP, N, TIGHT>(dq, st, im, t0, lane, 0);
        }
    }
    if constexpr (KS > 1) {                                // the second half's waves hand over their sums
        float* x = (float*)smem + rg * (DP / 2) * 64 + lane;
        __syncthreads();
        if (kh)
#pragma unroll
            for (int e = 0; e < DP / 2; ++e) x[e * 64] = dq[e >> 4][e & 15];
        __syncthreads();
        if (!kh)
#pragma unroll
            for (int e = 0; e < DP / 2; ++e) dq[e >> 4][e & 15] += x[e * 64];
    }
    if constexpr (MODE == DELTA) {
        dl += __shfl_xor(dl, 32, 64);
        if (live && h2 == 0) a.delta[si] = dl;
    } else store_rows<T, DP>(a.dq + qrow * a.sdq.rs + (long)w.head * a.sdq.hs, live && kh == 0, dq, a.scale, a.D, h2);
    if constexpr (MODE == DQ_TABLE) {
        sum_lo = wave_sum(sum_lo);
        sum_hi = wave_sum(sum_hi);
        if (lane == 0) { far[wave * 2] = sum_lo; far[wave * 2 + 1] = sum_hi; }
        __syncthreads();
        for (int i = threadIdx.x; i < ndist; i += 256) {
            float s = 0.f;
#pragma unroll
            for (int x = 0; x < 4; ++x) s += hist[x * ndist + i];
            dist[i] = s;
        }
        __syncthreads();
        float* part = a.part + ((long)(blockIdx.x / a.hq) * a.hq + w.head) * a.buckets;
        for (int b = threadIdx.x >> 4; b < a.buckets; b += 16) {            // 16 lanes a bucket
            const int first = a.ranges[2 * b], last = a.ranges[2 * b + 1], l16 = threadIdx.x & 15;      // distances of the bucket; none: first > last
            float s = 0.f;
            if (first <= last) {
                const int i0 = first <= -a.maxd ? 0 : first + a.maxd + NEAR_PAD, i1 = last >= a.maxd ? ndist - 1 : last + a.maxd + NEAR_PAD;
                if (l16 < 4 && first <= -a.maxd) s += far[2 * l16];
                if (l16 < 4 && last >= a.maxd) s += far[2 * l16 + 1];
                for (int i = i0 + l16; i <= i1; i += 16) s += dist[i];
            }
            s = group_sum<16>(s);
            if (l16 == 0) part[b] = s;
        }
    }
}

// dtable[b, head] (+)= sum over the query tiles, in their order, in 64 bits; one workgroup per (head, 16 buckets)
__global__ __launch_bounds__(256) void packed_attn_table_kernel(const float* part, float* dtable, int tiles, int hq, int buckets, int accumulate) {
    __shared__ double acc[16][16];
    const int head = blockIdx.x % hq, b = (blockIdx.x / hq) * 16 + (threadIdx.x & 15), g = threadIdx.x >> 4;
    double s = 0.0;
    if (b < buckets)
        for (int i = g; i < tiles; i += 16) s += (double)part[((long)i * hq + head) * buckets + b];
    acc[g][threadIdx.x & 15] = s;
    __syncthreads();
    if (g == 0 && b < buckets) {
        for (int i = 1; i < 16; ++i) s += acc[i][threadIdx.x];
        float* d = dtable + (long)b * hq + head;
        *d = accumulate ? (float)(s + (double)*d) : (float)s;
    }
}

// first query tile that a key of the tile is seen by, and how many workgroups share a key tile's stream of `total` query tiles
__device__ __forceinline__ int dkv_first(const PAttnArgs& a, int kt0, int q_len, int k_len) {
    return kt0 >= k_len ? q_len : a.causal ? max(0, kt0 - (k_len - q_len)) / KT * KT : 0;
}
__device__ __forceinline__ int dkv_parts(int total, int most, int chunk) { return max(1, min(most, (total + chunk - 1) / chunk)); }
// The place of a tile's first part, so that memory follows the work and not the longest recording times the tiles: the tiles before it in the list hold `before`
// query tiles per head (counted by the keys' capacity: at least as many as there are) and take the sum of ceil(their G / chunk) places, which
// floor(before G / chunk) + their number is never less than.
__device__ __forceinline__ long dkv_slot(const PAttnArgs& a, const int* rec, int ti, int kvh) {
    const unsigned long before = (unsigned)rec[6] | (unsigned long)(unsigned)rec[7] << 32;
    return kvh * a.slots + (long)(before * (unsigned)(a.hq / a.hkv) / (unsigned)a.chunk) + ti;
}

// dk, dv: 128 keys of one (recording, key head), a wave 32 (lanes = keys); the query heads of the group and the 64-query tiles stream by.
// A stream of more than `chunk` tiles is shared between up to nsplit workgroups: f32 partials, added in order by packed_attn_dkv_join_kernel.
// (heads of 128 in bf16: a few of v's operands are read from LDS at every tile; held in registers with the rest they spill, and a spill's reload
// waits for the next tile's DMA. Two workgroups still fit a CU's LDS.)
template <typename T, int DP, bool BIAS> constexpr int dkv_lds_frags() { return sizeof(T) == 2 && DP == 128 ? (BIAS ? 3 : 2) : 0; }
template <typename T, int DP, bool BIAS>
__global__ __launch_bounds__(256, (sizeof(T) == 2 && DP == 64 ? 3 : waves_per_simd<T, DP>())) void packed_attn_dkv_kernel(PAttnArgs a) {
    using I = Image<T, DP>;
    constexpr int TB = KT * I::RB;
    constexpr bool TIGHT = DP == 128;
    extern __shared__ __attribute__((aligned(1024))) char smem[];      // 2 x (Q | dO) | 2 x (lse | -delta) x 64 | bias by distance
    float* stat = (float*)(smem + 4 * TB);
    constexpr int LV = dkv_lds_frags<T, DP, BIAS>(), RV = DP / 16 - LV;      // operands of v kept in LDS / in registers
    char* kept = (char*)(stat + 4 * KT) + (threadIdx.x >> 6) * LV * 1024 + (threadIdx.x & 63) * 16;
    float* dist = stat + 4 * KT + LV * 1024;
    Dist bias;
    if constexpr (BIAS) bias.ask(a);
    const int kvh = blockIdx.x % a.hkv, rest = blockIdx.x / a.hkv, split = rest % a.nsplit, ti = rest / a.nsplit;
    const int* rec = a.tiles + 8 * (long)ti;
    const int seq = rec[0], kt0 = rec[1], q_row = rec[2], q_len = rec[3], k_row = rec[4], k_cap = rec[5];
    const int k_len = max(0, min(a.k_len[seq], k_cap)), off = k_len - q_len, G = a.hq / a.hkv;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 31, h2 = lane >> 5;
    const int kw0 = kt0 + wave * WR, key = kw0 + r;
    f32x16 dk[DP / 32], dv[DP / 32];
    zero_acc(dk);
    zero_acc(dv);
    const int qfirst = dkv_first(a, kt0, q_len, k_len);
    const int per = qfirst < q_len ? (q_len - qfirst + KT - 1) / KT : 0, total = per * G;
    const int ns = dkv_parts(total, a.nsplit, a.chunk);
    if (split >= ns) return;
    const int i0 = (int)((long)total * split / ns), i1 = (int)((long)total * (split + 1) / ns);
    if (i0 < i1) {
        typename I::Frag fk[DP / 16], fv[RV];
        {
            const long kr = (long)k_row + min(key, k_len - 1);
            const char* krp = a.k + kr * a.sk.rs + (long)kvh * a.sk.hs;
            const char* vrp = a.v + kr * a.sv.rs + (long)kvh * a.sv.hs;
#pragma unroll
            for (int kk = 0; kk < DP / 16; ++kk) { fk[kk] = global_frag<T, DP>(krp, kk, h2, a.D); if (kk < RV) fv[kk < RV ? kk : 0] = global_frag<T, DP>(vrp, kk, h2, a.D); }
            if constexpr (sizeof(T) == 2)
#pragma unroll
                for (int x = 0; x < LV; ++x) *(typename I::Frag*)(kept + x * 1024) = global_frag<T, DP>(vrp, RV + x, h2, a.D);
        }
        Stream<T, DP, KT, 4, TIGHT> qs, os;
        qs.init(a.sq.rs, a.D, wave);
        os.init(a.sdo.rs, a.D, wave);
        const unsigned lds0 = lds_addr(smem);
        typename I::Lane im = I::at(I::lane_offsets(lane), lds0 + 2 * TB);      // moved to the other buffer at every tile
        float reg = 0.f;                                   // threads 0..63: lse of the next tile, 64..127: delta
        auto fetch = [&](int it, unsigned dst) {
            const int g = it / per, q0 = qfirst + (it - g * per) * KT, head = kvh * G + g;
            const long row = (long)q_row + q0;
            if (threadIdx.x < 2 * KT) {
                const long s = (row + min((int)threadIdx.x & (KT - 1), q_len - 1 - q0)) * a.hq + head;
                reg = (threadIdx.x < KT ? a.lse : a.delta)[s];
            }
            qs.load(a.q + row * a.sq.rs + (long)head * a.sq.hs, q_len - q0, dst);
            os.load(a.dout + row * a.sdo.rs + (long)head * a.sdo.hs, q_len - q0, dst + TB);
        };
        fetch(i0, lds0);
        // the bias of all the part's heads at once where LDS has room, otherwise of one head at a time
        const int g0 = i0 / per, ndist = BIAS ? dist_count(a.maxd) : 0;
        const bool all = BIAS && (i1 - 1) / per - g0 < a.bias_heads;
        if constexpr (BIAS)
            if (all)
                for (int g = g0; g <= (i1 - 1) / per; ++g) { bias.look(a, kvh * G + g); bias.put(dist + (g - g0) * ndist, a, kvh * G + g); }
        int held = -1;                                     // the head that LDS holds
        for (int it = i0; it < i1; ++it) {
            const int par = (it - i0) & 1, g = it / per, q0 = qfirst + (it - g * per) * KT;
            float* ls = stat + par * 2 * KT;
            if (threadIdx.x < 2 * KT) {                    // rows past the end and rows without keys: probabilities 0
                const bool in = q0 + ((int)threadIdx.x & (KT - 1)) < q_len;
                ls[threadIdx.x] = threadIdx.x < KT ? (in && reg != -__builtin_inff() ? reg * LOG2E : __builtin_inff()) : in ? -reg : 0.f;
            }
            if constexpr (BIAS) {
                if (!all && g != held) {                   // uniform; the last tile's readers are past the barrier below before anything is overwritten
                    if (held >= 0) __syncthreads();
                    held = g;
                    dist_fill(dist, a, kvh * G + g);
                }
            }
            PA_LOADS_DONE();
            PA_SYNC_TILE();
            I::template move<TIGHT>(im, par ? 2 * TB : -2 * TB);
            if (it + 1 < i1) fetch(it + 1, lds0 + (par ^ 1) * 2 * TB);
            const int qp0 = q0 + off;                      // position of the tile's first query
            const float* near = dist + (all ? (g - g0) * ndist : 0);
            if (kw0 >= k_len) continue;
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const int qt0 = qp0 + t * 32;
                if (q0 + t * 32 >= q_len || (a.causal && qt0 + 31 < kw0)) continue;      // 32 queries that do not exist or see none of the wave's keys
                f32x16 s[1], dp[1];
                zero_acc(s);
                float bo = 0.f;
                if constexpr (BIAS) {
                    const int place = place_of(kw0 - (qt0 + 31), kw0 + WR - 1 - qt0, a.maxd);
                    if (place == NEAR) start_near<1, -1>(s, near + (key - qt0 - 4 * h2 + a.maxd + NEAR_PAD));
                    else bo = near[place < 0 ? 0 : ndist - 1] * a.c;
                }
#pragma unroll
                for (int gq = 0; gq < 4; ++gq) {           // dP - delta: the product starts from -delta of the row's query
                    const f32x4 dl = *(const f32x4*)(ls + KT + t * 32 + 8 * gq + 4 * h2);
#pragma unroll
                    for (int i = 0; i < 4; ++i) dp[0][4 * gq + i] = dl[i];
                }
#pragma unroll
                for (int kk = 0; kk < DP / 16; ++kk) {
                    I::M::mma(I::row_frag(im, t, kk), fk[kk], s[0]);      // rows = queries, lanes = keys
                    if (kk < RV) I::M::mma(I::row_frag(im, t, kk, TB), fv[kk < RV ? kk : 0], dp[0]);
                    else if constexpr (sizeof(T) == 2) I::M::mma(I::row_frag(im, t, kk, TB), *(const typename I::Frag*)(kept + (kk - RV) * 1024), dp[0]);
                    if (kk & 1) pace<TIGHT>();
                }
                if (kw0 + WR > k_len || (a.causal && qt0 < kw0 + WR - 1)) {            // some pair is masked: keep key < k_len and query >= key
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const int qp = qt0 + (e & 3) + 8 * (e >> 2) + 4 * h2;
                        s[0][e] = key < k_len && (!a.causal || qp >= key) ? s[0][e] : -__builtin_inff();
                    }
                }
#pragma unroll
                for (int gq = 0; gq < 4; ++gq) {
                    const f32x4 lv = *(const f32x4*)(ls + t * 32 + 8 * gq + 4 * h2);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int e = 4 * gq + i;
                        const float p = __builtin_amdgcn_exp2f(fmaf(s[0][e], a.c, bo - lv[i]));
                        s[0][e] = p;
                        dp[0][e] *= p;
                    }
                }
                acc_product<T, DP, 1, TIGHT>(dv, s, im, t, lane, TB);
                acc_product<T, DP, 1, TIGHT>(dk, dp, im, t, lane, 0);
            }
        }
    }
    int own = lane;                                        // found again here: nothing of the outputs' addresses lives through the loop
    asm volatile("" : "+v"(own));
    const int orow = wave * WR + (own & 31), okey = kt0 + orow, oh = own >> 5;
    const long krow = (long)k_row + min(okey, k_cap - 1);
    const bool live = okey < k_cap;                        // rows between a recording's length and its capacity get zeros
    if (ns == 1) {
        store_rows<T, DP>(a.dk + krow * a.sdk.rs + (long)kvh * a.sdk.hs, live, dk, a.scale, a.D, oh);
        store_rows<T, DP>(a.dv + krow * a.sdv.rs + (long)kvh * a.sdv.hs, live, dv, 1.f, a.D, oh);
    } else {
        float* p = a.part + ((dkv_slot(a, rec, ti, kvh) + split) * 2 * TILE + orow) * DP;
        store_rows<float, DP>((char*)p, true, dk, a.scale, DP, oh);
        store_rows<float, DP>((char*)(p + (long)TILE * DP), true, dv, 1.f, DP, oh);
    }
}
// adds the parts of a key tile, 256 pieces of 8 elements a workgroup
template <typename T, int DP>
__global__ __launch_bounds__(256) void packed_attn_dkv_join_kernel(PAttnArgs a) {
    constexpr int PIECES = 2 * TILE * DP / 8 / 256;
    const int at = blockIdx.x % PIECES, kvh = blockIdx.x / PIECES % a.hkv, ti = blockIdx.x / PIECES / a.hkv;
    const int* rec = a.tiles + 8 * (long)ti;
    const int kt0 = rec[1], q_len = rec[3], rows = min(TILE, rec[5] - kt0), k_len = max(0, min(a.k_len[rec[0]], rec[5]));
    const int qfirst = dkv_first(a, kt0, q_len, k_len), per = qfirst < q_len ? (q_len - qfirst + KT - 1) / KT : 0;
    const int ns = dkv_parts(per * (a.hq / a.hkv), a.nsplit, a.chunk);
    const int i = at * 256 + threadIdx.x, which = i / (TILE * DP / 8), row = i / (DP / 8) % TILE, d = i % (DP / 8) * 8;
    if (ns == 1 || row >= rows || d >= a.D) return;
    const float* p = a.part + (dkv_slot(a, rec, ti, kvh) * 2 + which) * TILE * DP + row * DP + d;
    float s[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int x = 0; x < ns; ++x) {
        float y[8];
        load8<float>(p + (long)x * 2 * TILE * DP, y);
#pragma unroll
        for (int k = 0; k < 8; ++k) s[k] += y[k];
    }
    const Strides st = which ? a.sdv : a.sdk;
    store8<T>((T*)((which ? a.dv : a.dk) + ((long)rec[4] + kt0 + row) * st.rs + (long)kvh * st.hs) + d, s);
}

// ---- launches ------------------------------------------------------------------------------------------------------------------------------
// more than 64 KB of LDS has to be asked for, once per kernel, device and thread
int ask_lds(const void* kernel, int bytes) {
    if (bytes <= 65536) return 0;
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess) return -1;
    static thread_local struct { const void* kernel; int dev; } done[64];
    static thread_local int n = 0;
    for (int i = 0; i < n; ++i) if (done[i].kernel == kernel && done[i].dev == dev) return 0;
    if (hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024) != hipSuccess) return -1;
    if (n < 64) { done[n].kernel = kernel; done[n].dev = dev; ++n; }
    return 0;
}

struct Plan {                   // the host array of pseld_hip.h
    long seqs, rows, max_q, k_rows, max_k, q_tiles, k_tiles, k_work, k_work_causal;
    const int *q_start, *q_len, *k_start, *k_cap, *k_len, *q_tile, *q_tile_causal, *k_tile, *k_tile_causal;
};
Plan plan_of(const long* p) {
    Plan x;
    x.seqs = p[0]; x.rows = p[1]; x.max_q = p[2]; x.k_rows = p[3]; x.max_k = p[4]; x.q_tiles = p[5]; x.k_tiles = p[6]; x.k_work = p[7]; x.k_work_causal = p[8];
    const int** a[] = {&x.q_start, &x.q_len, &x.k_start, &x.k_cap, &x.k_len, &x.q_tile, &x.q_tile_causal, &x.k_tile, &x.k_tile_causal};
    for (int i = 0; i < 9; ++i) *a[i] = (const int*)p[9 + i];
    return x;
}
int pad_of(int D) { return D <= 32 ? 32 : D <= 64 ? 64 : 128; }
constexpr int FEW_TABLE = 4096;          // table entries of one key head's group that the few-rows kernel keeps in LDS

// The few-rows kernel takes the call when one key head's query rows of every recording fit its 32-row operand and its LDS the group's part of the table. Other
// calls go to the query-tiled kernel, which does not share a recording's keys between workgroups: 9 frames of 4 grouped heads over one cache of 131072 keys are
// one workgroup a query head.
bool few_rows(const Plan& p, int hq, int hkv, int buckets) { return p.max_q * (hq / hkv) <= WR && (long)buckets * (hq / hkv) <= FEW_TABLE; }
// keys per workgroup: 512 workgroups by the capacities, whole rounds of the four waves' blocks (3 streams of 60-131 k keys, 16/4 heads of
// 64: 2048 workgroups 73 us, 1024 72, 512 68; 48 of 100-4096, 16/2 heads of 128: 48, 34, 33). Two fit a CU up to heads of 64 in bf16, above LDS holds one. The
// cut knows the capacities alone: of the 48 unequal streams some 322 workgroups have keys, 1.26 rounds of the 256 places. A recording of up to 512 keys stays
// whole (one launch instead of two). At most 16384 chunks, whose weights fit the joining launch's LDS.
int few_chunk(const Plan& p, int hkv) {
    if (p.max_k <= 512) return 512;
    const long want = (p.k_rows * hkv + 511) / 512;
    const long c = (want + 127) / 128 * 128, least = (p.max_k + 16383) / 16384 > 256 ? (p.max_k + 16383) / 16384 : 256, most = least > 8192 ? least : 8192;
    return (int)((c < least ? least : c > most ? most : c) + 127) / 128 * 128;
}
int few_splits(const Plan& p, int hkv) { const int c = few_chunk(p, hkv); return p.max_k > c ? (int)((p.max_k + c - 1) / c) : 1; }
// Chunks to reserve per key head (few_slot; 0: no recording is cut). A recording without capacity has one too, which answers for its rows.
long few_slots(const Plan& p, int hkv) {
    const long c = few_chunk(p, hkv);
    return p.max_k <= c ? 0 : p.seqs > 1 ? p.k_rows / c + p.seqs : (p.k_rows + c - 1) / c;
}
// Query tiles per workgroup of the dk/dv kernel: each key tile's stream is cut into parts of at most this many, where the key tiles alone would not fill the
// chip or end unevenly. 400 and 600 parts of the whole work were the fastest of those tried (1 x 8191, 16/2 heads of 128, forward + backward, two
// workgroups a CU: 256 parts 1577 us, 330 1372, 400 1283, 460 1608; 12 x 100-1200, 16/4 heads of 64, three a CU: 500 parts 208 us, 600 184, 700 199, 900 194): with
// the tiles' odd ends those packs make 464 workgroups for 512 places and 684 for 768. Other packs end otherwise: 2 x 3000, 8/8 heads of 128, causal, makes 576 for
// 512, 1 x 4000 + 60 x 100, 16/4 heads of 64, 832 for 768, and the last of them wait for a place. Below 4 tiles a part would spend longer on its f32
// partials than on its tiles. f32 tiles take longer: parts of any length (6 x 30-600, 8 heads of 64: 350 parts 196 us, 500 208, 700 196, 1500 197; 3 x 1000
// causal, 4 heads of 128, backward: 170 parts 344 us, 700 312).
int dkv_chunk(const Plan& p, int hq, int D, int causal, int dtype) {
    const long work = (causal ? p.k_work_causal : p.k_work) * hq;
    const long parts = dtype == PSELD_F32 ? 700 : D > 64 ? 400 : 600, c = (work + parts - 1) / parts, least = dtype == PSELD_F32 ? 1 : 4;
    return (int)(c < least ? least : c > (1 << 20) ? 1 << 20 : c);
}
int dkv_splits(const Plan& p, int hq, int hkv, int D, int causal, int dtype) {
    const long longest = (p.max_q + KT - 1) / KT * (hq / hkv), c = dkv_chunk(p, hq, D, causal, dtype);
    return longest > c ? (int)((longest + c - 1) / c) : 1;
}
// Parts of dk/dv to reserve per key head (dkv_slot; 0: nothing is cut). Only tiles of more than `chunk` steps are cut, the first n of the list, which is in the
// order of their steps: the last of them ends at most at ceil(all steps / chunk) + n - 1. That is at most twice the parts the work is cut into.
long dkv_slots(const Plan& p, int hq, int hkv, int D, int causal, int dtype) {
    if (dkv_splits(p, hq, hkv, D, causal, dtype) == 1) return 0;
    const long steps = (causal ? p.k_work_causal : p.k_work) * (hq / hkv), c = dkv_chunk(p, hq, D, causal, dtype), n = steps / c < p.k_tiles ? steps / c : p.k_tiles;
    return (steps + c - 1) / c + (n > 1 ? n - 1 : 0);
}
bool delta_pass(int dtype, bool table_grad) { return table_grad && dtype == PSELD_BF16; }

#define PA_TRY(x) do { const int rc__ = (x); if (rc__) return rc__; } while (0)
int check(const char* name, int dtype, const Plan& p, int hq, int hkv, int D, float scale, const float* table, const int* lut, int buckets, int maxd) {
    PSELD_CHECK_ARG(dtype == PSELD_F32 || dtype == PSELD_BF16, "%s: unknown dtype", name);
    PSELD_CHECK_ARG(p.seqs > 0 && p.rows >= 0 && p.k_rows >= 0 && p.max_q >= 0 && p.max_k >= 0 && p.rows <= (1l << 30) && p.k_rows <= (1l << 30) && p.q_start && p.q_len && p.k_start && p.k_cap && p.k_len, "%s: bad plan", name);
    PSELD_CHECK_ARG(hkv > 0 && hq >= hkv && hq % hkv == 0 && hq <= 1024, "%s: query heads must be a multiple of the key heads, at most 1024", name);
    PSELD_CHECK_ARG(D > 0 && D % 8 == 0 && D <= 128, "%s: head sizes are multiples of 8 up to 128", name);
    PSELD_CHECK_ARG(scale > 0.f && scale < 1e30f, "%s: scale must be positive and finite", name);
    PSELD_CHECK_ARG(!table || (lut && buckets > 0 && buckets <= 512 && maxd > 0 && maxd <= 1024), "%s: position buckets: at most 512 over distances of at most 1024", name);
    return PSELD_OK;
}
int check_operand(const char* name, const char* what, int dtype, const void* ptr, const long* st, Strides& out, bool needed) {
    const int e = dtype == PSELD_BF16 ? 2 : 4;
    PSELD_CHECK_ARG(!needed || ptr, "%s: null pointer (%s)", name, what);
    PSELD_CHECK_ARG(((uintptr_t)ptr & 15) == 0 && st[0] * e % 16 == 0 && st[1] * e % 16 == 0, "%s: %s: address, row and head strides must be whole 16-byte pieces", name, what);
    PSELD_CHECK_ARG(st[0] >= 0 && st[0] < (1l << 23) && st[1] >= 0, "%s: %s: row stride out of range", name, what);
    out.rs = st[0] * e;
    out.hs = st[1] * e;
    return PSELD_OK;
}
// a result: its (row, head) vectors must not overlap, rows outside heads or heads outside rows
int check_result(const char* name, const char* what, int dtype, const void* ptr, const long* st, Strides& out, long rows, int heads, int D) {
    PA_TRY(check_operand(name, what, dtype, ptr, st, out, rows > 0));
    const bool row_major = (rows <= 1 || st[0] >= (heads - 1) * st[1] + D) && (heads <= 1 || st[1] >= D);
    const bool head_major = (heads <= 1 || st[1] >= (rows - 1) * st[0] + D) && (rows <= 1 || st[0] >= D);
    PSELD_CHECK_ARG(row_major || head_major, "%s: the rows of %s overlap", name, what);
    return PSELD_OK;
}

#define PA_LAUNCH(kernel, grid, block, lds, ...)                                                                             \
    do {                                                                                                                     \
        const long g__ = (grid);                                                                                             \
        if (g__ > 0) {                                                                                                       \
            PSELD_CHECK_ARG(g__ < (1l << 31), "packed_attn: too many tiles x heads for one launch");                         \
            if (ask_lds((const void*)&kernel, (lds))) { pseld_set_error("packed_attn: cannot reserve LDS"); return PSELD_ERR_HIP; }       \
            hipLaunchKernelGGL(kernel, dim3((unsigned)g__), dim3(block), (lds), s, __VA_ARGS__);                             \
        }                                                                                                                    \
    } while (0)

int dist_bytes(const PAttnArgs& a) { return a.table ? (2 * (a.maxd + NEAR_PAD) + 1) * 4 : 0; }

template <typename T, int DP, bool BIAS>
int run_fwd(PAttnArgs& a, const Plan& p, hipStream_t s) {
    constexpr int TB = KT * DP * (int)sizeof(T);
    if (few_rows(p, a.hq, a.hkv, BIAS ? a.buckets : 0)) {
        constexpr int NW = DP * sizeof(T) > 256 ? 2 : 4;
        const int G = a.hq / a.hkv;
        a.chunk = few_chunk(p, a.hkv);
        a.nsplit = few_splits(p, a.hkv);
        a.slots = few_slots(p, a.hkv);
        a.max_rows = (int)p.max_q * G;
        const int lds = NW * 4 * WR * DP * (int)sizeof(T) + (NW + 1) * 256 + (BIAS ? a.buckets * G * 4 + (2 * a.maxd + 1) * 2 : 0);
        PA_LAUNCH((packed_attn_few_kernel<T, DP, NW, BIAS>), p.seqs * a.nsplit * a.hkv, 64 * NW, lds, a);
        if (a.nsplit > 1) PA_LAUNCH((packed_attn_join_kernel<T>), p.seqs * a.hkv * a.max_rows, 64, a.nsplit * 4, a);
        return PSELD_OK;
    }
    a.tiles = a.causal ? p.q_tile_causal : p.q_tile;
    PA_LAUNCH((packed_attn_fwd_kernel<T, DP, BIAS>), p.q_tiles * key_split<T>() * a.hq, 256, 4 * TB + dist_bytes(a), a);
    return PSELD_OK;
}
template <typename T, int DP, bool BIAS>
int run_bwd(PAttnArgs& a, const Plan& p, float* dtable, int accumulate, hipStream_t s) {
    constexpr int TB = KT * DP * (int)sizeof(T);
    const int nd = dist_bytes(a);
    const long q_tiles = p.q_tiles * key_split<T>();
    constexpr int dtype = sizeof(T) == 2 ? PSELD_BF16 : PSELD_F32;
    a.tiles = a.causal ? p.q_tile_causal : p.q_tile;
    if constexpr (BIAS && sizeof(T) == 2) {
        if (dtable) PA_LAUNCH((packed_attn_dq_kernel<T, DP, BIAS, DELTA>), q_tiles * a.hq, 256, 4 * TB + nd, a);
    }
    if (!delta_pass(dtype, BIAS && dtable)) PA_LAUNCH((packed_attn_delta_kernel<T>), (p.rows * a.hq + 15) / 16, 256, 0, a, p.rows * a.hq);
    bool table_done = false;
    if constexpr (BIAS) {
        if (dtable) {
            float* part = a.part;
            PA_LAUNCH((packed_attn_dq_kernel<T, DP, BIAS, DQ_TABLE>), q_tiles * a.hq, 256, (dq_buffers<T, DP, DQ_TABLE>()) * 2 * TB + 5 * nd + 64 + 16 * (diag_floats<dq_step<T, DP, DQ_TABLE>()>()), a);
            PA_LAUNCH(packed_attn_table_kernel, (long)a.hq * ((a.buckets + 15) / 16), 256, 0, part, dtable, (int)q_tiles, a.hq, a.buckets, accumulate);
            a.part += q_tiles * a.hq * a.buckets;
            a.part = (float*)(((uintptr_t)a.part + 15) & ~(uintptr_t)15);
            table_done = true;
        }
    }
    if (!table_done) PA_LAUNCH((packed_attn_dq_kernel<T, DP, BIAS, DQ>), q_tiles * a.hq, 256, 4 * TB + nd, a);
    a.tiles = a.causal ? p.k_tile_causal : p.k_tile;
    a.bias_heads = BIAS ? (DP == 128 || 2 * nd > 12288 ? 1 : min(a.hq / a.hkv, 12288 / nd)) : 0;      // (two workgroups per CU stay possible)
    a.nsplit = dkv_splits(p, a.hq, a.hkv, a.D, a.causal, dtype);
    a.chunk = dkv_chunk(p, a.hq, a.D, a.causal, dtype);
    a.slots = dkv_slots(p, a.hq, a.hkv, a.D, a.causal, dtype);
    PA_LAUNCH((packed_attn_dkv_kernel<T, DP, BIAS>), p.k_tiles * a.hkv * a.nsplit, 256, 4 * TB + 4 * KT * 4 + 4096 * (dkv_lds_frags<T, DP, BIAS>()) + a.bias_heads * nd, a);
    if (a.nsplit > 1) PA_LAUNCH((packed_attn_dkv_join_kernel<T, DP>), p.k_tiles * a.hkv * (TILE * DP / 1024), 256, 0, a);
    return PSELD_OK;
}
template <typename T, typename F> int by_head_size(int D, bool bias, F&& f) {
    if (D <= 32) return bias ? f(std::integral_constant<int, 32>{}, std::true_type{}) : f(std::integral_constant<int, 32>{}, std::false_type{});
    if (D <= 64) return bias ? f(std::integral_constant<int, 64>{}, std::true_type{}) : f(std::integral_constant<int, 64>{}, std::false_type{});
    return bias ? f(std::integral_constant<int, 128>{}, std::true_type{}) : f(std::integral_constant<int, 128>{}, std::false_type{});
}
void fill(PAttnArgs& a, const Plan& p, int hq, int hkv, int D, int causal, float scale, const float* table, const int* lut, int buckets, int maxd) {
    a.q_start = p.q_start; a.q_len = p.q_len; a.k_start = p.k_start; a.k_cap = p.k_cap; a.k_len = p.k_len;
    a.seqs = (int)p.seqs; a.hq = hq; a.hkv = hkv; a.D = D; a.causal = causal; a.nsplit = 1;
    a.scale = scale; a.c = scale * LOG2E;
    a.table = table; a.lut = lut; a.buckets = table ? buckets : 0; a.maxd = table ? maxd : 0;
    a.ranges = lut ? lut + 2 * maxd + 1 : nullptr;
}

}  // namespace

extern "C" long pseld_packed_attn_fwd_workspace(const long* plan, int hq, int hkv, int D, int buckets) {
    if (!plan || hkv <= 0 || hq < hkv || hq % hkv) return 0;
    const Plan p = plan_of(plan);
    if (!few_rows(p, hq, hkv, buckets)) return 0;
    return few_slots(p, hkv) * hkv * p.max_q * (hq / hkv) * (D + 4) * (long)sizeof(float);
}

extern "C" int pseld_packed_attn_fwd(int dtype, const void* q, const void* k, const void* v, void* out, float* lse, const long* strides,
                                     const long* plan, int hq, int hkv, int D, int causal, float scale, const float* table, const int* lut,
                                     int buckets, int max_distance, float* workspace, long workspace_bytes, void* stream) {
    PSELD_CHECK_ARG(plan && strides, "packed_attn_fwd: null pointer");
    const Plan p = plan_of(plan);
    PA_TRY(check("packed_attn_fwd", dtype, p, hq, hkv, D, scale, table, lut, buckets, max_distance));
    PAttnArgs a{};
    const bool rows = p.rows > 0, keys = rows && p.k_rows > 0;
    PA_TRY(check_operand("packed_attn_fwd", "q", dtype, q, strides, a.sq, rows));
    PA_TRY(check_operand("packed_attn_fwd", "k", dtype, k, strides + 2, a.sk, keys));
    PA_TRY(check_operand("packed_attn_fwd", "v", dtype, v, strides + 4, a.sv, keys));
    PA_TRY(check_result("packed_attn_fwd", "out", dtype, out, strides + 6, a.so, p.rows, hq, D));
    PSELD_CHECK_ARG(!rows || lse, "packed_attn_fwd: null pointer (lse)");
    const long need = pseld_packed_attn_fwd_workspace(plan, hq, hkv, D, table ? buckets : 0);
    PSELD_CHECK_ARG(need == 0 || (workspace && ((uintptr_t)workspace & 15) == 0 && workspace_bytes >= need), "packed_attn_fwd: workspace too small or not on a 16-byte boundary");
    PSELD_CHECK_ARG(!rows || (out != q && out != k && out != v), "packed_attn_fwd: out must not be an operand");
    if (!rows) return PSELD_OK;
    a.q = (const char*)q; a.k = (const char*)k; a.v = (const char*)v; a.out = (char*)out; a.lse = lse; a.part = workspace;
    fill(a, p, hq, hkv, D, causal, scale, table, lut, buckets, max_distance);
    const hipStream_t s = (hipStream_t)stream;
    const int rc = dtype == PSELD_BF16
        ? by_head_size<bf16_t>(D, table, [&](auto dp, auto bias) { return run_fwd<bf16_t, decltype(dp)::value, decltype(bias)::value>(a, p, s); })
        : by_head_size<float>(D, table, [&](auto dp, auto bias) { return run_fwd<float, decltype(dp)::value, decltype(bias)::value>(a, p, s); });
    if (rc) return rc;
    PSELD_LAUNCH_CHECK("packed_attn_fwd");
    return PSELD_OK;
}

extern "C" long pseld_packed_attn_bwd_workspace(int dtype, const long* plan, int hq, int hkv, int D, int causal, int buckets) {
    if (!plan || hkv <= 0 || hq < hkv || hq % hkv) return 0;
    const Plan p = plan_of(plan);
    const long q_tiles = p.q_tiles * (dtype == PSELD_F32 ? key_split<float>() : key_split<bf16_t>());
    return ((p.rows * hq + 3) / 4 * 4 + q_tiles * hq * buckets + 4 + hkv * dkv_slots(p, hq, hkv, D, causal, dtype) * 2 * TILE * pad_of(D)) * (long)sizeof(float);
}

extern "C" int pseld_packed_attn_bwd(int dtype, const void* dout, const void* q, const void* k, const void* v, const void* out, const float* lse,
                                     void* dq, void* dk, void* dv, const long* strides, const long* plan, int hq, int hkv, int D, int causal, float scale,
                                     const float* table, const int* lut, int buckets, int max_distance, float* dtable, int accumulate,
                                     float* workspace, long workspace_bytes, void* stream) {
    PSELD_CHECK_ARG(plan && strides, "packed_attn_bwd: null pointer");
    const Plan p = plan_of(plan);
    PA_TRY(check("packed_attn_bwd", dtype, p, hq, hkv, D, scale, table, lut, buckets, max_distance));
    PSELD_CHECK_ARG(!dtable || table, "packed_attn_bwd: a table gradient needs the table");
    PAttnArgs a{};
    const bool rows = p.rows > 0, keys = p.k_rows > 0;
    const char* n = "packed_attn_bwd";
    PA_TRY(check_operand(n, "dout", dtype, dout, strides, a.sdo, rows));
    PA_TRY(check_operand(n, "q", dtype, q, strides + 2, a.sq, rows));
    PA_TRY(check_operand(n, "k", dtype, k, strides + 4, a.sk, keys));
    PA_TRY(check_operand(n, "v", dtype, v, strides + 6, a.sv, keys));
    PA_TRY(check_operand(n, "out", dtype, out, strides + 8, a.so, rows));
    PA_TRY(check_result(n, "dq", dtype, dq, strides + 10, a.sdq, p.rows, hq, D));
    PA_TRY(check_result(n, "dk", dtype, dk, strides + 12, a.sdk, p.k_rows, hkv, D));
    PA_TRY(check_result(n, "dv", dtype, dv, strides + 14, a.sdv, p.k_rows, hkv, D));
    const void* const results[] = {dq, dk, dv};
    for (int i = 0; i < 3; ++i) {
        const void* const others[] = {dout, q, k, v, out, results[(i + 1) % 3]};
        for (const void* x : others) PSELD_CHECK_ARG(!x || x != results[i], "%s: a gradient must not be an operand or another gradient", n);
    }
    PSELD_CHECK_ARG(!rows || lse, "packed_attn_bwd: null pointer (lse)");
    const long need = pseld_packed_attn_bwd_workspace(dtype, plan, hq, hkv, D, causal, dtable ? buckets : 0);
    PSELD_CHECK_ARG(workspace && ((uintptr_t)workspace & 15) == 0 && workspace_bytes >= need, "packed_attn_bwd: workspace too small or not on a 16-byte boundary");
    a.dout = (const char*)dout; a.q = (const char*)q; a.k = (const char*)k; a.v = (const char*)v; a.o = (const char*)out; a.lse = const_cast<float*>(lse);
    a.dq = (char*)dq; a.dk = (char*)dk; a.dv = (char*)dv;
    a.delta = workspace;
    a.part = workspace + (p.rows * hq + 3) / 4 * 4;
    fill(a, p, hq, hkv, D, causal, scale, table, lut, buckets, max_distance);
    const hipStream_t s = (hipStream_t)stream;
    const int rc = dtype == PSELD_BF16
        ? by_head_size<bf16_t>(D, table, [&](auto dp, auto bias) { return run_bwd<bf16_t, decltype(dp)::value, decltype(bias)::value>(a, p, dtable, accumulate, s); })
        : by_head_size<float>(D, table, [&](auto dp, auto bias) { return run_bwd<float, decltype(dp)::value, decltype(bias)::value>(a, p, dtable, accumulate, s); });
    if (rc) return rc;
    PSELD_LAUNCH_CHECK("packed_attn_bwd");
    return PSELD_OK;
}
