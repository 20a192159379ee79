// The MoE layer for a few tokens (up to 16) in two kernels.
//
//   z = x Wrᵀ (+ bias), (p, e) = top-k softmax(z), w = softmax(p) after the capacity trim
//   h = silu(Wg x) · (Wu x) per routed slot and shared expert,   y = Wd h
//   out = Σ_j w_j y_j + Σ_s mix_s y_s + 0.1 skip
//
// (model/moe/gate.py:1122-1247, opss/infer/fused_moe.py:69-119, model/moe/expert.py:475-489,
// model/moe/layer.py:741-753, :812-865). At one to sixteen tokens the touched experts' weights are
// nearly all the bytes, each is used once or a few times, and what the layer loses against the
// stream of those bytes are launches and waits. So there are two launches:
//
// 1. few_front_kernel: everything that needs no routing. The router's logits, as K-split partial
//    sums, and the gate/up products of the shared experts; it also clears the counters of 2.
// 2. few_experts_kernel: every work-group computes the routing from the logits by itself (N·k <= 256
//    slots in LDS; cheaper than another launch), then the gate/up products of the routed experts
//    are dealt out as (16-row tile, 16 columns of F) items, and once all of them are there each
//    work-group takes 16 columns of H of *all* tiles, so that the weighted sum, the shared mixture
//    and the skip residual end in its LDS: no expert output leaves the chip.
//
// Between the two halves of 2 work-groups wait for each other. The gate/up items are taken from
// counters and never assigned to a work-group beforehand, so every item that a wait is for is held
// by a work-group that runs and that waits for nothing: the wait ends whichever part of the grid is
// resident, also beside other kernels. (Should two calls be given one workspace at the same time,
// which is an error, the wait is left after kSpinLimit looks and out becomes NaN.)
//
// Rounding: weights enter exactly (codes as bf16, scales on the fp32 sums), h is rounded once to
// bf16 for the second product's MFMAs, the outputs once at the end.
#include <algorithm>

#include "yvmoe_frag.h"
#include "yvmoe_internal.h"
#include "yvmoe_topk.h"

namespace yvmoe {
namespace {

constexpr int kFewSlots = kFewTokens * YVMOE_MAX_TOPK;
constexpr int kFewTiles = kFewSlots + YVMOE_MAX_SHARED;
constexpr int kWaves = 8, kThreads = 64 * kWaves;
constexpr int kYRows = 512;            // rows of partial expert outputs that a work-group holds
constexpr int kRanges = 8;             // ranges of gate/up items, one per XCD
constexpr int kCounterStride = 32;     // ints between counters (a cache line each)
constexpr int kSpinLimit = 1 << 21;    // looks at the counter, about a microsecond each

struct FewArgs {
    const void* x;
    int N, H, F, E, S, k;
    const void *w_gate, *w_up, *w_down, *s_gate, *s_up, *s_down;
    // routing: from the logits' partial sums [nsplit][N][ld] (self), or given
    int self;
    const void* w_router;
    float* logits;
    int ncols, ld, nsplit;
    const float *bias, *b1, *w2, *b2;
    int cap_mode, min_cap;  // cap_mode: 0 none, 2 dynamic, 3 static factor
    double cap_factor;
    const void* rweights;
    int rweights_bf16;
    const int64_t* rindices;
    yvmoe_routing out_routing;  // self: the routing's outputs
    int* invalid;               // given: slots with an index outside [0, E), or NULL
    const float* mix;
    const void* skip;
    void* out;
    void* shared_out;
    void* h;        // [N k + S N][F], routed rows by expert, then the shared experts' tokens
    int* counters;  // [kRanges + 1] x kCounterStride: items taken per range, work-groups' items done
};

// ---------------------------------------------------------------- weights and activations
// A wavefront multiplies 16 rows of a weight matrix (the first MFMA operand) with 16 activation
// rows over 64-wide k-steps. Lane l = 16 g + r holds columns 16 g .. 16 g + 15 of weight row r and of
// activation row r; the accumulator holds weight rows 4 g + i of activation row r.
//
// Raw: a k-step's weights as stored. Act: a k-step's activations. UNIT: k-steps per chunk.
// GROUPED: the scale belongs to a row (int4) or 128 rows (fp8) and 128 columns, that is two k-steps.
template <int WF>
struct Wt;

struct ActB16 {
    Frag16 f;
    static constexpr int BYTES = 2;
    __device__ __forceinline__ void load(const char* row, int ks) {
        const uint4* p = (const uint4*)(row + (size_t)ks * 128);
        f.u[0] = p[0];
        f.u[1] = p[1];
    }
};

__device__ __forceinline__ f32x4 mfma16(const bf16x8& a, const bf16x8& b, const f32x4& c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// Blocked storage (include/yvmoe.h): the lane's address of its piece in the first block of the
// 16 rows from n0.
__device__ __forceinline__ const char* block_ptr(const void* base, long long bytes, int n0, int K, int blk,
                                                 int piece, int lane) {
    return (const char*)base + bytes + (long long)(n0 >> 4) * (K / 64) * blk + lane * piece;
}

template <>
struct Wt<YVMOE_W_BF16> {
    typedef Frag16 Raw;
    typedef ActB16 Act;
    static constexpr int UNIT = 2;
    static constexpr bool GROUPED = false;
    static __device__ __forceinline__ const char* ptr(const void* b, long long e, int n0, int K, int lane) {
        return block_ptr(b, e * 2, n0, K, 2048, 16, lane);
    }
    static __device__ __forceinline__ void load(Raw& r, const char* p, int ks) {
        r.u[0] = nt_load16(p + (size_t)ks * 2048);
        r.u[1] = nt_load16(p + (size_t)ks * 2048 + 1024);
    }
    static __device__ __forceinline__ void mma(const Raw& w, const Act& a, f32x4& acc) {
        acc = mfma16(w.v[0], a.f.v[0], acc);
        acc = mfma16(w.v[1], a.f.v[1], acc);
    }
};

template <>
struct Wt<YVMOE_W_INT8> {
    typedef uint4 Raw;
    typedef ActB16 Act;
    static constexpr int UNIT = 2;
    static constexpr bool GROUPED = false;
    static __device__ __forceinline__ const char* ptr(const void* b, long long e, int n0, int K, int lane) {
        return block_ptr(b, e, n0, K, 1024, 16, lane);
    }
    static __device__ __forceinline__ void load(Raw& r, const char* p, int ks) {
        r = nt_load16(p + (size_t)ks * 1024);
    }
    static __device__ __forceinline__ void mma(const Raw& r, const Act& a, f32x4& acc) {
        const unsigned w[4] = {r.x, r.y, r.z, r.w};
        unsigned o[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {  // codes are bf16 values: the upper halves of their fp32 forms
            const unsigned b0 = __float_as_uint((float)(int)(signed char)(w[i] & 0xffu));
            const unsigned b1 = __float_as_uint((float)(int)(signed char)((w[i] >> 8) & 0xffu));
            const unsigned b2 = __float_as_uint((float)(int)(signed char)((w[i] >> 16) & 0xffu));
            const unsigned b3 = __float_as_uint((float)((int)w[i] >> 24));
            o[2 * i] = __builtin_amdgcn_perm(b1, b0, 0x07060302u);
            o[2 * i + 1] = __builtin_amdgcn_perm(b3, b2, 0x07060302u);
        }
        Frag16 f;
        f.u[0] = make_uint4(o[0], o[1], o[2], o[3]);
        f.u[1] = make_uint4(o[4], o[5], o[6], o[7]);
        acc = mfma16(f.v[0], a.f.v[0], acc);
        acc = mfma16(f.v[1], a.f.v[1], acc);
    }
};

template <>
struct Wt<YVMOE_W_FP8> {
    typedef uint4 Raw;
    typedef ActB16 Act;
    static constexpr int UNIT = 2;
    static constexpr bool GROUPED = true;
    static __device__ __forceinline__ const char* ptr(const void* b, long long e, int n0, int K, int lane) {
        return block_ptr(b, e, n0, K, 1024, 16, lane);
    }
    static __device__ __forceinline__ void load(Raw& r, const char* p, int ks) {
        r = nt_load16(p + (size_t)ks * 1024);
    }
    static __device__ __forceinline__ void mma(const Raw& r, const Act& a, f32x4& acc) {
        const unsigned w[4] = {r.x, r.y, r.z, r.w};
        unsigned o[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {  // exact: e4m3 has fewer bits than bf16
            o[2 * i] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)w[i], 1.0f, false));
            o[2 * i + 1] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)w[i], 1.0f, true));
        }
        Frag16 f;
        f.u[0] = make_uint4(o[0], o[1], o[2], o[3]);
        f.u[1] = make_uint4(o[4], o[5], o[6], o[7]);
        acc = mfma16(f.v[0], a.f.v[0], acc);
        acc = mfma16(f.v[1], a.f.v[1], acc);
    }
};

// int4: a nibble q at bits 3-6 of 0x4180 is the bf16 number 16 + q, so two codes cost one shift and
// one and-or; the products' sum is Σ x (16 + q), and one more MFMA with a constant operand gives
// -24 Σ x for the group, which makes it Σ x (q - 8). Both are fp32 sums of exact products. Dword
// j of an operand then holds columns j and j + 4 of eight, and the activations are put in that order.
template <>
struct Wt<YVMOE_W_INT4> {
    typedef uint2 Raw;
    struct Act : ActB16 {
        __device__ __forceinline__ void order() {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const uint4 v = f.u[h];
                f.u[h] = make_uint4(__builtin_amdgcn_perm(v.z, v.x, 0x05040100u),
                                    __builtin_amdgcn_perm(v.z, v.x, 0x07060302u),
                                    __builtin_amdgcn_perm(v.w, v.y, 0x05040100u),
                                    __builtin_amdgcn_perm(v.w, v.y, 0x07060302u));
            }
        }
    };
    static constexpr int UNIT = 2;
    static constexpr bool GROUPED = true;
    static __device__ __forceinline__ const char* ptr(const void* b, long long e, int n0, int K, int lane) {
        return block_ptr(b, e / 2, n0, K, 512, 8, lane);
    }
    static __device__ __forceinline__ void load(Raw& r, const char* p, int ks) {
        r = nt_load8(p + (size_t)ks * 512);
    }
    static __device__ __forceinline__ uint4 codes(unsigned w) {
        return make_uint4(((w << 3) & 0x00780078u) | 0x41804180u, ((w >> 1) & 0x00780078u) | 0x41804180u,
                          ((w >> 5) & 0x00780078u) | 0x41804180u, ((w >> 9) & 0x00780078u) | 0x41804180u);
    }
    static __device__ __forceinline__ void offset(const Act& a, f32x4& corr) {
        Frag16 c;
        c.u[0] = make_uint4(0xC1C0C1C0u, 0xC1C0C1C0u, 0xC1C0C1C0u, 0xC1C0C1C0u);  // -24
        corr = mfma16(c.v[0], a.f.v[0], corr);
        corr = mfma16(c.v[0], a.f.v[1], corr);
    }
    static __device__ __forceinline__ void mma(const Raw& r, const Act& a, f32x4& acc) {
        Frag16 f;
        f.u[0] = codes(r.x);
        f.u[1] = codes(r.y);
        acc = mfma16(f.v[0], a.f.v[0], acc);
        acc = mfma16(f.v[1], a.f.v[1], acc);
    }
};

// fp32: rows as they are, 64 bytes per lane and k-step, on the fp32 MFMAs.
template <>
struct Wt<YVMOE_W_F32> {
    struct Raw {
        float4 v[4];
    };
    struct Act {
        float4 v[4];
        static constexpr int BYTES = 4;
        __device__ __forceinline__ void load(const char* row, int ks) {
            const float4* p = (const float4*)(row + (size_t)ks * 256);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = p[i];
        }
    };
    static constexpr int UNIT = 1;
    static constexpr bool GROUPED = false;
    static __device__ __forceinline__ const char* ptr(const void* b, long long e, int n0, int K, int lane) {
        return (const char*)b + (e + (long long)(n0 + (lane & 15)) * K + 16 * (lane >> 4)) * 4;
    }
    static __device__ __forceinline__ void load(Raw& r, const char* p, int ks) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint4 u = nt_load16(p + (size_t)ks * 256 + 16 * i);
            r.v[i] = make_float4(__uint_as_float(u.x), __uint_as_float(u.y), __uint_as_float(u.z), __uint_as_float(u.w));
        }
    }
    static __device__ __forceinline__ void mma(const Raw& w, const Act& a, f32x4& acc) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            acc = __builtin_amdgcn_mfma_f32_16x16x4f32(w.v[i].x, a.v[i].x, acc, 0, 0, 0);
            acc = __builtin_amdgcn_mfma_f32_16x16x4f32(w.v[i].y, a.v[i].y, acc, 0, 0, 0);
            acc = __builtin_amdgcn_mfma_f32_16x16x4f32(w.v[i].z, a.v[i].z, acc, 0, 0, 0);
            acc = __builtin_amdgcn_mfma_f32_16x16x4f32(w.v[i].w, a.v[i].w, acc, 0, 0, 0);
        }
    }
};

// NM matrices' 16 rows from n0 against one set of activation rows.
template <int WF, int NM>
struct Operands {
    const char* w[NM];
    const void* s[NM];  // GROUPED: the scales of these rows (int4: of the lane's row)
    const char* act;    // the lane's activation row at its columns

    __device__ __forceinline__ void set(int m, const void* base, const void* scales, long long e, int out, int K,
                                        int n0, int lane) {
        w[m] = Wt<WF>::ptr(base, e * out * K, n0, K, lane);
        if constexpr (WF == YVMOE_W_INT4)
            s[m] = (const unsigned short*)scales + (e * out + n0 + (lane & 15)) * (K / 128);
        else if constexpr (WF == YVMOE_W_FP8)
            s[m] = (const float*)scales + (e * (out / 128) + n0 / 128) * (K / 128);
        else s[m] = nullptr;
    }
    __device__ __forceinline__ void rows(const void* base, long long row, int K, int lane) {
        act = (const char*)base + (row * K + 16 * (lane >> 4)) * Wt<WF>::Act::BYTES;
    }
};

template <int WF, int NM>
struct Chunk {
    typedef Wt<WF> W;
    static constexpr int U = W::UNIT;
    typename W::Raw w[U][NM];
    typename W::Act a[U];
    float s[W::GROUPED ? U / 2 : 1][NM];

    // k-steps past the end: the last one again, not used
    __device__ __forceinline__ void load_weights(const Operands<WF, NM>& o, int c, int nks) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int ks = min(c * U + u, nks - 1);
#pragma unroll
            for (int m = 0; m < NM; ++m) {
                W::load(w[u][m], o.w[m], ks);
                if constexpr (W::GROUPED)
                    if (u % 2 == 0)
                        s[u / 2][m] = WF == YVMOE_W_INT4 ? bf16_to_f32(((const unsigned short*)o.s[m])[ks / 2])
                                                         : ((const float*)o.s[m])[ks / 2];
            }
        }
    }
    __device__ __forceinline__ void load_acts(const Operands<WF, NM>& o, int c, int nks) {
#pragma unroll
        for (int u = 0; u < U; ++u) a[u].load(o.act, min(c * U + u, nks - 1));
    }
    __device__ __forceinline__ void mma(int c, int nks, f32x4 (&acc)[NM]) {
        if constexpr (!W::GROUPED) {
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (c * U + u < nks)
#pragma unroll
                    for (int m = 0; m < NM; ++m) W::mma(w[u][m], a[u], acc[m]);
        } else {
#pragma unroll
            for (int p = 0; p < U; p += 2) {
                if (c * U + p >= nks) break;
                f32x4 part[NM], corr = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int m = 0; m < NM; ++m) part[m] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int u = p; u < p + 2; ++u) {
                    if constexpr (WF == YVMOE_W_INT4) {
                        a[u].order();
                        W::offset(a[u], corr);
                    }
#pragma unroll
                    for (int m = 0; m < NM; ++m) W::mma(w[u][m], a[u], part[m]);
                }
#pragma unroll
                for (int m = 0; m < NM; ++m)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        if constexpr (WF == YVMOE_W_INT4) {
                            // the scale of weight row 4 g + i, from the lane that loaded it
                            const float si = __int_as_float(__builtin_amdgcn_ds_bpermute(
                                4 * (4 * ((threadIdx.x & 63) >> 4) + i), __float_as_int(s[p / 2][m])));
                            acc[m][i] = __builtin_fmaf(si, part[m][i] + corr[i], acc[m][i]);
                        } else {
                            acc[m][i] = __builtin_fmaf(s[p / 2][m], part[m][i], acc[m][i]);
                        }
                    }
            }
        }
    }
};

// acc += the products over chunks c0, c0 + step, ... below c1, the next chunk's loads in flight
// during the current one's MFMAs.
template <int WF, int NM>
__device__ __forceinline__ void stream(const Operands<WF, NM>& o, int nks, int c0, int c1, int step,
                                       f32x4 (&acc)[NM]) {
    Chunk<WF, NM> q0, q1;
    auto load = [&](Chunk<WF, NM>& q, int c) {
        q.load_weights(o, c, nks);
        q.load_acts(o, c, nks);
    };
    int c = c0;
    if (c < c1) load(q0, c);
    for (; c + step < c1; c += 2 * step) {
        load(q1, c + step);
        __builtin_amdgcn_sched_barrier(0);
        q0.mma(c, nks, acc);
        if (c + 2 * step < c1) load(q0, c + 2 * step);
        __builtin_amdgcn_sched_barrier(0);
        q1.mma(c + step, nks, acc);
    }
    if (c < c1) q0.mma(c, nks, acc);
}

template <int WF>
__device__ __forceinline__ int chunks(int K) {
    return (K / 64 + Wt<WF>::UNIT - 1) / Wt<WF>::UNIT;
}

// int8: the scales of weight rows n0 + 4 g .. n0 + 4 g + 3 on an accumulator; other formats' are in it.
template <int WF>
__device__ __forceinline__ void row_scale(f32x4& acc, const void* scales, long long row, int lane) {
    if constexpr (WF == YVMOE_W_INT8) {
        const ushort4 s = *(const ushort4*)((const unsigned short*)scales + row + 4 * (lane >> 4));
        acc[0] = acc[0] * bf16_to_f32(s.x);
        acc[1] = acc[1] * bf16_to_f32(s.y);
        acc[2] = acc[2] * bf16_to_f32(s.z);
        acc[3] = acc[3] * bf16_to_f32(s.w);
    }
}

// Sum of the wavefronts' accumulators, in wavefront order.
template <int NM>
__device__ __forceinline__ void sum_waves(const f32x4 (&red)[kWaves][2][64], int lane, f32x4 (&sum)[NM]) {
#pragma unroll
    for (int m = 0; m < NM; ++m) {
        sum[m] = red[0][m][lane];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) {
            const f32x4 v = red[w][m][lane];
#pragma unroll
            for (int i = 0; i < 4; ++i) sum[m][i] = sum[m][i] + v[i];
        }
    }
}

// h of the lane's activation row and four columns from col, rounded once. PUBLISH: written through to
// where every XCD reads it.
template <int WF, bool PUBLISH>
__device__ __forceinline__ void store_h(void* h, long long row, int F, int col, const f32x4& g, const f32x4& u) {
    float v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = silu(g[i]) * u[i];
    unsigned long long w[2];
    char* p;
    constexpr int NW = WF == YVMOE_W_F32 ? 2 : 1;
    if constexpr (WF == YVMOE_W_F32) {
        p = (char*)h + (row * F + col) * 4;
#pragma unroll
        for (int i = 0; i < 2; ++i)
            w[i] = (unsigned long long)__float_as_uint(v[2 * i]) | (unsigned long long)__float_as_uint(v[2 * i + 1]) << 32;
    } else {
        p = (char*)h + (row * F + col) * 2;
        w[0] = (unsigned long long)pack_bf16(v[0], v[1]) | (unsigned long long)pack_bf16(v[2], v[3]) << 32;
    }
#pragma unroll
    for (int i = 0; i < NW; ++i) {
        if constexpr (PUBLISH)
            __hip_atomic_store((unsigned long long*)p + i, w[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        else
            ((unsigned long long*)p)[i] = w[i];
    }
}

// One gate/up item: 16 columns of F from n0 of expert e for n rows, the lane's activation row in
// token. The wavefronts deal out K; the wavefront that ends it writes h rows from row0.
template <int WF, bool PUBLISH>
__device__ __forceinline__ void gate_up_item(const FewArgs& a, int e, int n0, int token, int n, long long row0,
                                             f32x4 (&red)[kWaves][2][64], int wave, int lane, int closer) {
    Operands<WF, 2> o;
    o.set(0, a.w_gate, a.s_gate, e, a.F, a.H, n0, lane);
    o.set(1, a.w_up, a.s_up, e, a.F, a.H, n0, lane);
    o.rows(a.x, token, a.H, lane);
    f32x4 acc[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
    stream<WF, 2>(o, a.H / 64, wave, chunks<WF>(a.H), kWaves, acc);
    red[wave][0][lane] = acc[0];
    red[wave][1][lane] = acc[1];
    __syncthreads();
    if (wave != closer) return;
    f32x4 sum[2];
    sum_waves<2>(red, lane, sum);
    row_scale<WF>(sum[0], a.s_gate, (long long)e * a.F + n0, lane);
    row_scale<WF>(sum[1], a.s_up, (long long)e * a.F + n0, lane);
    const int r = lane & 15;
    if (r < n) store_h<WF, PUBLISH>(a.h, row0 + r, a.F, n0 + 4 * (lane >> 4), sum[0], sum[1]);
}

// ---------------------------------------------------------------- first kernel
// Work-groups: the router's (16 columns, K split) items, then the shared experts' gate/up items.
template <int WF>
__global__ __launch_bounds__(kThreads, 4) void few_front_kernel(FewArgs a) {
    constexpr int RF = WF == YVMOE_W_F32 ? YVMOE_W_F32 : YVMOE_W_BF16;
    __shared__ f32x4 red[kWaves][2][64];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 15;
    int b = blockIdx.x;
    if (b == 0 && threadIdx.x <= kRanges) a.counters[threadIdx.x * kCounterStride] = 0;
    const int nrouter = a.self ? a.ncols / 16 * a.nsplit : 0;
    if (b < nrouter) {
        const int n0 = b / a.nsplit * 16, z = b % a.nsplit, nch = chunks<RF>(a.H);
        Operands<RF, 1> o;
        o.set(0, a.w_router, nullptr, 0, a.ld, a.H, n0, lane);
        o.rows(a.x, min(r, a.N - 1), a.H, lane);
        f32x4 acc[1] = {f32x4{0.f, 0.f, 0.f, 0.f}};
        stream<RF, 1>(o, a.H / 64, z * nch / a.nsplit + wave, (z + 1) * nch / a.nsplit, kWaves, acc);
        red[wave][0][lane] = acc[0];
        __syncthreads();
        if (wave != 0 || r >= a.N) return;
        f32x4 sum[1];
        sum_waves<1>(red, lane, sum);
        *(f32x4*)(a.logits + ((long long)z * a.N + r) * a.ld + n0 + 4 * (lane >> 4)) = sum[0];
        return;
    }
    b -= nrouter;
    const int nfb = a.F / 16;
    if (b >= a.S * nfb) return;
    const int s = b / nfb;
    gate_up_item<WF, false>(a, a.E + s, b % nfb * 16, min(r, a.N - 1), a.N, (long long)a.N * (a.k + s), red, wave,
                            lane, 0);
}

// ---------------------------------------------------------------- second kernel
struct FewTables {
    short expert[kFewSlots];  // of each slot, -1: none
    float p[kFewSlots];       // its probability
    float w[kFewSlots];       // its weight
    short pos[kFewSlots];     // its row, -1: none
    short slot[kFewSlots];    // slot of each routed row
    short first[kFewSlots];   // a routed row's place among its expert's
    short tile_e[kFewTiles], tile_row0[kFewTiles], tile_n[kFewTiles];
    float score[kFewTokens];
    int counts[YVMOE_MAX_EXPERTS];
    int wave_starts[4];
    int nrows, ntiles, cap, item[2];
};

// The routing of up to 16 tokens, from the logits or as given, and the tiles: up to 16 rows of one
// expert each. Every work-group computes it; the first one also writes it out.
__device__ __forceinline__ void few_routing(const FewArgs& a, FewTables& t, bool writer) {
#pragma clang fp contract(off)
    const int tid = threadIdx.x, N = a.N, E = a.E, k = a.k, ns = N * k;
    if (tid == 0) {
        t.nrows = 0;
        t.cap = -1;
    }
    for (int e = tid; e < YVMOE_MAX_EXPERTS; e += kThreads) t.counts[e] = 0;
    if (a.self) {
        const long long sstride = (long long)N * a.ld;
        if (tid < 16 * N) {  // 16 lanes a token
            const int tok = tid / kLanes, l = tid % kLanes;
            const float* lg = a.logits + (long long)tok * a.ld;
            auto logit = [&](int e) {
                float v = lg[e];
                for (int z = 1; z < a.nsplit; ++z) v = v + lg[z * sstride + e];
                return v;
            };
            int id;
            float p, w;
            if (E <= 64) topk_token<4>(logit, a.bias, l, E, k, id, p, w);
            else topk_token<16>(logit, a.bias, l, E, k, id, p, w);
            if (l < k) {
                t.expert[tok * k + l] = id < E ? (short)id : -1;
                t.p[tok * k + l] = p;
                t.w[tok * k + l] = w;
                if (writer) a.out_routing.indices[tok * k + l] = id;
            }
        }
        const int pt = tid - 256;
        if (a.cap_mode == 2 && pt >= 0 && pt < 16 * N) {
            const int tok = pt / kLanes;
            const float* pr = a.logits + (long long)tok * a.ld + (E + 15) / 16 * 16;
            const int terms = (a.ld - (E + 15) / 16 * 16) / kPredDim;
            const float sc = predictor_token([&](int c) {
                float v = pr[c];
                for (int z = 1; z < a.nsplit; ++z) v = v + pr[z * sstride + c];
                return v;
            }, terms, a.b1, a.w2, a.b2, pt % kLanes);
            if (pt % kLanes == 0) t.score[tok] = sc;
        }
    } else if (tid < ns) {
        const int64_t id = a.rindices[tid];
        t.expert[tid] = id >= 0 && id < E ? (short)id : -1;
        t.w[tid] = a.rweights_bf16 ? bf16_to_f32(((const unsigned short*)a.rweights)[tid])
                                   : ((const float*)a.rweights)[tid];
    }
    __syncthreads();
    if (tid == 0 && a.self && a.cap_mode != 0) {
        // capacity (gate.py:1096-1120) in double, the scores' mean in fp32 in token order
        double cf = a.cap_factor;
        if (a.cap_mode == 2 && N > 0) {
            float sum = 0.0f;
            for (int i = 0; i < N; ++i) sum = sum + t.score[i];
            cf = 0.5 + 1.5 * (double)(sum / (float)N);
            cf = cf > 2.0 ? 2.0 : cf < 0.5 ? 0.5 : cf;
        }
        const int cap = (int)((double)N * cf / (double)E);
        t.cap = cap < a.min_cap || N == 0 ? a.min_cap : cap;
    }
    // a slot's row: after all slots of lower experts and the earlier ones of its own
    int mine = -1, before = 0, better = 0;
    if (tid < ns) {
        mine = t.expert[tid];
        const float p = a.self ? t.p[tid] : 0.0f;
        int pos = 0;
        if (mine >= 0) {
            for (int s = 0; s < ns; ++s) {
                const int e = t.expert[s];
                pos += e >= 0 && e < mine ? 1 : 0;
                if (e == mine) {
                    before += s < tid ? 1 : 0;
                    if (a.self) better += t.p[s] > p || (t.p[s] == p && s < tid) ? 1 : 0;
                }
            }
            pos += before;
            t.slot[pos] = (short)tid;
            t.first[pos] = (short)before;
            atomicAdd(&t.counts[mine], 1);
            atomicAdd(&t.nrows, 1);
        }
        t.pos[tid] = mine >= 0 ? (short)pos : (short)-1;
    }
    __syncthreads();
    // the trim (gate.py:1228-1236): an expert keeps its cap slots of the highest probability
    if (t.cap >= 0 && mine >= 0 && better >= t.cap) t.w[tid] = 0.0f;
    const int nrows = t.nrows;
    bool start = false;
    int below = 0;
    if (tid < kFewSlots) {
        start = tid < nrows && (t.first[tid] & 15) == 0;
        const unsigned long long m = __ballot(start);
        below = __popcll(m & ((1ull << (tid & 63)) - 1ull));
        if ((tid & 63) == 0) t.wave_starts[tid >> 6] = __popcll(m);
    }
    __syncthreads();
    if (a.self && a.cap_mode != 0 && tid < N) {  // renormalised (gate.py:1239-1241), a thread a token
        float tot = 0.0f;
        for (int j = 0; j < k; ++j) tot = tot + t.w[tid * k + j];
        const float den = tot > 1e-8f ? tot : 1e-8f;
        for (int j = 0; j < k; ++j) t.w[tid * k + j] = t.w[tid * k + j] / den;
    }
    if (start) {
        int i = below;
        for (int w = 0; w < (tid >> 6); ++w) i += t.wave_starts[w];
        const int e = t.expert[t.slot[tid]];
        t.tile_e[i] = (short)e;
        t.tile_row0[i] = (short)tid;
        t.tile_n[i] = (short)min(16, t.counts[e] - t.first[tid]);
    }
    if (tid < a.S) {
        const int i = t.wave_starts[0] + t.wave_starts[1] + t.wave_starts[2] + t.wave_starts[3] + tid;
        t.tile_e[i] = (short)(E + tid);
        t.tile_row0[i] = (short)(ns + tid * N);
        t.tile_n[i] = (short)N;
    }
    if (tid == 0) t.ntiles = t.wave_starts[0] + t.wave_starts[1] + t.wave_starts[2] + t.wave_starts[3];
    __syncthreads();
    if (!writer) return;
    if (!a.self) {
        if (tid == 0 && a.invalid != nullptr) *a.invalid = ns - nrows;
        return;
    }
    const yvmoe_routing& o = a.out_routing;
    if (tid < ns) {
        o.weights[tid] = t.w[tid];
        o.pos[tid] = t.pos[tid];
        if (t.pos[tid] >= 0) o.perm[t.pos[tid]] = tid;
    }
    if (tid < E) {
        int off = 0;
        for (int e = 0; e < tid; ++e) off += t.counts[e];
        o.counts[tid] = t.counts[tid];
        o.offsets[tid] = off;
        if (tid == E - 1) o.offsets[E] = off + t.counts[tid];
    }
    if (tid == 0) *o.capacity = t.cap;
}

// How many parts of K each tile's down product is cut into, so that the wavefronts end together:
// the fewest with the least work of the busiest wavefront.
__device__ __forceinline__ int down_parts(int tiles, int rows, int nch) {
    int best = 1, cost = (tiles + kWaves - 1) / kWaves * 840;  // 840: a multiple of 1 .. 8
    for (int q = 2; q <= 8; ++q) {
        const int c = (tiles * q + kWaves - 1) / kWaves * (840 / q);
        if (c < cost && q * rows <= kYRows && q <= nch) {
            best = q;
            cost = c;
        }
    }
    return best;
}

template <int WF>
__global__ __launch_bounds__(kThreads, 4) void few_experts_kernel(FewArgs a) {
    constexpr bool F32 = WF == YVMOE_W_F32;
    __shared__ FewTables t;
    __shared__ union {
        f32x4 red[2][kWaves][2][64];
        float y[kYRows][16];
    } u;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = lane & 15;
    few_routing(a, t, blockIdx.x == 0);
    if (a.N == 0) return;
    const int ns = a.N * a.k;

    // gate/up: the items' ranges, one per XCD, taken by its work-groups first
    const int nfb = a.F / 16, nitems = t.ntiles * nfb;
    int range = blockIdx.x % kRanges, done = 0;
    auto range_start = [&](int i) { return (int)((long long)nitems * i / kRanges); };
    auto take = [&]() {  // thread 0: the next item, -1: none left
        for (int i = 0; i < kRanges; ++i) {
            const int n = range_start(range + 1) - range_start(range);
            const int got = __hip_atomic_fetch_add(a.counters + range * kCounterStride, 1, __ATOMIC_RELAXED,
                                                   __HIP_MEMORY_SCOPE_AGENT);
            if (got < n) return range_start(range) + got;
            range = (range + 1) % kRanges;
        }
        return -1;
    };
    if (tid == 0) t.item[0] = take();
    __syncthreads();
    for (int it = 0;; ++it) {
        const int item = __builtin_amdgcn_readfirstlane(t.item[it & 1]);
        if (item < 0) break;
        if (tid == 0) t.item[(it + 1) & 1] = take();
        const int tile = item / nfb, n0 = item % nfb * 16;
        const int e = t.tile_e[tile], row0 = t.tile_row0[tile], n = t.tile_n[tile];
        const int token = t.slot[row0 + min(r, n - 1)] / a.k;
        gate_up_item<WF, true>(a, e, n0, token, n, row0, u.red[it & 1], wave, lane, it & (kWaves - 1));
        ++done;
    }
    // h is written through; once this work-group's stores are there, say so
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    int* flag = a.counters + kRanges * kCounterStride;
    if (tid == 0) {
        if (done > 0) __hip_atomic_fetch_add(flag, done, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        int ok = 0;
        for (int i = 0; i < kSpinLimit && !ok; ++i) {
            ok = __hip_atomic_load(flag, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == nitems;
            if (!ok) __builtin_amdgcn_s_sleep(2);
        }
        t.item[0] = ok;
    }
    __syncthreads();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");
    const bool ok = t.item[0] != 0;

    // down: 16 columns of H of every tile, the units (tile, part of K) dealt out to the wavefronts
    const int ntiles = t.ntiles + a.S, nrows = ns + a.S * a.N, nch = chunks<WF>(a.F);
    const int parts = down_parts(ntiles, nrows, nch);
    for (int hb = blockIdx.x; hb < a.H / 16; hb += gridDim.x) {
        const int n0 = hb * 16;
        for (int unit = wave; unit < ntiles * parts; unit += kWaves) {
            const int tile = unit / parts, q = unit % parts;
            const int e = t.tile_e[tile], row0 = t.tile_row0[tile], n = t.tile_n[tile];
            Operands<WF, 1> o;
            o.set(0, a.w_down, a.s_down, e, a.H, a.F, n0, lane);
            o.rows(a.h, row0 + min(r, n - 1), a.F, lane);
            f32x4 acc[1] = {f32x4{0.f, 0.f, 0.f, 0.f}};
            stream<WF, 1>(o, a.F / 64, q * nch / parts, (q + 1) * nch / parts, 1, acc);
            row_scale<WF>(acc[0], a.s_down, (long long)e * a.H + n0, lane);
            if (r < n) *(f32x4*)&u.y[q * nrows + row0 + r][4 * (lane >> 4)] = acc[0];
        }
        __syncthreads();
        if (tid < 16 * a.N) {
            const int tok = tid / 16, c = tid % 16;
            auto row = [&](int i) {
                float v = u.y[i][c];
                for (int q = 1; q < parts; ++q) v = v + u.y[q * nrows + i][c];
                return v;
            };
            float v = 0.0f;
            for (int j = 0; j < a.k; ++j) {
                const int p = t.pos[tok * a.k + j];
                if (p >= 0) v = v + t.w[tok * a.k + j] * row(p);
                else if (a.self) v = __builtin_nanf("");  // logits that are not numbers choose nothing
            }
            const long long at = (long long)tok * a.H + n0 + c;
            float sh = 0.0f;
            for (int s = 0; s < a.S; ++s) sh = sh + a.mix[s] * row(ns + s * a.N + tok);
            v = v + sh;
            if (a.skip != nullptr)
                v = v + 0.1f * (F32 ? ((const float*)a.skip)[at] : bf16_to_f32(((const unsigned short*)a.skip)[at]));
            if (!ok) v = __builtin_nanf("");
            if constexpr (F32) {
                ((float*)a.out)[at] = v;
                if (a.shared_out != nullptr) ((float*)a.shared_out)[at] = sh;
            } else {
                ((unsigned short*)a.out)[at] = f32_to_bf16_rne(v);
                if (a.shared_out != nullptr) ((unsigned short*)a.shared_out)[at] = f32_to_bf16_rne(sh);
            }
        }
        __syncthreads();
    }
}

}  // namespace

int few_launch(const void* x, int act, int N, int k, const yvmoe_router* r, const void* rweights, int rweights_bf16,
               const int64_t* rindices, const yvmoe_expert_weights* w, const float* mix, const void* skip, void* out,
               void* shared_out, const yvmoe_routing* routing, int* invalid, char* ws, hipStream_t st) {
    const int E = w->num_routed, S = w->num_shared, H = w->hidden, F = w->ffn;
    const FewWs L = few_ws(N, k, E, S, H, F, act);
    FewArgs a{};
    a.x = x;
    a.N = N, a.H = H, a.F = F, a.E = E, a.S = S, a.k = k;
    a.w_gate = w->w_gate, a.w_up = w->w_up, a.w_down = w->w_down;
    a.s_gate = w->s_gate, a.s_up = w->s_up, a.s_down = w->s_down;
    a.self = r != nullptr;
    a.logits = (float*)(ws + L.logits);
    if (r != nullptr) {
        a.w_router = r->w_router;
        a.cap_mode = r->fixed_shape_mode ? 0 : r->dynamic_capacity ? 2 : 3;
        a.ld = router_ld(E, act);
        a.ncols = a.cap_mode == 2 ? a.ld : pad16(E);  // the predictor's columns only where it decides
        a.nsplit = few_splits(H);
        a.bias = r->bias, a.b1 = r->b1, a.w2 = r->w2, a.b2 = r->b2;
        a.min_cap = r->min_capacity;
        a.cap_factor = r->capacity_factor;
        a.out_routing = *routing;
    }
    a.rweights = rweights, a.rweights_bf16 = rweights_bf16, a.rindices = rindices;
    a.invalid = invalid;
    a.mix = mix, a.skip = skip, a.out = out, a.shared_out = shared_out;
    a.h = ws + L.h;
    a.counters = (int*)(ws + L.counters);
    const int front = (a.self ? a.ncols / 16 * a.nsplit : 0) + S * (F / 16);
    // two work-groups per CU, fewer where neither half has work for them
    const int items = std::max(std::min(N * k, E) * (F / 16), H / 16);
    const int grid = N == 0 ? 1 : std::min(512, items);
#define YV_FEW(WFV)                                                                          \
    do {                                                                                     \
        if (N > 0) {                                                                         \
            few_front_kernel<WFV><<<std::max(front, 1), kThreads, 0, st>>>(a);               \
            YV_LAUNCH_CHECK("few_front");                                                    \
        }                                                                                    \
        few_experts_kernel<WFV><<<grid, kThreads, 0, st>>>(a);                               \
        YV_LAUNCH_CHECK("few_experts");                                                      \
    } while (0)
    switch (w->format) {
        case YVMOE_W_F32: YV_FEW(YVMOE_W_F32); break;
        case YVMOE_W_BF16: YV_FEW(YVMOE_W_BF16); break;
        case YVMOE_W_INT8: YV_FEW(YVMOE_W_INT8); break;
        case YVMOE_W_INT4: YV_FEW(YVMOE_W_INT4); break;
        case YVMOE_W_FP8: YV_FEW(YVMOE_W_FP8); break;
        default: set_error("unknown weight format %d", w->format); return YVMOE_ERR_DTYPE;
    }
#undef YV_FEW
    return YVMOE_OK;
}

}  // namespace yvmoe
