// Linear layer with 4-bit weights and a scale per 128 columns of a row, for gfx950.
//
//   y[n][o] = Σ_i x[n][i] (q[o][i] - 8) s[o][i / 128] + b[o]
//
// (model/utils/quantization.py:486-496 with the codes of opss/quantize/engine.py:889-941.)
//
// Products. v_mfma_f32_16x16x32_bf16 with 16 rows of x as first and 16 weight rows as second operand:
// lane l = 16 g + r holds 8 columns of x row r and of weight row r, the accumulator x rows 4 g + i of
// weight row r, so that a row's scales stay in the lanes that hold its codes. A byte of value q < 16 is the
// e4m3 number q / 512, so two codes cost a conversion to bf16 and a share of the masks; Σ x q / 512 over a
// group, plus -8 / 512 Σ x from MFMAs with a constant operand, is Σ x (q - 8) / 512, all exact products in
// fp32 sums. 512 s multiplies that sum, so nothing is rounded before y. fp32 rows of x go in as three bf16
// terms, which hold all 24 bits.
//
// Storage (include/yvmoe.h): per 16 rows and 128 columns 1 KB, lane l's 16 bytes at 16 l: columns
// 32 g .. 32 g + 31 of row r, a dword eight of them, its bytes' lower nibbles columns 0 .. 3, their upper
// nibbles columns 4 .. 7, which gives an operand's pairs in order.
//
// Forms. Rows that fit into LDS, up to 16: int4_few_kernel, bound by the stream of codes (out·in / 2 bytes: 1 x
// 4096 x 100003 in 38 us, 5.6 TB/s) and at small sizes by one trip to memory. Else int4_rows_kernel, bound by
// what a CU gets from L2 while rows are few (each work-group reads them all: 48 x 5120 x 8192 in 16 us), then
// by the instructions that make operands of codes (4096 x 8192 x 8192: 927 TFLOP/s).
#include <algorithm>

#include "yvmoe_frag.h"
#include "yvmoe_internal.h"
#include "yvmoe_linear_stream.h"

namespace yvmoe {
namespace {

constexpr int kGroup = 128;

struct LinArgs {
    const void* x;
    int N, K, O, groups, blocks;   // blocks of 16 outputs
    const char* codes;             // [blocks][groups][1 KB]
    const unsigned short* scales;  // [blocks][groups][16]
    const void* bias;
    void* out;
};

// 16 bytes from any address.
struct __attribute__((packed, aligned(2))) Any16 {
    unsigned v[4];
};
__device__ __forceinline__ uint4 load_any16(const void* p) {
    const Any16 a = *(const Any16*)p;
    return make_uint4(a.v[0], a.v[1], a.v[2], a.v[3]);
}

union Frag8 {
    uint4 u;
    bf16x8 v;
};

// The eight weights of a dword, q / 512.
__device__ __forceinline__ bf16x8 codes8(unsigned w) {
    const int lo = (int)(w & 0x0F0F0F0Fu), hi = (int)(w >> 4 & 0x0F0F0F0Fu);
    Frag8 f;
    f.u = make_uint4(__builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false)),
                     __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true)),
                     __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false)),
                     __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true)));
    return f.v;
}
__device__ __forceinline__ bf16x8 minus8() {  // -8 / 512
    Frag8 f;
    f.u = make_uint4(0xBC80BC80u, 0xBC80BC80u, 0xBC80BC80u, 0xBC80BC80u);
    return f.v;
}
__device__ __forceinline__ float scale512(unsigned short s) { return 512.0f * bf16_to_f32(s); }
__device__ __forceinline__ f32x4 mfma16(const bf16x8& a, const bf16x8& b, const f32x4& c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// Eight elements of x. The load is free of branches, so that it can stay in flight: callers let it start 8
// before the end of x at the latest, and it may run into the next row; fix() then moves the elements to their
// places and clears those from `valid` on. load_tiny: for an x of fewer than eight elements.
__device__ __forceinline__ unsigned pick(bool c, unsigned a, unsigned b) { return c ? a : b; }
template <bool F32>
struct X8;
template <>
struct X8<false> {
    static constexpr int TERMS = 1;
    uint4 v;
    __device__ __forceinline__ void load(const void* x, size_t at) { v = load_any16((const unsigned short*)x + at); }
    __device__ __forceinline__ void load_tiny(const void* x, int at, int total) {
        const unsigned short* p = (const unsigned short*)x;
        unsigned d[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
            d[i] = (at + 2 * i < total ? p[at + 2 * i] : 0) |
                   (unsigned)(at + 2 * i + 1 < total ? p[at + 2 * i + 1] : 0) << 16;
        v = make_uint4(d[0], d[1], d[2], d[3]);
    }
    __device__ __forceinline__ void fix(int shift, int valid) {
        unsigned d[5] = {v.x, v.y, v.z, v.w, 0};
#pragma unroll
        for (int i = 0; i < 4; ++i) d[i] = pick(shift & 1, d[i] >> 16 | d[i + 1] << 16, d[i]);
#pragma unroll
        for (int i = 0; i < 4; ++i) d[i] = pick(shift & 2, d[i + 1], d[i]);
#pragma unroll
        for (int i = 0; i < 4; ++i) d[i] = pick(shift & 4, i < 2 ? d[i + 2] : 0u, d[i]);
#pragma unroll
        for (int i = 0; i < 4; ++i) d[i] = pick(valid >= 2 * i + 2, d[i], pick(valid == 2 * i + 1, d[i] & 0xffffu, 0u));
        v = make_uint4(d[0], d[1], d[2], d[3]);
    }
    __device__ __forceinline__ void terms(bf16x8 (&t)[1]) const {
        Frag8 f;
        f.u = v;
        t[0] = f.v;
    }
};
template <>
struct X8<true> {
    static constexpr int TERMS = 3;
    uint4 v[2];
    __device__ __forceinline__ void load(const void* x, size_t at) {
        v[0] = load_any16((const unsigned*)x + at);
        v[1] = load_any16((const unsigned*)x + at + 4);
    }
    __device__ __forceinline__ void load_tiny(const void* x, int at, int total) {
        const unsigned* p = (const unsigned*)x;
        unsigned d[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) d[i] = at + i < total ? p[at + i] : 0u;
        v[0] = make_uint4(d[0], d[1], d[2], d[3]);
        v[1] = make_uint4(d[4], d[5], d[6], d[7]);
    }
    __device__ __forceinline__ void fix(int shift, int valid) {
        unsigned d[8] = {v[0].x, v[0].y, v[0].z, v[0].w, v[1].x, v[1].y, v[1].z, v[1].w};
#pragma unroll
        for (int bit = 1; bit < 8; bit *= 2)
#pragma unroll
            for (int i = 0; i < 8; ++i) d[i] = pick(shift & bit, i + bit < 8 ? d[i + bit] : 0u, d[i]);
#pragma unroll
        for (int i = 0; i < 8; ++i) d[i] = pick(i < valid, d[i], 0u);
        v[0] = make_uint4(d[0], d[1], d[2], d[3]);
        v[1] = make_uint4(d[4], d[5], d[6], d[7]);
    }
    // Three bf16 terms, each the rest's rounding: their sum has 24 bits, as x has.
    __device__ __forceinline__ void terms(bf16x8 (&t)[3]) const {
        const unsigned w[8] = {v[0].x, v[0].y, v[0].z, v[0].w, v[1].x, v[1].y, v[1].z, v[1].w};
        float rest[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) rest[i] = __uint_as_float(w[i]);
#pragma unroll
        for (int q = 0; q < 3; ++q) {
            unsigned d[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                d[i] = pack_bf16(rest[2 * i], rest[2 * i + 1]);
                rest[2 * i] = rest[2 * i] - __uint_as_float(d[i] << 16);
                rest[2 * i + 1] = rest[2 * i + 1] - __uint_as_float(d[i] & 0xffff0000u);
            }
            Frag8 f;
            f.u = make_uint4(d[0], d[1], d[2], d[3]);
            t[q] = f.v;
        }
    }
};

template <bool F32>
__device__ __forceinline__ void put(const LinArgs& a, int n, int o, float v) {
    const long long at = (long long)n * a.O + o;
    if constexpr (F32) {
        if (a.bias != nullptr) v = v + ((const float*)a.bias)[o];
        ((float*)a.out)[at] = v;
    } else {
        if (a.bias != nullptr) v = v + bf16_to_f32(((const unsigned short*)a.bias)[o]);
        ((unsigned short*)a.out)[at] = f32_to_bf16_rne(v);
    }
}

// ---------------------------------------------------------------- rows that fit into LDS
// A work-group keeps all rows of x in LDS (as bf16 terms) beside each group's -8 / 512 Σ x, and computes 16 RB
// outputs at a time; its eight wavefronts deal out the groups of K. A wavefront's stream of codes runs on
// over the ends of outputs, D - 1 groups ahead.
//   LDS: x [T][N][stride] | corrections [groups][16] fp32 | sums [2][7][RB][64 x 16 B]
struct FewLds {
    int stride, corr, sums, bytes;
};
__host__ __device__ inline FewLds few_lds(int N, int groups, int terms, int rb) {
    FewLds l;
    l.stride = groups * kGroup * 2 + 16;  // the 16 rows of an operand fall on different banks
    l.corr = terms * N * l.stride;
    l.sums = l.corr + groups * 64;
    l.bytes = l.sums + 2 * 7 * rb * 1024;
    return l;
}

template <bool F32, int RB, int D, bool TINY>
__global__ __launch_bounds__(512, 4) void int4_few_kernel(LinArgs a) {
    constexpr int T = X8<F32>::TERMS;
    extern __shared__ __align__(16) char lds[];
    const FewLds l = few_lds(a.N, a.groups, T, RB);
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int g = lane >> 4, r = lane & 15;
    struct W {
        uint4 w[RB];
        unsigned short s[RB];
    };
    CodeStream<RB> ahead(a.blocks, a.groups, wave, blockIdx.x, gridDim.x);
    const int items = ahead.items;
    auto load_w = [&](W& q) {  // after the last group: that one again, not used
#pragma unroll
        for (int b = 0; b < RB; ++b) {
            const long long at = ahead.at(b);
            q.w[b] = nt_load16(a.codes + at * 1024 + lane * 16);
            q.s[b] = a.scales[at * 16 + r];
        }
        ahead.next();
    };
    W q[D];
#pragma unroll
    for (int d = 0; d + 1 < D; ++d) load_w(q[d]);
    const char* xr = lds + min(r, a.N - 1) * l.stride + 64 * g;
    float* corrs = (float*)(lds + l.corr);
    auto operand = [&](int k, int kg, int j) {
        Frag8 f;
        f.u = *(const uint4*)&xr[k * a.N * l.stride + kg * 256 + 16 * j];
        return f.v;
    };
    {
        constexpr int BATCH = 4;
        const int per_row = a.groups * 16, pieces = a.N * per_row;
        const int total = a.N * a.K;  // fits LDS
        for (int p0 = tid; p0 < pieces; p0 += 512 * BATCH) {
            X8<F32> px[BATCH];
            int row[BATCH], c[BATCH];
#pragma unroll
            for (int i = 0; i < BATCH; ++i) {
                const int p = min(p0 + 512 * i, pieces - 1);
                row[i] = p / per_row, c[i] = p % per_row * 8;
                const int at = row[i] * a.K + c[i];
                if constexpr (TINY) px[i].load_tiny(a.x, at, total);
                else px[i].load(a.x, min(at, total - 8));
            }
#pragma unroll
            for (int i = 0; i < BATCH; ++i) {
                if (p0 + 512 * i >= pieces) continue;
                if (c[i] + 8 > a.K) {
                    const int at = row[i] * a.K + c[i];
                    px[i].fix(TINY ? 0 : min(at - min(at, total - 8), 7), a.K - c[i]);
                }
                bf16x8 t[T];
                px[i].terms(t);
#pragma unroll
                for (int k = 0; k < T; ++k) {
                    Frag8 f;
                    f.v = t[k];
                    *(uint4*)&lds[(k * a.N + row[i]) * l.stride + c[i] * 2] = f.u;
                }
            }
        }
    }
    __syncthreads();
    for (int kg = wave; kg < a.groups; kg += 8) {  // each wavefront the groups that it will use
        f32x4 corr = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int k = 0; k < T; ++k) corr = mfma16(operand(k, kg, j), minus8(), corr);
        if (r == 0) *(f32x4*)&corrs[kg * 16 + 4 * g] = corr;
    }
    f32x4 acc[RB];
#pragma unroll
    for (int b = 0; b < RB; ++b) acc[b] = f32x4{0.f, 0.f, 0.f, 0.f};
    auto group = [&](const W& q, W& qn, int kg) {
        load_w(qn);
        f32x4 part[RB];
#pragma unroll
        for (int b = 0; b < RB; ++b) part[b] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            bf16x8 v[T];
#pragma unroll
            for (int k = 0; k < T; ++k) v[k] = operand(k, kg, j);
#pragma unroll
            for (int b = 0; b < RB; ++b) {
                const unsigned d[4] = {q.w[b].x, q.w[b].y, q.w[b].z, q.w[b].w};
                const bf16x8 c = codes8(d[j]);
#pragma unroll
                for (int k = 0; k < T; ++k) part[b] = mfma16(v[k], c, part[b]);
            }
        }
        const f32x4 corr = *(const f32x4*)&corrs[kg * 16 + 4 * g];
#pragma unroll
        for (int b = 0; b < RB; ++b) {
            const float s = scale512(q.s[b]);
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[b][i] = __builtin_fmaf(s, part[b][i] + corr[i], acc[b][i]);
        }
    };
    // The end of an item: the wavefronts take turns in adding up the eight sums. They lie in one of two
    // places in turn, so that one barrier parts the writes of an item from the reads, and these from the
    // writes two items on.
    auto finish = [&](int item) {
        f32x4* place = (f32x4*)(lds + l.sums) + (item & 1) * 7 * RB * 64 + lane;
        const int owner = item & 7, slot = (wave - owner - 1) & 7;
        if (slot < 7)
#pragma unroll
            for (int b = 0; b < RB; ++b) place[(slot * RB + b) * 64] = acc[b];
        __syncthreads();
        if (slot == 7) {
            const int set = (int)blockIdx.x + item * (int)gridDim.x;
#pragma unroll
            for (int b = 0; b < RB; ++b) {
                f32x4 sum = acc[b];
#pragma unroll
                for (int w = 0; w < 7; ++w) {
                    const f32x4 v = place[(w * RB + b) * 64];
#pragma unroll
                    for (int e = 0; e < 4; ++e) sum[e] = sum[e] + v[e];
                }
                const int o = (set * RB + b) * 16 + r;
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (o < a.O && 4 * g + e < a.N) put<F32>(a, 4 * g + e, o, sum[e]);
            }
        }
#pragma unroll
        for (int b = 0; b < RB; ++b) acc[b] = f32x4{0.f, 0.f, 0.f, 0.f};
    };
    if (wave >= a.groups) {
        for (int item = 0; item < items; ++item) finish(item);
        return;
    }
    for (int item = 0, kg = wave;;) {
#pragma unroll
        for (int d = 0; d < D; ++d) {
            group(q[d], q[(d + D - 1) % D], kg);
            kg += 8;
            if (kg >= a.groups) {
                kg = wave;
                finish(item);
                if (++item == items) return;
            }
        }
    }
}

// ---------------------------------------------------------------- more rows
// A work-group of WO x WT x WK wavefronts computes 16 RB WO outputs of 16 TB WT rows, WK groups of K at a time.
// The rows' columns go through LDS (as bf16 terms, two stages, padded by 16 bytes so that the 16 rows of an
// operand fall on different banks), loaded a step ahead; the codes go straight to the wavefront that converts
// them, D - 1 steps ahead, once for the TB MFMAs of every term. The sums of the WK wavefronts meet in LDS.
//
// FOLD: with 64 x 64 products per wavefront the MFMAs of -8 / 512 Σ x would be a fifth of all. There the
// wavefronts that share rows share them, and every 32 groups Σ_groups 512 s (-8 / 512 Σ x) is one more product, with
// the scales (bf16 after the factor too) as one operand and the sums in three bf16 terms (24 bits) as the other
// (the factor on the scales, as elsewhere, so that large rows overflow here no sooner than there). That takes
// the additions out of the group's end as well: 8192 x 8192 at 4096 rows 672 -> 593 us (927 TFLOP/s), and
// slower where a wavefront has 64 x 16 (100 x 4096 x 28672: 59 -> 68 us).
template <bool F32, int TB, int RB, int WO, int WT, int D, int ROWS>
__global__ __launch_bounds__(512, 2) void int4_rows_kernel(LinArgs a) {
    constexpr int WK = 8 / WO / WT;
    constexpr int T = X8<F32>::TERMS, STRIDE = kGroup * 2 + 16;
    constexpr int PER = ROWS * WK * 16 / 512;  // pieces of 8 columns that a thread brings
    __shared__ __align__(16) char xs[2][T][WK * ROWS * STRIDE];
    constexpr bool FOLD = !F32 && WK == 1 && TB == WO && RB == 4;
    constexpr int SUMS = 32, SUMLD = SUMS + 4;
    __shared__ __align__(16) float sums[FOLD ? ROWS * SUMLD : 4];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int g = lane >> 4, r = lane & 15;
    const int wr = wave % WO, wt = wave / WO % WT, wk = wave / (WO * WT);
    // blocks of rows fastest: work-groups that run together share their codes
    const int nrt = (a.N + ROWS - 1) / ROWS;
    const int n0 = (int)(blockIdx.x % nrt) * ROWS, b0 = ((int)(blockIdx.x / nrt) * WO + wr) * RB;
    const char* codes[RB];
    const unsigned short* scales[RB];
#pragma unroll
    for (int b = 0; b < RB; ++b) {
        const long long at = (long long)min(b0 + b, a.blocks - 1) * a.groups;
        codes[b] = a.codes + at * 1024 + lane * 16;
        scales[b] = a.scales + at * 16 + r;
    }
    struct W {
        uint4 w[RB];
        unsigned short s[RB];
    };
    auto load_w = [&](W& q, int step) {  // groups past the end: the last one's, not used
        const int kg = min(step * WK + wk, a.groups - 1);
#pragma unroll
        for (int b = 0; b < RB; ++b) {
            q.w[b] = *(const uint4*)(codes[b] + (long long)kg * 1024);
            q.s[b] = scales[b][(long long)kg * 16];
        }
    };
    // x from an element near the tile's first one on, so that 32 bits hold the rest of an address
    const long long total = (long long)a.N * a.K, first = (long long)n0 * a.K;
    const long long base = first < total - 8 ? first : total - 8;
    const unsigned last = (unsigned)min(total - 8 - base, 0xFFFFFFFFLL);
    const char* xb = (const char*)a.x + base * (F32 ? 4 : 2);
    unsigned at[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int piece = tid + 512 * i, row = piece / (16 * WK), c = piece % (16 * WK);
        at[i] = (unsigned)(first - base) + (unsigned)min(row, a.N - 1 - n0) * a.K + 8 * c;
    }
    X8<F32> px[PER];
    auto load_x = [&](int step) {
#pragma unroll
        for (int i = 0; i < PER; ++i) px[i].load(xb, min(at[i] + step * (WK * kGroup), last));
    };
    auto store_x = [&](int step) {
        if ((step + 1) * (WK * kGroup) > a.K) {
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                const unsigned from = at[i] + step * (WK * kGroup);
                const int c = (tid + 512 * i) % (16 * WK) * 8 + step * (WK * kGroup);
                px[i].fix((int)min(from - min(from, last), 7u), a.K - c);
            }
        }
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int piece = tid + 512 * i, row = piece / (16 * WK), c = piece % (16 * WK);
            bf16x8 t[T];
            px[i].terms(t);
#pragma unroll
            for (int q = 0; q < T; ++q) {
                Frag8 f;
                f.v = t[q];
                *(uint4*)&xs[step & 1][q][(c / 16 * ROWS + row) * STRIDE + 16 * (c % 16)] = f.u;
            }
        }
    };
    f32x4 acc[RB][TB];
#pragma unroll
    for (int b = 0; b < RB; ++b)
#pragma unroll
        for (int t = 0; t < TB; ++t) acc[b][t] = f32x4{0.f, 0.f, 0.f, 0.f};
    // acc += 512 s (-8 / 512 Σ x) over n groups
    auto fold = [&](int g0, int n) {
        bf16x8 sc[RB];
#pragma unroll
        for (int b = 0; b < RB; ++b) {
            float e[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) e[i] = scale512(scales[b][(long long)min(g0 + 8 * g + i, a.groups - 1) * 16]);
            Frag8 f;
            f.u = make_uint4(pack_bf16(e[0], e[1]), pack_bf16(e[2], e[3]), pack_bf16(e[4], e[5]), pack_bf16(e[6], e[7]));
            sc[b] = f.v;
        }
#pragma unroll
        for (int t = 0; t < TB; ++t) {
            const float* p = &sums[((wt * TB + t) * 16 + r) * SUMLD + 8 * g];
            X8<true> x;
            x.v[0] = *(const uint4*)p, x.v[1] = *(const uint4*)(p + 4);
            x.fix(0, n - 8 * g);
            bf16x8 v[3];
            x.terms(v);
#pragma unroll
            for (int b = 0; b < RB; ++b)
#pragma unroll
                for (int k = 0; k < 3; ++k) acc[b][t] = mfma16(v[k], sc[b], acc[b][t]);
        }
    };
    auto group = [&](const W& q, W& qn, int step) {
        load_x(step + 1);
        load_w(qn, step + D - 1);
        if constexpr (FOLD) {
            auto operand = [&](int t, int j) {
                Frag8 f;
                f.u = *(const uint4*)&xs[step & 1][0][((wt * TB + t) * 16 + r) * STRIDE + 64 * g + 16 * j];
                return f.v;
            };
            f32x4 sum = {0.f, 0.f, 0.f, 0.f};  // wavefront wr's share of the rows
#pragma unroll
            for (int j = 0; j < 4; ++j) sum = mfma16(operand(wr, j), minus8(), sum);
            f32x4 part[RB][TB];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                bf16x8 c[RB], v[TB];
#pragma unroll
                for (int t = 0; t < TB; ++t) v[t] = operand(t, j);
#pragma unroll
                for (int b = 0; b < RB; ++b) {
                    const unsigned d[4] = {q.w[b].x, q.w[b].y, q.w[b].z, q.w[b].w};
                    c[b] = codes8(d[j]);
                }
#pragma unroll
                for (int b = 0; b < RB; ++b)
#pragma unroll
                    for (int t = 0; t < TB; ++t)
                        part[b][t] = mfma16(v[t], c[b], j == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : part[b][t]);
            }
#pragma unroll
            for (int b = 0; b < RB; ++b) {
                const float s = scale512(q.s[b]);
#pragma unroll
                for (int t = 0; t < TB; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[b][t][i] = __builtin_fmaf(s, part[b][t][i], acc[b][t][i]);
            }
            if (r == 0)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    sums[((wt * TB + wr) * 16 + 4 * g + i) * SUMLD + step % SUMS] = sum[i];
        } else {
            bf16x8 c[RB][4];
#pragma unroll
            for (int b = 0; b < RB; ++b) {
                const unsigned d[4] = {q.w[b].x, q.w[b].y, q.w[b].z, q.w[b].w};
#pragma unroll
                for (int j = 0; j < 4; ++j) c[b][j] = codes8(d[j]);
            }
#pragma unroll
            for (int t = 0; t < TB; ++t) {
                f32x4 part[RB], corr = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int b = 0; b < RB; ++b) part[b] = corr;
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int i = 0; i < T; ++i) {
                        Frag8 f;
                        const int row = wk * ROWS + ((wt * TB + t) * 16 + r) % ROWS;
                        f.u = *(const uint4*)&xs[step & 1][i][row * STRIDE + 64 * g + 16 * j];
                        corr = mfma16(f.v, minus8(), corr);
#pragma unroll
                        for (int b = 0; b < RB; ++b) part[b] = mfma16(f.v, c[b][j], part[b]);
                    }
#pragma unroll
                for (int b = 0; b < RB; ++b) {
                    const float s = scale512(q.s[b]);
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[b][t][i] = __builtin_fmaf(s, part[b][i] + corr[i], acc[b][t][i]);
                }
            }
        }
        store_x(step + 1);
        __syncthreads();
        if constexpr (FOLD) {
            if (step % SUMS == SUMS - 1 || step == a.groups - 1) {
                fold(step - step % SUMS, step % SUMS + 1);
                __syncthreads();
            }
        }
    };
    const int steps = (a.groups + WK - 1) / WK;
    W q[D];
    load_x(0);
#pragma unroll
    for (int d = 0; d + 1 < D; ++d) load_w(q[d], d);
    store_x(0);
    __syncthreads();
    for (int step = 0;;) {
#pragma unroll
        for (int d = 0; d < D; ++d) {
            group(q[d], q[(d + D - 1) % D], step);
            if (++step == steps) break;
        }
        if (step == steps) break;
    }
    // the last step's barrier is behind: xs is free
    if constexpr (WK > 1) {
        f32x4* red = (f32x4*)&xs[0][0][0] + lane;
#pragma unroll
        for (int k = WK / 2; k >= 1; k /= 2) {
            const int at = (wr + WO * (wt + WT * (wk % k))) * RB * TB * 64;
            if (wk >= k && wk < 2 * k)
#pragma unroll
                for (int i = 0; i < RB * TB; ++i) red[at + 64 * i] = acc[i / TB][i % TB];
            __syncthreads();
            if (wk < k)
#pragma unroll
                for (int i = 0; i < RB * TB; ++i) {
                    const f32x4 v = red[at + 64 * i];
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[i / TB][i % TB][e] = acc[i / TB][i % TB][e] + v[e];
                }
            __syncthreads();
        }
        if (wk > 0) return;
    }
#pragma unroll
    for (int b = 0; b < RB; ++b) {
        const int o = (b0 + b) * 16 + r;
#pragma unroll
        for (int t = 0; t < TB; ++t) {
            const int n = n0 + (wt * TB + t) * 16 + 4 * g;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (o < a.O && n + i < a.N) put<F32>(a, n + i, o, acc[b][t][i]);
        }
    }
}

constexpr int kLds = 163840;
constexpr long long kAny = 1ll << 62;

// Whether the rows fit into LDS beside the sums of RB outputs, and the launch if they do. Two work-groups per
// CU if both fit: more of them (768, 1024 in all) cost 1 x 4096 x 100003 a fifth.
template <bool F32, int RB, int D, bool TINY>
bool few_launch(const LinArgs& a, int least, hipStream_t st) {
    if (a.blocks < least || a.groups > kLds / (kGroup * 2)) return false;
    const FewLds l = few_lds(a.N, a.groups, X8<F32>::TERMS, RB);
    if (l.bytes > kLds) return false;
    const int grid = std::min(ceil_div(a.blocks, RB), l.bytes <= kLds / 2 ? 512 : 256);
    int4_few_kernel<F32, RB, D, TINY><<<grid, 512, l.bytes, st>>>(a);
    return true;
}
// More outputs at a time make fewer reads of x from LDS, fewer keep more CUs at work: 1 x 4096 x 16384 takes
// 9.9 us with two blocks and 11.2 with three, 16 x 1024 x 65536 13.4 with four and 14.0 with three. Where
// four do not fit beside the rows (16 x 4096) two do.
template <bool F32>
bool few_launch(const LinArgs& a, hipStream_t st) {
    if ((long long)a.N * a.K < 8) return few_launch<F32, 2, 3, true>(a, 0, st);
    return few_launch<F32, 4, 2, false>(a, 1536, st) || few_launch<F32, 2, 3, false>(a, 512, st) ||
           few_launch<F32, 1, 3, false>(a, 0, st);
}

// int4_rows_kernel, and whether it is launched: if that takes from least to most work-groups.
template <bool F32, int TB, int RB, int WO, int WT, int D, int ROWS = 16 * TB * WT>
bool rows_launch(const LinArgs& a, long long least, long long most, hipStream_t st) {
    const long long wgs = (long long)ceil_div(a.N, ROWS) * ceil_div(a.blocks, WO * RB);
    if (wgs < least || wgs > most) return false;
    int4_rows_kernel<F32, TB, RB, WO, WT, D, ROWS><<<(unsigned)wgs, 512, 0, st>>>(a);
    return true;
}
template <bool F32, int TB, int WO>
void rows_launch(const LinArgs& a, hipStream_t st) {
    if (!rows_launch<F32, TB, 2, WO, 1, 3>(a, 512, kAny, st)) rows_launch<F32, TB, 1, WO, 1, 3>(a, 0, kAny, st);
}

// The more wavefronts deal out K, the fewer steps there are and the smaller the work-groups' outputs; LDS has
// room for eight groups of 8 rows in fp32 (7 x 5000 x 3001: 10.3 us, 15.0 with four groups of 16 rows) and of
// 16 or 32 rows in bf16 (16 x 14336 x 4096: 14.8 us with eight, 19.0 with four; 32 x 14336 x 4096: 20.4 and
// 26.5, but 32 x 5120 x 8192, with outputs for all CUs, 18.9 and 13.2). With more rows, the smallest tiles that
// all run at once: bf16 100 x 2048 x 1024 7.2 us in 32 rows x 32 outputs, 10.2 in 64 x 32, 14.6 in 128 x 32
// (4096 x 4096, 200 rows: 27, 30, 26); fp32 64 x 14336 x 1024 33 us in 16 x 32, 105 in 32 x 64, 171 in 64 x 64,
// 100 x 5120 x 8192 90, 67, 69 and 47 in 32 x 128. Then the largest that give every CU one.
template <bool F32>
void launch(const LinArgs& a, hipStream_t st) {
    const int N = a.N;
    if (N <= 16 && few_launch<F32>(a, st)) return;
    if (N <= 8) {
        if (!rows_launch<F32, 1, 2, 1, 1, 3, 8>(a, 256, kAny, st)) rows_launch<F32, 1, 1, 1, 1, 3, 8>(a, 0, kAny, st);
    } else if constexpr (F32) {
        if (N <= 16) rows_launch<F32, 1, 2>(a, st);
        else if (N <= 32) rows_launch<F32, 2, 4>(a, st);
        else if (!rows_launch<F32, 1, 1, 2, 1, 3>(a, 0, 512, st) && !rows_launch<F32, 2, 1, 4, 1, 3>(a, 0, 256, st) &&
                 !rows_launch<F32, 2, 2, 4, 1, 3>(a, 0, 256, st) &&
                 !rows_launch<F32, 2, 4, 4, 2, 2>(a, 256, kAny, st) &&
                 !rows_launch<F32, 2, 2, 4, 2, 2>(a, 256, kAny, st))
            rows_launch<F32, 2, 1, 4, 2, 2>(a, 0, kAny, st);
    } else {
        if (N <= 16) rows_launch<F32, 1, 1>(a, st);
        else if (N <= 32 && a.blocks <= 256) rows_launch<F32, 2, 1, 1, 1, 3>(a, 0, kAny, st);
        else if (N <= 32) rows_launch<F32, 2, 2>(a, st);
        else if (rows_launch<F32, 2, 1, 2, 1, 3>(a, 0, 256, st)) return;
        else if (N <= 48) rows_launch<F32, 3, 2>(a, st);
        else if (N <= 64) rows_launch<F32, 4, 2>(a, st);
        else if (!rows_launch<F32, 4, 1, 2, 1, 3>(a, 0, 256, st) &&
                 !rows_launch<F32, 4, 4, 4, 2, 2>(a, 256, kAny, st) &&
                 !rows_launch<F32, 4, 2, 4, 2, 2>(a, 256, kAny, st) &&
                 !rows_launch<F32, 4, 1, 4, 2, 2>(a, 256, kAny, st))
            rows_launch<F32, 4, 1, 2, 2, 2>(a, 0, kAny, st);
    }
}

}  // namespace

int int4_linear_launch(const void* x, int act, int N, const yvmoe_int4_matrix* w, const void* bias, void* out,
                       hipStream_t st) {
    LinArgs a{};
    a.x = x;
    a.N = N, a.K = w->in_features, a.O = w->out_features;
    a.groups = ceil_div(a.K, kGroup);
    a.blocks = ceil_div(a.O, 16);
    a.codes = (const char*)w->codes;
    a.scales = (const unsigned short*)w->scales;
    a.bias = bias, a.out = out;
    if (act == YVMOE_ACT_F32) launch<true>(a, st);
    else launch<false>(a, st);
    YV_LAUNCH_CHECK("int4_linear");
    return YVMOE_OK;
}

}  // namespace yvmoe
