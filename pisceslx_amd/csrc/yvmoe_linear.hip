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
// Forms. Up to 64 rows of x: int4_few_kernel, bound by the stream of codes (out·in / 2 bytes) and at small
// sizes by one trip to memory. More: int4_rows_kernel, bound by the MFMAs.
#include "yvmoe_frag.h"
#include "yvmoe_internal.h"

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

// Eight columns of a row of x from column c, zero past the row's end.
template <bool F32>
struct X8;
template <>
struct X8<false> {
    static constexpr int TERMS = 1;
    uint4 v;
    __device__ __forceinline__ void load(const void* row, int c, int K) {
        const unsigned short* p = (const unsigned short*)row + c;
        if (c + 8 <= K) {
            v = load_any16(p);
        } else {
            unsigned d[4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
                d[i] = (c + 2 * i < K ? p[2 * i] : 0) | (unsigned)(c + 2 * i + 1 < K ? p[2 * i + 1] : 0) << 16;
            v = make_uint4(d[0], d[1], d[2], d[3]);
        }
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
    __device__ __forceinline__ void load(const void* row, int c, int K) {
        const unsigned* p = (const unsigned*)row + c;
        if (c + 8 <= K) {
            v[0] = load_any16(p);
            v[1] = load_any16(p + 4);
        } else {
            unsigned d[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) d[i] = c + i < K ? p[i] : 0u;
            v[0] = make_uint4(d[0], d[1], d[2], d[3]);
            v[1] = make_uint4(d[4], d[5], d[6], d[7]);
        }
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

// ---------------------------------------------------------------- up to 64 rows
// A work-group computes 16 RB outputs of 16 TB rows; its eight wavefronts deal out the groups of K, each
// with the next group's codes and the next half group's rows in flight, and add up in LDS at the end.
template <bool F32, int TB, int RB>
__global__ __launch_bounds__(512, 2) void int4_few_kernel(LinArgs a) {
    constexpr int T = X8<F32>::TERMS;
    __shared__ f32x4 red[8][RB * TB][64];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = lane >> 4, r = lane & 15;
    const int n0 = blockIdx.y * 16 * TB, b0 = blockIdx.x * RB;
    const char* xrow[TB];
#pragma unroll
    for (int t = 0; t < TB; ++t)
        xrow[t] = (const char*)a.x + (long long)min(n0 + 16 * t + r, a.N - 1) * a.K * (F32 ? 4 : 2);
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
    struct X {
        X8<F32> x[2][TB];
    };
    auto load_w = [&](W& q, int kg) {  // groups past the end: the last one again, not used
        kg = min(kg, a.groups - 1);
#pragma unroll
        for (int b = 0; b < RB; ++b) {
            q.w[b] = nt_load16(codes[b] + (long long)kg * 1024);
            q.s[b] = scales[b][(long long)kg * 16];
        }
    };
    auto load_x = [&](X& x, int kg, int half) {
        kg = min(kg, a.groups - 1);
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int t = 0; t < TB; ++t) x.x[j][t].load(xrow[t], kg * kGroup + 32 * g + 16 * half + 8 * j, a.K);
    };
    f32x4 acc[RB][TB];
#pragma unroll
    for (int b = 0; b < RB; ++b)
#pragma unroll
        for (int t = 0; t < TB; ++t) acc[b][t] = f32x4{0.f, 0.f, 0.f, 0.f};
    auto group = [&](W& q, W& qn, X& x0, X& x1, int kg) {
        f32x4 part[RB][TB], corr[TB];
#pragma unroll
        for (int t = 0; t < TB; ++t) {
            corr[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int b = 0; b < RB; ++b) part[b][t] = corr[t];
        }
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            X& x = half ? x1 : x0;
            if (half) {
                load_w(qn, kg + 8);
                load_x(x0, kg + 8, 0);
            } else {
                load_x(x1, kg, 1);
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                bf16x8 c[RB];
#pragma unroll
                for (int b = 0; b < RB; ++b) {
                    const unsigned d[4] = {q.w[b].x, q.w[b].y, q.w[b].z, q.w[b].w};
                    c[b] = codes8(d[2 * half + j]);
                }
#pragma unroll
                for (int t = 0; t < TB; ++t) {
                    bf16x8 v[T];
                    x.x[j][t].terms(v);
#pragma unroll
                    for (int i = 0; i < T; ++i) {
                        corr[t] = mfma16(v[i], minus8(), corr[t]);
#pragma unroll
                        for (int b = 0; b < RB; ++b) part[b][t] = mfma16(v[i], c[b], part[b][t]);
                    }
                }
            }
        }
#pragma unroll
        for (int b = 0; b < RB; ++b) {
            const float s = scale512(q.s[b]);
#pragma unroll
            for (int t = 0; t < TB; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[b][t][i] = __builtin_fmaf(s, part[b][t][i] + corr[t][i], acc[b][t][i]);
        }
    };
    if (wave < a.groups) {
        W q0, q1;
        X x0, x1;
        load_w(q0, wave);
        load_x(x0, wave, 0);
        int kg = wave;
        for (; kg + 8 < a.groups; kg += 16) {
            group(q0, q1, x0, x1, kg);
            group(q1, q0, x0, x1, kg + 8);
        }
        if (kg < a.groups) group(q0, q1, x0, x1, kg);
    }
#pragma unroll
    for (int b = 0; b < RB; ++b)
#pragma unroll
        for (int t = 0; t < TB; ++t) red[wave][b * TB + t][lane] = acc[b][t];
    __syncthreads();
    for (int i = wave; i < RB * TB; i += 8) {
        f32x4 sum = red[0][i][lane];
#pragma unroll
        for (int w = 1; w < 8; ++w) {
            const f32x4 v = red[w][i][lane];
#pragma unroll
            for (int e = 0; e < 4; ++e) sum[e] = sum[e] + v[e];
        }
        const int o = (b0 + i / TB) * 16 + r, n = n0 + i % TB * 16 + 4 * g;
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (o < a.O && n + e < a.N) put<F32>(a, n + e, o, sum[e]);
    }
}

// ---------------------------------------------------------------- more rows
// A work-group of 4 x 2 wavefronts computes 64 RB outputs of 32 TB rows; a wavefront 16 RB outputs of
// 16 TB rows. Each group's 128 columns of the rows go through LDS (as bf16 terms, two stages, rows padded by
// 16 bytes, so that the 16 rows of an operand fall on different banks), loaded a group ahead; the codes
// go straight to the wavefront that converts them, each once for its TB MFMAs of every term.
template <bool F32, int TB, int RB>
__global__ __launch_bounds__(512, 2) void int4_rows_kernel(LinArgs a) {
    constexpr int T = X8<F32>::TERMS, ROWS = 32 * TB, STRIDE = kGroup * 2 + 16;
    constexpr int PER = ROWS * 16 / 512;  // pieces of 8 columns that a thread brings
    __shared__ __align__(16) char xs[2][T][ROWS * STRIDE];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int g = lane >> 4, r = lane & 15;
    const int wr = wave & 3, wt = wave >> 2;
    // blocks of rows fastest: work-groups that run together share their codes
    const int nrt = (a.N + ROWS - 1) / ROWS;
    const int n0 = (int)(blockIdx.x % nrt) * ROWS, b0 = ((int)(blockIdx.x / nrt) * 4 + wr) * RB;
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
    auto load_w = [&](W& q, int kg) {
        kg = min(kg, a.groups - 1);
#pragma unroll
        for (int b = 0; b < RB; ++b) {
            q.w[b] = *(const uint4*)(codes[b] + (long long)kg * 1024);
            q.s[b] = scales[b][(long long)kg * 16];
        }
    };
    X8<F32> px[PER];
    auto load_x = [&](int kg) {
        kg = min(kg, a.groups - 1);
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int piece = tid + 512 * i, row = piece / 16, c = piece % 16;
            px[i].load((const char*)a.x + (long long)min(n0 + row, a.N - 1) * a.K * (F32 ? 4 : 2), kg * kGroup + 8 * c, a.K);
        }
    };
    auto store_x = [&](int stage) {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int piece = tid + 512 * i, row = piece / 16, c = piece % 16;
            bf16x8 t[T];
            px[i].terms(t);
#pragma unroll
            for (int q = 0; q < T; ++q) {
                Frag8 f;
                f.v = t[q];
                *(uint4*)&xs[stage][q][row * STRIDE + 16 * c] = f.u;
            }
        }
    };
    f32x4 acc[RB][TB];
#pragma unroll
    for (int b = 0; b < RB; ++b)
#pragma unroll
        for (int t = 0; t < TB; ++t) acc[b][t] = f32x4{0.f, 0.f, 0.f, 0.f};
    auto group = [&](const W& q, W& qn, int kg) {
        load_x(kg + 1);
        load_w(qn, kg + 1);
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
                    f.u = *(const uint4*)&xs[kg & 1][i][((wt * TB + t) * 16 + r) * STRIDE + 64 * g + 16 * j];
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
        store_x((kg + 1) & 1);
        __syncthreads();
    };
    W q0, q1;
    load_x(0);
    load_w(q0, 0);
    store_x(0);
    __syncthreads();
    int kg = 0;
    for (; kg + 1 < a.groups; kg += 2) {
        group(q0, q1, kg);
        group(q1, q0, kg + 1);
    }
    if (kg < a.groups) group(q0, q1, kg);
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

template <bool F32, int TB>
void few_launch_rb(const LinArgs& a, hipStream_t st) {
    // 16, 32 or 64 outputs per work-group: as many as leave four work-groups per CU
    const int y = ceil_div(a.N, 16 * TB);
    const long long wgs = (long long)a.blocks * y;
    constexpr int MOST = F32 || TB > 2 ? 2 : 4;
    if (MOST >= 4 && wgs >= 4096) int4_few_kernel<F32, TB, MOST><<<dim3(ceil_div(a.blocks, MOST), y), 512, 0, st>>>(a);
    else if (wgs >= 1024) int4_few_kernel<F32, TB, 2><<<dim3(ceil_div(a.blocks, 2), y), 512, 0, st>>>(a);
    else int4_few_kernel<F32, TB, 1><<<dim3(a.blocks, y), 512, 0, st>>>(a);
}

template <bool F32>
void rows_launch(const LinArgs& a, hipStream_t st) {
    constexpr int TB = F32 ? 2 : 4;
    const int nrt = ceil_div(a.N, 32 * TB);
    if ((long long)nrt * ceil_div(a.blocks, 16) >= 256)
        int4_rows_kernel<F32, TB, 4><<<nrt * ceil_div(a.blocks, 16), 512, 0, st>>>(a);
    else if ((long long)nrt * ceil_div(a.blocks, 8) >= 128)
        int4_rows_kernel<F32, TB, 2><<<nrt * ceil_div(a.blocks, 8), 512, 0, st>>>(a);
    else int4_rows_kernel<F32, TB, 1><<<nrt * ceil_div(a.blocks, 4), 512, 0, st>>>(a);
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
    if (act == YVMOE_ACT_F32) {
        if (N <= 16) few_launch_rb<true, 1>(a, st);
        else if (N <= 32) few_launch_rb<true, 2>(a, st);
        else rows_launch<true>(a, st);
    } else {
        if (N <= 16) few_launch_rb<false, 1>(a, st);
        else if (N <= 32) few_launch_rb<false, 2>(a, st);
        else if (N <= 48) few_launch_rb<false, 3>(a, st);
        else if (N <= 64) few_launch_rb<false, 4>(a, st);
        else rows_launch<false>(a, st);
    }
    YV_LAUNCH_CHECK("int4_linear");
    return YVMOE_OK;
}

}  // namespace yvmoe
