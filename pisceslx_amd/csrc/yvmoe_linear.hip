// Linear layer with 4-bit weights and a scale per 128 columns of a row, for gfx950.
//
//   y[n][o] = Σ_i x[n][i] (q[o][i] - 8) s[o][i / 128] + b[o]
//
// (model/utils/quantization.py:486-496 with the codes of opss/quantize/engine.py:889-941). A few rows
// are bound by the stream of codes, half a byte each: out·in / 2 bytes.
//
// Products. v_mfma_f32_16x16x32_bf16 with 16 weight rows as first and 16 rows of x as second operand:
// lane l = 16 g + r holds 8 columns of weight row r and of x row r, the accumulator 4 weight rows of x
// row r. A nibble q at bits 3-6 of 0x4180 is the bf16 number 16 + q, so two codes cost a shift and an
// and-or and no conversion; Σ x (16 + q) over a group, plus -24 Σ x from MFMAs with a constant
// operand, is Σ x (q - 8), all exact products in fp32 sums. The group's scale multiplies that sum, so
// nothing is rounded before y. fp32 rows of x go in as three bf16 terms, which hold all 24 bits.
//
// Storage (include/yvmoe.h): per 16 rows and 128 columns 1 KB, lane l's 16 bytes at 16 l, columns
// 32 g .. 32 g + 31 of row r; in a dword columns 0, 2, 4, 6 are the lower and 1, 3, 5, 7 the upper
// four nibbles, which gives an operand's pairs in order.
#include "yvmoe_frag.h"
#include "yvmoe_internal.h"

namespace yvmoe {
namespace {

constexpr int kGroup = 128;

struct LinArgs {
    const void* x;
    int N, K, O, groups;
    const char* codes;             // [O / 16][groups][1 KB]
    const unsigned short* scales;  // [O / 16][groups][16]
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
    unsigned short h[8];
};

// The eight weights of a dword as 16 + q.
__device__ __forceinline__ bf16x8 codes8(unsigned w) {
    Frag8 f;
    f.u = make_uint4(((w << 3) & 0x00780078u) | 0x41804180u, ((w >> 1) & 0x00780078u) | 0x41804180u,
                     ((w >> 5) & 0x00780078u) | 0x41804180u, ((w >> 9) & 0x00780078u) | 0x41804180u);
    return f.v;
}
__device__ __forceinline__ bf16x8 minus24() {
    Frag8 f;
    f.u = make_uint4(0xC1C0C1C0u, 0xC1C0C1C0u, 0xC1C0C1C0u, 0xC1C0C1C0u);
    return f.v;
}
__device__ __forceinline__ f32x4 mfma16(const bf16x8& a, const bf16x8& b, const f32x4& c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// 32 columns of a row of x from column c, zero past the row's end.
template <bool F32>
struct XCols;
template <>
struct XCols<false> {
    static constexpr int TERMS = 1;
    uint4 v[4];
    __device__ __forceinline__ void load(const void* row, int c, int K) {
        const unsigned short* p = (const unsigned short*)row + c;
        if (c + 32 <= K) {
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = load_any16(p + 8 * j);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                unsigned d[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int at = 8 * j + 2 * i;
                    d[i] = (c + at < K ? p[at] : 0) | (unsigned)(c + at + 1 < K ? p[at + 1] : 0) << 16;
                }
                v[j] = make_uint4(d[0], d[1], d[2], d[3]);
            }
        }
    }
    __device__ __forceinline__ void terms(int j, bf16x8 (&t)[1]) const {
        Frag8 f;
        f.u = v[j];
        t[0] = f.v;
    }
};
template <>
struct XCols<true> {
    static constexpr int TERMS = 3;
    uint4 v[8];
    __device__ __forceinline__ void load(const void* row, int c, int K) {
        const unsigned* p = (const unsigned*)row + c;
        if (c + 32 <= K) {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = load_any16(p + 4 * j);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                unsigned d[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) d[i] = c + 4 * j + i < K ? p[4 * j + i] : 0u;
                v[j] = make_uint4(d[0], d[1], d[2], d[3]);
            }
        }
    }
    // Three bf16 terms, each the rest's rounding: their sum has 24 bits, as x has.
    __device__ __forceinline__ void terms(int j, bf16x8 (&t)[3]) const {
        const unsigned w[8] = {v[2 * j].x, v[2 * j].y, v[2 * j].z, v[2 * j].w,
                               v[2 * j + 1].x, v[2 * j + 1].y, v[2 * j + 1].z, v[2 * j + 1].w};
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

// 16 outputs and 16 rows of x per work-group; the wavefronts deal out the groups.
template <bool F32>
__global__ __launch_bounds__(512) void int4_few_kernel(LinArgs a) {
    constexpr int T = XCols<F32>::TERMS;
    __shared__ f32x4 red[8][64];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = lane >> 4, r = lane & 15;
    const int n0 = blockIdx.y * 16, o0 = blockIdx.x * 16;
    const char* xrow = (const char*)a.x + (long long)min(n0 + r, a.N - 1) * a.K * (F32 ? 4 : 2);
    const char* codes = a.codes + (long long)blockIdx.x * a.groups * 1024 + lane * 16;
    const unsigned short* scales = a.scales + (long long)blockIdx.x * a.groups * 16 + 4 * g;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    for (int kg = wave; kg < a.groups; kg += 8) {
        const uint4 w = nt_load16(codes + (long long)kg * 1024);
        const ushort4 s = *(const ushort4*)(scales + (long long)kg * 16);
        XCols<F32> x;
        x.load(xrow, kg * kGroup + 32 * g, a.K);
        const unsigned d[4] = {w.x, w.y, w.z, w.w};
        f32x4 part = {0.f, 0.f, 0.f, 0.f}, corr = part;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            bf16x8 t[T];
            x.terms(j, t);
            const bf16x8 q = codes8(d[j]);
#pragma unroll
            for (int i = 0; i < T; ++i) {
                corr = mfma16(minus24(), t[i], corr);
                part = mfma16(q, t[i], part);
            }
        }
        acc[0] = __builtin_fmaf(bf16_to_f32(s.x), part[0] + corr[0], acc[0]);
        acc[1] = __builtin_fmaf(bf16_to_f32(s.y), part[1] + corr[1], acc[1]);
        acc[2] = __builtin_fmaf(bf16_to_f32(s.z), part[2] + corr[2], acc[2]);
        acc[3] = __builtin_fmaf(bf16_to_f32(s.w), part[3] + corr[3], acc[3]);
    }
    red[wave][lane] = acc;
    __syncthreads();
    if (wave != 0 || n0 + r >= a.N) return;
    f32x4 sum = red[0][lane];
#pragma unroll
    for (int w = 1; w < 8; ++w) {
        const f32x4 v = red[w][lane];
#pragma unroll
        for (int i = 0; i < 4; ++i) sum[i] = sum[i] + v[i];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int o = o0 + 4 * g + i;
        if (o >= a.O) break;
        const long long at = (long long)(n0 + r) * a.O + o;
        float v = sum[i];
        if constexpr (F32) {
            if (a.bias != nullptr) v = v + ((const float*)a.bias)[o];
            ((float*)a.out)[at] = v;
        } else {
            if (a.bias != nullptr) v = v + bf16_to_f32(((const unsigned short*)a.bias)[o]);
            ((unsigned short*)a.out)[at] = f32_to_bf16_rne(v);
        }
    }
}

}  // namespace

int int4_linear_launch(const void* x, int act, int N, const yvmoe_int4_matrix* w, const void* bias, void* out,
                       hipStream_t st) {
    LinArgs a{};
    a.x = x;
    a.N = N, a.K = w->in_features, a.O = w->out_features;
    a.groups = ceil_div(a.K, kGroup);
    a.codes = (const char*)w->codes;
    a.scales = (const unsigned short*)w->scales;
    a.bias = bias, a.out = out;
    const dim3 grid(ceil_div(a.O, 16), ceil_div(N, 16));
    if (act == YVMOE_ACT_F32) int4_few_kernel<true><<<grid, 512, 0, st>>>(a);
    else int4_few_kernel<false><<<grid, 512, 0, st>>>(a);
    YV_LAUNCH_CHECK("int4_linear");
    return YVMOE_OK;
}

}  // namespace yvmoe
