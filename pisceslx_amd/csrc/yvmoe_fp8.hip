// 8-bit floating point products with a scale per 128 values, for gfx950:
//
//   rows     s[b][n] = max(max |x[n][k in b]| / 448, 1e-12), q[n][k] = e4m3(x[n][k] / s[b][n])
//   linear   y[n][o] = Σ_b s[b][n] w[o / 128][b] Σ_{k in b} q[n][k] c[o][k] + bias[o]
//   block    g, u = linear(x; gate), linear(x; up), h = silu(g) u, y = linear(h; down)
//
// (the format of opss/quantize/engine.py:841-883 with a scale per 128 x 128 weights and per 128 values of a row).
//
// Products. v_mfma_f32_16x16x128_f8f6f4 on a block of 128 contraction elements from a sum of zero, then the block's
// two scales times that sum onto the fp32 result: 4 multiply-adds a lane beside 32 cycles of the matrix unit. 16
// weight rows are the first operand, so a lane holds four consecutive outputs of one row, and the row's scale is one
// number a lane. The unit's sum of 128 products keeps about 16 bits: against 64 bits its results are off by 1.4e-5
// relative (normal values; the same for v_mfma_f32_16x16x32_fp8_fp8, four of them in a row), a hundredth of a bf16
// output's own rounding, which is why outputs are bf16 only.
// Where h is rounded to 8 bits, a code whose border lies within that error of h falls on the other side: about one in a
// thousand, by a step of up to 2^-3. Over many h they add 0.0014 relative to y's own 0.0017; over few a single one can
// be 0.006 of y. So g and u of few rows, and of up to kExactH h, are products of the codes as bf16, on the bf16 unit at
// half the rate, with fp32's error (111 rows x 768 x 32: y 0.0067 off 64 bits on the 8-bit unit, 0.0017 so).
//
// Weights lie in blocks of 16 rows x 64 columns, 1 KB, lane l = 16 g + r's 16 bytes at 16 l: row r, columns
// 16 g .. 16 g + 15 (the order of the experts' matrices); two consecutive blocks are an operand of 128, in which
// lane group g holds elements 16 g .. + 15 and 64 + 16 g .. + 15.
#include <algorithm>

#include "yvmoe_frag.h"
#include "yvmoe_internal.h"

namespace yvmoe {
namespace {

typedef __attribute__((address_space(3))) void* lds_ptr_t;
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));

constexpr int kBlock = 128;
constexpr float kMax = 448.0f, kMinScale = 1e-12f;
constexpr long long kExactH = 1 << 18;

union Op8 {  // an operand of 128 elements: two pieces of 16 bytes
    uint4 u[2];
    i32x8 v;
};
__device__ __forceinline__ f32x4 mfma8(const Op8& a, const Op8& b) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a.v, b.v, f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0, 0, 0, 0);
}
// The same codes as bf16, which holds them exactly, in four operands of v_mfma_f32_16x16x32_bf16, whose sums are fp32's.
struct OpB {
    bf16x8 v[4];
};
__device__ __forceinline__ OpB to_bf16(const Op8& a) {
    OpB r;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        union { unsigned u[4]; bf16x8 v; } f;
#pragma unroll
        for (int d = 0; d < 2; ++d) {
            const int w = a.v[2 * q + d];
            f.u[2 * d] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, false));
            f.u[2 * d + 1] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, true));
        }
        r.v[q] = f.v;
    }
    return r;
}
__device__ __forceinline__ f32x4 mfma8(const OpB& a, const OpB& b) {
    f32x4 c = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int q = 0; q < 4; ++q) c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.v[q], b.v[q], c, 0, 0, 0);
    return c;
}
template <bool EXACT>
__device__ __forceinline__ auto operand(const Op8& a) {
    if constexpr (EXACT) return to_bf16(a);
    else return a;
}

// The scale of values whose largest size has the bits m. NaN (its bits are above every other's) stays NaN.
__device__ __forceinline__ float scale_of(unsigned m) {
    const float s = __uint_as_float(m) / kMax;
    return s < kMinScale ? kMinScale : s;
}
// Values over one s and their codes. A quotient is the value times 1 / s, and its remainder times 1 / s added: off the exact
// quotient by 2^-22 of an fp32 step before the last rounding, so that it is the rounded quotient, but perhaps where that
// lies as near the middle of two fp32 numbers; next to the middle of two codes, where it would count, no quotient of two fp32
// numbers whose s could do so does (by trying them all: s within 24 steps of a multiple of 1/8 of its power of two).
struct Divisor {
    float s, inverse;
    __device__ __forceinline__ explicit Divisor(float by) : s(by == INFINITY ? 0.0f : by), inverse(1.0f / by) {}
    __device__ __forceinline__ float under(float a) const {
        const float q = a * inverse;
        return copysignf(fmaf(fmaf(-q, s, a), inverse, q), a);  // of -0 too
    }
    // e4m3 codes of four values, lowest first
    __device__ __forceinline__ unsigned codes4(float a, float b, float c, float d) const {
        int w = __builtin_amdgcn_cvt_pk_fp8_f32(under(a), under(b), 0, false);
        return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(under(c), under(d), w, true);
    }
};
__device__ __forceinline__ unsigned size_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// ------------------------------------------------------------------ rows
typedef unsigned Any16 __attribute__((ext_vector_type(4), aligned(2)));  // 16 bytes at any address
// ONCE: nothing reads them again soon.
template <bool ONCE>
__device__ __forceinline__ Any16 any16(const void* p) {
    return ONCE ? __builtin_nontemporal_load((const Any16*)p) : *(const Any16*)p;
}
// Eight values from element `at` of a tensor, those from `left` on zero.
template <bool F32, bool ONCE>
__device__ __forceinline__ void load8(const void* x, size_t at, int left, float (&v)[8]) {
    if (left >= 8) {
        if (F32) {
            const Any16 a = any16<ONCE>((const float*)x + at), b = any16<ONCE>((const float*)x + at + 4);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(a[i]), v[4 + i] = __uint_as_float(b[i]);
        } else {
            const Any16 a = any16<ONCE>((const unsigned short*)x + at);
#pragma unroll
            for (int i = 0; i < 4; ++i)
                v[2 * i] = bf16_to_f32((unsigned short)a[i]), v[2 * i + 1] = bf16_to_f32((unsigned short)(a[i] >> 16));
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            v[i] = i >= left ? 0.0f : F32 ? ((const float*)x)[at + i] : bf16_to_f32(((const unsigned short*)x)[at + i]);
    }
}

// Where h comes from: h itself (parts = 0), or g and u as sums of `parts` fp32 planes each, [parts][2][N][ld].
struct Hidden {
    const float* p;
    int parts, ld;
    long long plane;  // N ld
};
__device__ __forceinline__ void load8(const Hidden& h, size_t at, int left, float (&v)[8]) {
    if (h.parts == 0) return load8<true, false>(h.p, at, left, v);
    // ld is a multiple of 128, so all eight are in the planes; columns behind the last one may never have been written, and
    // what is read there is dropped (left)
    f32x4 s[2][2];
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int q = 0; q < 2; ++q) s[m][q] = *(const f32x4*)(h.p + m * h.plane + at + 4 * q);
    for (int k = 1; k < h.parts; ++k)
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int q = 0; q < 2; ++q) s[m][q] = s[m][q] + *(const f32x4*)(h.p + (2 * k + m) * h.plane + at + 4 * q);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i >= left ? 0.0f : silu_fast(s[0][i / 4][i % 4]) * s[1][i / 4][i % 4];
}

// 16 lanes hold a group of 128, eight values each: its scale, and the lane's codes.
__device__ __forceinline__ float quantize8(const float (&v)[8], uint2& codes) {
    unsigned m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, size_bits(v[i]));
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) m = max(m, (unsigned)__shfl_xor((int)m, o, 16));
    const float s = scale_of(m);
    const Divisor by(s);
    codes = make_uint2(by.codes4(v[0], v[1], v[2], v[3]), by.codes4(v[4], v[5], v[6], v[7]));
    return s;
}

enum Source { kCodes, kBf16, kF32, kHidden };
// Values of row n, group b that the lane holds.
template <int SRC, bool ONCE>
__device__ __forceinline__ void values8(const void* x, const Hidden& h, int n, int K, int b, int lane16, float (&v)[8]) {
    const int k = b * kBlock + lane16 * 8;
    if (SRC == kHidden) load8(h, (size_t)n * h.ld + k, K - k, v);
    else load8<SRC == kF32, ONCE>(x, (size_t)n * K + k, K - k, v);
}

// One pass over the rows, bound by memory: U groups for 16 lanes, all of their loads in flight at once. Many rows are
// read past the caches, which keep the codes and weights of the product behind (8192 x 4096 x 8192 321 -> 308 us).
template <int SRC, int U>
__global__ __launch_bounds__(256) void fp8_rows_kernel(const void* x, Hidden h, int N, int K, int groups,
                                                       unsigned char* codes, float* scales) {
    const long long items = (long long)N * groups;
    const int l = threadIdx.x & 15;
    for (long long first = (long long)blockIdx.x * 16 * U + (threadIdx.x >> 4); first < items;
         first += (long long)gridDim.x * 16 * U) {
        float v[U][8];
        int n[U], b[U];
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const long long it = std::min(first + 16 * i, items - 1);
            n[i] = (int)(it / groups), b[i] = (int)(it - (long long)n[i] * groups);
            values8<SRC, (U > 1)>(x, h, n[i], K, b[i], l, v[i]);
        }
#pragma unroll
        for (int i = 0; i < U; ++i) {
            if (first + 16 * i >= items) break;
            uint2 c;
            const float s = quantize8(v[i], c);
            *(uint2*)(codes + (first + 16 * i) * kBlock + l * 8) = c;
            if (l == 0) scales[(long long)b[i] * N + n[i]] = s;
        }
    }
}

// ------------------------------------------------------------------ products
enum Epi { kLinear, kSwiGLU };

struct Fp8Args {
    const char* codes;    // rows [N][groups * 128]
    const float* scales;  // [groups][N]
    int N, O, groups, blocks;      // outputs (kSwiGLU: columns of h), blocks of 16
    const char* w[2];              // [blocks][groups] of 2 KB; kSwiGLU: gate, up
    const float* ws[2];            // [ceil(O / 128)][groups]
    const unsigned short* bias;    // [O] or NULL
    unsigned short* out;           // [N][O]
    const void* x;                 // few rows: rounded to 8 bits in the kernel, [N][K]
    Hidden hidden;                 // or the rows' source
    int K;
    float* h;                      // kSwiGLU: [N][ldh], ldh = O rounded up to 128; or sums of g and u (Hidden)
    int parts;                     // splits of the contraction
    float* part;                   // kLinear with several: their sums [parts][N][ldp]
    int ldp;
    unsigned char* hq;             // or its codes [N][ldh] and scales [ldh / 128][N]
    float* hs;
    int ldh;
    int ncb, tiles, total;         // column blocks, tiles, tiles x splits
    int len;                       // blocks of 128 contraction elements of a tile's split
};

__device__ __forceinline__ uint4 load16(const char* p) { return *(const uint4*)p; }

// Few rows (16 MR at most): a work-group of eight wavefronts owns 16 outputs (kSwiGLU: gate and up), the wavefronts
// deal out the blocks of 128 contraction elements and add their sums in LDS, in order. Bound by the stream of the
// weights, which go to registers in their stored order, kAhead steps ahead. SRC: the rows' codes come from L2, or the
// work-group makes them in LDS while its first weights are on their way (a launch and a round trip less; each
// work-group repeats the work, so only for few values). 49 to 64 rows of kSwiGLU take all 256 registers and spill eight.
template <int EPI, int MR, int SRC>
__global__ __launch_bounds__(512) void fp8_few_kernel(Fp8Args p) {
    constexpr int NM = EPI == kSwiGLU ? 2 : 1;  // matrices
    constexpr int kAhead = MR == 1 ? 4 : 2;
    extern __shared__ __attribute__((aligned(16))) unsigned char few_lds[];
    f32x4(*part)[NM * MR][64] = (f32x4(*)[NM * MR][64])few_lds;
    unsigned char* lcodes = few_lds + sizeof(f32x4) * 8 * NM * MR * 64;  // [N][pitch]
    const int pitch = p.groups * kBlock + 16;
    float* lscales = (float*)(lcodes + (size_t)p.N * pitch);             // [N][groups]
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int blk = blockIdx.x % p.blocks, split = blockIdx.x / p.blocks, stride = 8 * p.parts;
    const int row = lane & 15;
    struct Step {
        Op8 w[NM], a[MR];
        float s[MR], ws[NM];
    } buf[kAhead];
    // step t of the wavefront: block first + t stride
    const int first = split * 8 + wave;
    const int steps = first < p.groups ? (p.groups - first + stride - 1) / stride : 0;
    auto load = [&](Step& q, int t) {
        const int b = first + t * stride;
#pragma unroll
        for (int m = 0; m < NM; ++m) {
            const char* at = p.w[m] + ((long long)blk * p.groups + b) * 2048 + lane * 16;
            q.w[m].u[0] = nt_load16(at);
            q.w[m].u[1] = nt_load16(at + 1024);
            q.ws[m] = p.ws[m][(long long)(blk >> 3) * p.groups + b];
        }
        if constexpr (SRC == kCodes) {
#pragma unroll
            for (int r = 0; r < MR; ++r) {
                // rows past the last one read it again; their sums are not stored
                const int n = min(16 * r + row, p.N - 1);
                const char* at = p.codes + ((long long)n * p.groups + b) * kBlock + (lane >> 4) * 16;
                q.a[r].u[0] = load16(at);
                q.a[r].u[1] = load16(at + 64);
                q.s[r] = p.scales[(long long)b * p.N + n];
            }
        }
    };
    f32x4 acc[NM][MR];
#pragma unroll
    for (int m = 0; m < NM; ++m)
#pragma unroll
        for (int r = 0; r < MR; ++r) acc[m][r] = f32x4{0.f, 0.f, 0.f, 0.f};
    constexpr bool EXACT = EPI == kSwiGLU;
    auto add = [&](Step& q, int t) {
        if constexpr (SRC != kCodes) {
            const int b = first + t * stride, n = min(row, p.N - 1);
            const unsigned char* at = lcodes + n * pitch + b * kBlock + (lane >> 4) * 16;
            q.a[0].u[0] = *(const uint4*)at;
            q.a[0].u[1] = *(const uint4*)(at + 64);
            q.s[0] = lscales[n * p.groups + b];
        }
#pragma unroll
        for (int m = 0; m < NM; ++m)
#pragma unroll
            for (int r = 0; r < MR; ++r) {
                const f32x4 d = mfma8(operand<EXACT>(q.w[m]), operand<EXACT>(q.a[r]));
                const float f = q.s[r] * q.ws[m];
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[m][r][i] = fmaf(d[i], f, acc[m][r][i]);
            }
    };
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
        if (i < steps) load(buf[i], i);
    if constexpr (SRC != kCodes) {
        const int l = threadIdx.x & 15;
        for (int it = threadIdx.x >> 4; it < p.N * p.groups; it += 32) {
            const int n = it / p.groups, b = it - n * p.groups;
            float v[8];
            values8<SRC, false>(p.x, p.hidden, n, p.K, b, l, v);
            uint2 c;
            const float s = quantize8(v, c);
            *(uint2*)(lcodes + n * pitch + b * kBlock + l * 8) = c;
            if (l == 0) lscales[it] = s;
        }
        __syncthreads();
    }
    int t = 0;
    for (; t + 2 * kAhead <= steps; t += kAhead)
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            add(buf[i], t + i);
            load(buf[i], t + kAhead + i);
        }
    for (; t < steps; t += kAhead)
#pragma unroll
        for (int i = 0; i < kAhead; ++i)
            if (t + i < steps) {
                add(buf[i], t + i);
                if (t + kAhead + i < steps) load(buf[i], t + kAhead + i);
            }
#pragma unroll
    for (int m = 0; m < NM; ++m)
#pragma unroll
        for (int r = 0; r < MR; ++r) part[wave][m * MR + r][lane] = acc[m][r];
    __syncthreads();
    // wavefront r finishes rows 16 r .. + 15
    if (wave >= MR) return;
    f32x4 v[NM];
#pragma unroll
    for (int m = 0; m < NM; ++m) {
        v[m] = part[0][m * MR + wave][lane];
#pragma unroll
        for (int k = 1; k < 8; ++k) v[m] = v[m] + part[k][m * MR + wave][lane];
    }
    const int n = 16 * wave + row, o = blk * 16 + 4 * (lane >> 4);
    if (n >= p.N) return;
    if constexpr (EPI == kSwiGLU) {
        const long long at = (long long)n * p.ldh + o, plane = (long long)p.N * p.ldh;
        if (p.parts == 1) {
            f32x4 h;
#pragma unroll
            for (int i = 0; i < 4; ++i) h[i] = silu_fast(v[0][i]) * v[NM - 1][i];
            *(f32x4*)(p.h + at) = h;
        } else {
            *(f32x4*)(p.h + 2 * split * plane + at) = v[0];
            *(f32x4*)(p.h + (2 * split + 1) * plane + at) = v[NM - 1];
        }
    } else if (p.parts > 1) {
        *(f32x4*)(p.part + ((long long)split * p.N + n) * p.ldp + o) = v[0];
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (o + i < p.O) {
                const float b = p.bias != nullptr ? bf16_to_f32(p.bias[o + i]) : 0.0f;
                p.out[(long long)n * p.O + o + i] = f32_to_bf16_rne(v[0][i] + b);
            }
    }
}

// s_waitcnt immediate (gfx9 encoding): vmcnt and lgkmcnt 0, loads from memory and reads of LDS
constexpr int all_done() { return 0x7 << 4; }

// Direct loads to LDS at m0 + 16 (4) x lane, from base + off; an offset of kNone reads zeros (the buffer's bounds are
// 2^31 bytes, which no other offset reaches, and no lane reads behind a tensor).
constexpr unsigned kNone = 0xfffffff0u;
__device__ __forceinline__ i32x4 rsrc_of(const void* base) {
    const unsigned long long p = (unsigned long long)base;
    return i32x4{(int)(unsigned)p, (int)(unsigned)(p >> 32) & 0xffff, (int)0x80000000u, 0x00020000};
}
__device__ __forceinline__ void load_lds16(const void* base, unsigned off, unsigned m0) {
    asm volatile("buffer_load_dwordx4 %0, %1, 0 offen lds" : : "v"(off), "s"(rsrc_of(base)), "{m0}"(m0) : "memory");
}
__device__ __forceinline__ void load_lds4(const void* base, unsigned off, unsigned m0) {
    asm volatile("buffer_load_dword %0, %1, 0 offen lds" : : "v"(off), "s"(rsrc_of(base)), "{m0}"(m0) : "memory");
}

constexpr int kBand = 8;

// 16-byte piece c of a 128-byte row r lies at c ^ swizzle(r): the 16 lanes that read together, of two neighbouring lane
// groups g and 16 rows, then lie in different banks.
__device__ __forceinline__ int swizzle(int r) { return (r >> 1 & 3) | ((r ^ r >> 3) & 1) << 2; }

// Tiles: WR x WC wavefronts of 16 MB rows x 16 NB columns each (kSwiGLU: the wavefront's first NB / 2 blocks are gate
// columns, the others the up columns of the same h columns). A step is a block of 128 contraction elements: rows
// (swizzled 128-byte lines), weights (stored order) and both scales go to LDS by direct loads, one step ahead of the
// products, in two stages with one barrier a step. 256 x 256 tiles: 8192 x 4096 x 8192 in 257 us (264 on another card;
// medians of a long run), 2.1 PFLOP/s, the matrix unit busy half of the time. In copies with a part left out: without the
// outputs' stores 243, without scales 250, without the loads past a tile's first step 200. In 64 x 128 tiles, several
// work-groups a CU, 340. Wavefronts 8 x 1, 4 x 4 or 8 x 2 and fragments read a step ahead are no faster.
template <int EPI, int WR, int WC, int MB, int NB, bool EXACT>
__global__ __launch_bounds__(64 * WR * WC) void fp8_tile_kernel(Fp8Args p) {
    constexpr int NW = WR * WC, TM = WR * 16 * MB, TN = WC * 16 * NB;
    constexpr bool DUAL = EPI == kSwiGLU;
    constexpr int A_BYTES = TM * kBlock, B_BYTES = TN * kBlock;
    constexpr int DA = A_BYTES / 1024 / NW, DB = B_BYTES / 1024 / NW;
    constexpr int STAGE = A_BYTES + B_BYTES + NW * 256;  // and 64 scales of every wavefront's load
    static_assert(TM / 64 < NW && DA * NW * 1024 == A_BYTES && DB * NW * 1024 == B_BYTES, "loads deal out evenly");
    static_assert(16 * NB <= kBlock, "a wavefront's columns share their weight scales");
    __shared__ __attribute__((aligned(1024))) unsigned char lds[2][STAGE];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wr = wave / WC, wc = wave % WC;
    const int per = (p.total + 7) / 8, local = blockIdx.x / 8;
    const int item = (blockIdx.x % 8) * per + local;
    if (local >= per || item >= p.total) return;
    // eight row blocks and all columns, row block fastest, then the next eight: the tiles that an XCD works on at a
    // time (32 in a row) share 8 panels of rows and 4 of columns, not one and 32
    const int split = item / p.tiles, tile = item - split * p.tiles;
    const int band = tile / (kBand * p.ncb), in = tile - band * kBand * p.ncb;
    const int height = min(kBand, (p.N + TM - 1) / TM - band * kBand);
    const int m0 = (band * kBand + in % height) * TM;
    const int n0 = (in / height) * (DUAL ? TN / 2 : TN);
    const long long ldx = (long long)p.groups * kBlock, ldw = (long long)p.groups * 2048;

    // rows: line r = 8 blk + lane / 8, piece c at c ^ swizzle(r)
    unsigned a_off[DA], b_off[DB];
#pragma unroll
    for (int j = 0; j < DA; ++j) {
        const int r = (wave * DA + j) * 8 + lane / 8;
        const int c = (lane % 8) ^ swizzle(r);
        a_off[j] = m0 + r < p.N ? (unsigned)(r * ldx + c * 16) : kNone;
    }
    // weights: piece q = half q & 1 of the tile's block q / 2; kSwiGLU: the tile's second half are up blocks
    const int q0 = wave * DB;
    const bool up = DUAL && q0 >= TN / 16;  // uniform: a wavefront's pieces are of one matrix
    static_assert(!DUAL || (TN / 16) % DB == 0, "a wavefront's pieces are of one matrix");
#pragma unroll
    for (int j = 0; j < DB; ++j) {
        const int q = q0 + j - (up ? TN / 16 : 0);
        const int blk = q >> 1;
        b_off[j] = (n0 >> 4) + blk < p.blocks ? (unsigned)(blk * ldw + (q & 1) * 1024 + lane * 16) : kNone;
    }
    const char* pa = p.codes + m0 * ldx;
    const char* pb = (up ? p.w[1] : p.w[0]) + (n0 >> 4) * ldw;
    // scales: wavefront w loads those of rows 64 w .., the next one the weights' (lane i: of columns 128 i .., kSwiGLU:
    // gate and up), the others none
    const float* ps = p.scales;
    unsigned s_off = kNone;
    long long s_step = 4ll * p.N;
    if (wave < TM / 64) {
        ps += m0 + wave * 64;
        if (m0 + wave * 64 + lane < p.N) s_off = lane * 4;
    } else if (wave == TM / 64) {
        s_step = 4;
        const int ob = n0 / kBlock;
        ps = p.ws[0] + (long long)ob * p.groups;
        if (DUAL) {
            // two tensors: lane 0 reads the gate's, and the up's go with a base of their own (below)
            s_off = lane == 0 ? 0 : kNone;
        } else if (lane < (TN + kBlock - 1) / kBlock && (ob + lane) * kBlock < p.O) {
            s_off = (unsigned)(4ll * lane * p.groups);
        }
    } else if (DUAL && wave == TM / 64 + 1) {
        s_step = 4;
        ps = p.ws[1] + (long long)(n0 / kBlock) * p.groups;
        s_off = lane == 0 ? 0 : kNone;
    }
    const char* psc = (const char*)ps;
    const int first = split * p.len, steps = min(p.len, p.groups - first);
    pa += (long long)first * kBlock;
    pb += (long long)first * 2048;
    psc += first * s_step;
    const unsigned lds0 = (unsigned)(size_t)(lds_ptr_t)&lds[0][0];
    auto load = [&](int st) {
        const unsigned base = lds0 + st * STAGE;
#pragma unroll
        for (int j = 0; j < DA; ++j) load_lds16(pa, a_off[j], base + (wave * DA + j) * 1024);
#pragma unroll
        for (int j = 0; j < DB; ++j) load_lds16(pb, b_off[j], base + A_BYTES + (q0 + j) * 1024);
        load_lds4(psc, s_off, base + A_BYTES + B_BYTES + wave * 256);
        pa += kBlock;
        pb += 2048;
        psc += s_step;
    };

    const int g = lane >> 4, r16 = lane & 15;
    const int ar = wr * 16 * MB + r16;
    const int a_rd = ar * 128 + ((g ^ swizzle(ar)) << 4);  // the second piece: ^ 64
    // tile block of the wavefront's column block j
    auto block_of = [&](int j) { return DUAL ? (j < NB / 2 ? wc * (NB / 2) + j : TN / 32 + wc * (NB / 2) + j - NB / 2) : wc * NB + j; };
    f32x4 acc[MB][NB];
#pragma unroll
    for (int i = 0; i < MB; ++i)
#pragma unroll
        for (int j = 0; j < NB; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    load(0);
    for (int b = 0; b < steps; ++b) {
        const int st = b & 1;
        // this wavefront's loads of step b have landed and its reads of step b - 1 are over, and after the barrier everybody's
        __builtin_amdgcn_s_waitcnt(all_done());
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        if (b + 1 < steps) load(st ^ 1);
        const unsigned char* A = &lds[st][0];
        const unsigned char* B = A + A_BYTES;
        const float* S = (const float*)(B + B_BYTES);
        decltype(operand<EXACT>(Op8{})) a[MB];
        float f[MB], f1[MB];
        const float w0 = S[DUAL ? TM : TM + (wc * 16 * NB) / kBlock], w1 = DUAL ? S[TM + 64] : 0.0f;
#pragma unroll
        for (int i = 0; i < MB; ++i) {
            Op8 r;
            r.u[0] = *(const uint4*)(A + a_rd + i * 2048);
            r.u[1] = *(const uint4*)(A + (a_rd ^ 64) + i * 2048);
            a[i] = operand<EXACT>(r);
            const float s = S[ar + 16 * i];
            f[i] = s * w0;
            f1[i] = s * w1;
        }
#pragma unroll
        for (int j = 0; j < NB; ++j) {
            Op8 r;
            const unsigned char* at = B + block_of(j) * 2048 + lane * 16;
            r.u[0] = *(const uint4*)at;
            r.u[1] = *(const uint4*)(at + 1024);
            const auto w = operand<EXACT>(r);
#pragma unroll
            for (int i = 0; i < MB; ++i) {
                const f32x4 d = mfma8(w, a[i]);
                const float s = DUAL && j >= NB / 2 ? f1[i] : f[i];
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[i][j][e] = fmaf(d[e], s, acc[i][j][e]);
            }
        }
    }

    // block (i, j): row 16 i + lane % 16, columns 16 j + 4 g .. + 3
    if (p.parts > 1) {
        const int ld = DUAL ? p.ldh : p.ldp;
        float* part = DUAL ? p.h + 2 * split * (long long)p.N * ld : p.part + split * (long long)p.N * ld;
        constexpr int NH = DUAL ? NB / 2 : NB;
#pragma unroll
        for (int i = 0; i < MB; ++i) {
            const int n = m0 + ar + 16 * i;
#pragma unroll
            for (int j = 0; j < NB; ++j) {
                const int o = n0 + (wc * NH + j % NH) * 16 + 4 * g;
                if (n < p.N && o < ld) *(f32x4*)(part + (j / NH * (long long)p.N + n) * ld + o) = acc[i][j];
            }
        }
        return;
    }
    if constexpr (!DUAL) {
        // The wavefront's outputs through LDS, so that its stores are whole lines (stores of 8 bytes in 16 rows each took
        // 24 of 272 us of 8192 x 4096 x 8192 more). Piece c of eight columns of row r lies at c ^ r.
        constexpr int PC = 2 * NB, ROWS = 16 * MB;
        static_assert(NW * ROWS * PC * 16 <= 2 * STAGE, "the tile in LDS");
        unsigned char* mine = &lds[0][0] + wave * (ROWS * PC * 16);
        auto piece = [&](int r, int c) { return mine + (r * PC + (c ^ (r & (PC - 1)))) * 16; };
        __syncthreads();
#pragma unroll
        for (int j = 0; j < NB; ++j) {
            const int o = n0 + (wc * NB + j) * 16 + 4 * g;
            float bias[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) bias[e] = p.bias != nullptr && o + e < p.O ? bf16_to_f32(p.bias[o + e]) : 0.0f;
#pragma unroll
            for (int i = 0; i < MB; ++i)
                *(uint2*)(piece(16 * i + r16, 2 * j + (g >> 1)) + (g & 1) * 8) =
                    make_uint2(pack_bf16(acc[i][j][0] + bias[0], acc[i][j][1] + bias[1]),
                               pack_bf16(acc[i][j][2] + bias[2], acc[i][j][3] + bias[3]));
        }
        wave_order();
#pragma unroll
        for (int t = 0; t < ROWS * PC / 64; ++t) {
            const int r = (t * 64 + lane) / PC, c = lane % PC;
            const uint4 v = *(const uint4*)piece(r, c);
            const int n = m0 + wr * ROWS + r, o = n0 + wc * 16 * NB + c * 8;
            if (n >= p.N) continue;
            unsigned short* dst = p.out + (long long)n * p.O + o;
            if (o + 8 <= p.O) {
                *(Any16*)dst = Any16{v.x, v.y, v.z, v.w};
            } else {
                const unsigned w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (o + e < p.O) dst[e] = (unsigned short)(w[e / 2] >> 16 * (e & 1));
            }
        }
    } else {
        constexpr int NH = NB / 2;
#pragma unroll
        for (int i = 0; i < MB; ++i)
#pragma unroll
            for (int j = 0; j < NH; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[i][j][e] = silu_fast(acc[i][j][e]) * acc[i][j + NH][e];
        if constexpr (TN / 2 == kBlock) {
            // the tile holds whole groups of h: their largest sizes through LDS, then codes
            unsigned(*top)[TM] = (unsigned(*)[TM])&lds[0][0];
            __syncthreads();
#pragma unroll
            for (int i = 0; i < MB; ++i) {
                unsigned m = 0;
#pragma unroll
                for (int j = 0; j < NH; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) m = max(m, size_bits(acc[i][j][e]));
                m = max(m, (unsigned)__shfl_xor((int)m, 16));
                m = max(m, (unsigned)__shfl_xor((int)m, 32));
                if (g == 0) top[wc][ar + 16 * i] = m;
            }
            __syncthreads();
            // and codes through LDS as the outputs above: block j of row r at j ^ r / 4
            unsigned char* mine = &lds[0][0] + sizeof(unsigned) * WC * TM + wave * (16 * MB * NH * 16);
            static_assert(NH == 4 && sizeof(unsigned) * WC * TM + NW * 16 * MB * NH * 16 <= 2 * STAGE, "the codes in LDS");
            auto piece = [&](int r, int j) { return mine + (r * NH + (j ^ (r >> 2 & 3))) * 16; };
#pragma unroll
            for (int i = 0; i < MB; ++i) {
                const int n = m0 + ar + 16 * i;
                unsigned m = top[0][ar + 16 * i];
#pragma unroll
                for (int c = 1; c < WC; ++c) m = max(m, top[c][ar + 16 * i]);
                const float s = scale_of(m);
                const Divisor by(s);
#pragma unroll
                for (int j = 0; j < NH; ++j)
                    *(unsigned*)(piece(16 * i + r16, j) + 4 * g) = by.codes4(acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]);
                if (g == 0 && wc == 0 && n < p.N) p.hs[(long long)(n0 / kBlock) * p.N + n] = s;
            }
            wave_order();
#pragma unroll
            for (int t = 0; t < MB; ++t) {
                const int r = 16 * t + lane / NH, j = lane % NH;
                const int n = m0 + wr * 16 * MB + r;
                if (n < p.N) *(uint4*)(p.hq + (long long)n * p.ldh + n0 + (wc * NH + j) * 16) = *(const uint4*)piece(r, j);
            }
        } else {
#pragma unroll
            for (int i = 0; i < MB; ++i) {
                const int n = m0 + ar + 16 * i;
                if (n >= p.N) continue;
#pragma unroll
                for (int j = 0; j < NH; ++j) *(f32x4*)(p.h + (long long)n * p.ldh + n0 + (wc * NH + j) * 16 + 4 * g) = acc[i][j];
            }
        }
    }
}

// Sums of the splits, in order, and the bias.
__global__ __launch_bounds__(256) void fp8_sum_kernel(Fp8Args p) {
    const int per = p.ldp / 4;
    const long long total = (long long)p.N * per, plane = (long long)p.N * p.ldp;
    for (long long e = (long long)blockIdx.x * 256 + threadIdx.x; e < total; e += (long long)gridDim.x * 256) {
        const int n = (int)(e / per), o = (int)(e - (long long)n * per) * 4;
        const float* at = p.part + (long long)n * p.ldp + o;
        f32x4 v = *(const f32x4*)at;
        for (int s = 1; s < p.parts; ++s) v = v + *(const f32x4*)(at + s * plane);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (o + i < p.O) {
                const float b = p.bias != nullptr ? bf16_to_f32(p.bias[o + i]) : 0.0f;
                p.out[(long long)n * p.O + o + i] = f32_to_bf16_rne(v[i] + b);
            }
    }
}

// ------------------------------------------------------------------ host
inline int groups_of(int k) { return (k + kBlock - 1) / kBlock; }

template <int SRC>
void rows_launch(const void* x, const Hidden& h, int N, int K, void* codes, float* scales, hipStream_t st) {
    const int groups = groups_of(K);
    const long long items = (long long)N * groups;
    unsigned char* c = (unsigned char*)codes;
    // four groups at once where there are enough of them for the CUs; h, whose loads are four times as many, one
    constexpr int U = SRC == kHidden ? 1 : 4;
    if (U > 1 && items >= 1 << 17)
        fp8_rows_kernel<SRC, U><<<(unsigned)std::min<long long>((items + 16 * U - 1) / (16 * U), 1 << 16), 256, 0, st>>>(x, h, N, K, groups, c, scales);
    else
        fp8_rows_kernel<SRC, 1><<<(unsigned)std::min<long long>((items + 15) / 16, 1 << 16), 256, 0, st>>>(x, h, N, K, groups, c, scales);
}

// Each block of 16 outputs reads all rows from L2: with many blocks, tiles take over from 33 rows on (1024 x 16384: 64
// rows 18.1 us, 65 in tiles 11.4; 4096 x 4096: 15.1 and 15.4).
inline bool few_rows(int N, int blocks) { return N <= (blocks > 512 ? 32 : 64); }

// Rows whose codes the few-row kernel makes itself: at most three groups for 16 of its lanes, one after the other (1 x
// 4096 x 4096: 5.2 us against 2.4 + 4.9 in two launches, 7 x 5000 x 3001, nine groups, 12.7 against 2.8 + 5.5), and
// at most 16 MB read by all work-groups together.
inline bool own_rows(int N, int K, int blocks, int bytes) {
    return N <= 16 && (long long)N * groups_of(K) <= 96 && (long long)N * K * bytes * blocks <= 16 << 20;
}
// Form of a product of N rows with `cols` weight rows (kSwiGLU: gate and up) over `groups` blocks of 128, and splits
// of the contraction: the least of an estimate. Few rows: a block of 16 outputs is a work-group, whose eight
// wavefronts take a step of 128 in `step` us, and splits pay their sums' launch (g and u: the pass over h, which is
// there anyway). Tiles: a CU's work-group takes `alone` us a step by itself, `shared` us of the CU's time beside others.
struct Plan {
    int tile;    // rows of a tile, 0: few rows
    int splits;
    int len;     // steps of a split
};
Plan plan_of(int N, int cols, int groups, bool dual) {
    Plan best{0, 1, groups};
    const int blocks = ceil_div(cols, dual ? 32 : 16);
    if (few_rows(N, blocks)) {
        // enough work-groups for the CUs, at least a step for every wavefront; without a pass over h at least eight
        best.splits = std::max(1, std::min({4, (256 + blocks / 2) / blocks, groups / (dual ? 8 : 32)}));
        return best;
    }
    static const struct { int rows, cols; float alone, shared; } kinds[2] = {{256, 256, 2.1f, 2.2f}, {64, 128, 0.58f, 0.38f}};
    float least = 1e30f;
    for (const auto& k : kinds) {
        const long long tiles = (long long)ceil_div(N, k.rows) * ceil_div(cols, k.cols);
        const int most = k.rows == 256 && dual ? 1 : 16;  // 256 columns are a group of h: they go on as codes
        for (int s = 1; s <= most && (s == 1 || groups / s >= 4); ++s) {
            const int len = ceil_div(groups, s);
            float us = std::max(k.alone, (float)((tiles * s + 255) / 256) * k.shared) * len;
            if (s > 1) us += (dual ? 0.0f : 4.0f) + (float)s * N * cols * 8.0f / 4e6f;
            if (us < least) least = us, best = {k.rows, ceil_div(groups, len), len};
        }
    }
    return best;
}
inline bool swiglu_codes(const Plan& q) { return q.tile == 256; }  // h leaves the kernel as codes
// Bytes of the sums of kLinear's splits.
inline size_t part_bytes(int N, int O, int groups) {
    const Plan q = plan_of(N, O, groups, false);
    return q.splits > 1 ? align_up((size_t)q.splits * N * ceil_div(O, 16) * 16 * 4, 256) : 0;
}

template <int EPI, int MR, int SRC>
void few_grid(const Fp8Args& p, hipStream_t st) {
    const size_t lds = sizeof(f32x4) * 8 * (EPI == kSwiGLU ? 2 : 1) * MR * 64 +
                       (SRC == kCodes ? 0 : (size_t)p.N * (p.groups * (kBlock + 4) + 16));
    fp8_few_kernel<EPI, MR, SRC><<<(unsigned)(p.blocks * p.parts), 512, lds, st>>>(p);
}

template <int EPI, int WR, int WC, int MB, int NB, bool EXACT = false>
void tile_grid(Fp8Args p, hipStream_t st) {
    constexpr int TM = WR * 16 * MB, TN = WC * 16 * NB;
    p.ncb = ceil_div(p.O, EPI == kSwiGLU ? TN / 2 : TN);
    p.tiles = ceil_div(p.N, TM) * p.ncb;
    p.total = p.tiles * p.parts;
    fp8_tile_kernel<EPI, WR, WC, MB, NB, EXACT><<<(unsigned)(ceil_div(p.total, 8) * 8), 64 * WR * WC, 0, st>>>(p);
}

// Rows as codes, or (few rows, SRC) made into codes in the kernel; part: the workspace of kLinear's splits.
template <int EPI, int SRC = kCodes>
void product_launch(Fp8Args p, float* part, hipStream_t st) {
    const Plan q = plan_of(p.N, EPI == kSwiGLU ? 2 * p.O : p.O, p.groups, EPI == kSwiGLU);
    p.parts = q.splits;
    p.len = q.len;
    p.part = part;
    p.ldp = p.blocks * 16;
    if (SRC != kCodes) few_grid<EPI, 1, SRC>(p, st);
    else if (q.tile == 0 && p.N <= 16) few_grid<EPI, 1, kCodes>(p, st);
    else if (q.tile == 0 && p.N <= 32) few_grid<EPI, 2, kCodes>(p, st);
    else if (q.tile == 0 && p.N <= 48) few_grid<EPI, 3, kCodes>(p, st);
    else if (q.tile == 0) few_grid<EPI, 4, kCodes>(p, st);
    else if (q.tile == 256) tile_grid<EPI, 4, 2, 4, 8>(p, st);
    else if (EPI == kSwiGLU && (long long)p.N * p.O <= kExactH) tile_grid<EPI, 2, 2, 2, 4, EPI == kSwiGLU>(p, st);
    else tile_grid<EPI, 2, 2, 2, 4>(p, st);
    if (EPI == kLinear && p.parts > 1) {
        const long long quads = (long long)p.N * (p.ldp / 4);
        fp8_sum_kernel<<<(unsigned)std::min<long long>((quads + 255) / 256, 8192), 256, 0, st>>>(p);
    }
}

Fp8Args product_of(const void* codes, const float* scales, int N, const yvmoe_fp8_matrix* w) {
    Fp8Args p{};
    p.codes = (const char*)codes;
    p.scales = scales;
    p.N = N;
    p.K = w->in_features;
    p.O = w->out_features;
    p.groups = groups_of(w->in_features);
    p.blocks = ceil_div(w->out_features, 16);
    p.w[0] = (const char*)w->codes;
    p.ws[0] = (const float*)w->scales;
    return p;
}

inline size_t codes_bytes(int N, int K) { return align_up((size_t)N * groups_of(K) * kBlock, 256); }
inline size_t scales_bytes(int N, int K) { return align_up((size_t)N * groups_of(K) * 4, 256); }

}  // namespace

int fp8_rows_launch(const void* x, int act, int N, int K, void* codes, float* scales, hipStream_t st) {
    if (act == YVMOE_ACT_F32) rows_launch<kF32>(x, Hidden{}, N, K, codes, scales, st);
    else rows_launch<kBf16>(x, Hidden{}, N, K, codes, scales, st);
    YV_LAUNCH_CHECK("fp8 rows");
    return YVMOE_OK;
}

size_t fp8_product_ws(int N, int K, int O) { return part_bytes(N, O, groups_of(K)); }
size_t fp8_linear_ws(int N, int K, int O) { return codes_bytes(N, K) + scales_bytes(N, K) + fp8_product_ws(N, K, O); }

int fp8_product_launch(const void* codes, const float* scales, int N, const yvmoe_fp8_matrix* w, const void* bias,
                       void* out, char* ws, hipStream_t st) {
    Fp8Args p = product_of(codes, scales, N, w);
    p.bias = (const unsigned short*)bias;
    p.out = (unsigned short*)out;
    product_launch<kLinear>(p, (float*)ws, st);
    YV_LAUNCH_CHECK("fp8 linear");
    return YVMOE_OK;
}

int fp8_linear_launch(const void* x, int N, const yvmoe_fp8_matrix* w, const void* bias, void* out, char* ws,
                      hipStream_t st) {
    float* scales = (float*)(ws + codes_bytes(N, w->in_features));
    float* part = (float*)((char*)scales + scales_bytes(N, w->in_features));
    Fp8Args p = product_of(ws, scales, N, w);
    p.bias = (const unsigned short*)bias;
    p.out = (unsigned short*)out;
    p.x = x;
    if (own_rows(N, p.K, p.blocks, 2)) {
        product_launch<kLinear, kBf16>(p, part, st);
    } else {
        rows_launch<kBf16>(x, Hidden{}, N, p.K, ws, scales, st);
        product_launch<kLinear>(p, part, st);
    }
    YV_LAUNCH_CHECK("fp8 linear");
    return YVMOE_OK;
}

size_t fp8_swiglu_ws(int N, int H, int F) {
    const Plan q = plan_of(N, 2 * F, groups_of(H), true);
    const size_t h = (size_t)N * groups_of(F) * kBlock * 4;
    return fp8_linear_ws(N, F, H) + codes_bytes(N, H) + scales_bytes(N, H) +
           (swiglu_codes(q) ? 0 : align_up((q.splits > 1 ? 2 * q.splits : 1) * h, 256));
}

int fp8_swiglu_launch(const void* x, int N, const yvmoe_fp8_matrix* gate, const yvmoe_fp8_matrix* up,
                      const yvmoe_fp8_matrix* down, void* out, char* ws, hipStream_t st) {
    const int H = gate->in_features, F = gate->out_features;
    char* xq = ws;
    float* xs = (float*)(xq + codes_bytes(N, H));
    char* hq = (char*)xs + scales_bytes(N, H);
    float* hs = (float*)(hq + codes_bytes(N, F));
    float* part = (float*)((char*)hs + scales_bytes(N, F));
    float* h = (float*)((char*)part + fp8_product_ws(N, F, H));
    Fp8Args p = product_of(xq, xs, N, gate);
    p.w[1] = (const char*)up->codes;
    p.ws[1] = (const float*)up->scales;
    p.ldh = groups_of(F) * kBlock;
    p.h = h;
    p.hq = (unsigned char*)hq;
    p.hs = hs;
    p.x = x;
    const Plan plan = plan_of(N, 2 * F, p.groups, true);
    if (own_rows(N, H, p.blocks * plan.splits, 2)) {
        product_launch<kSwiGLU, kBf16>(p, nullptr, st);
    } else {
        rows_launch<kBf16>(x, Hidden{}, N, H, xq, xs, st);
        product_launch<kSwiGLU>(p, nullptr, st);
    }
    const Hidden hidden{h, plan.splits > 1 ? plan.splits : 0, p.ldh, (long long)N * p.ldh};
    Fp8Args q = product_of(hq, hs, N, down);
    q.out = (unsigned short*)out;
    q.hidden = hidden;
    if (own_rows(N, F, q.blocks, plan.splits > 1 ? 8 * plan.splits : 4)) {
        product_launch<kLinear, kHidden>(q, part, st);
    } else {
        if (!swiglu_codes(plan)) rows_launch<kHidden>(nullptr, hidden, N, F, hq, hs, st);
        product_launch<kLinear>(q, part, st);
    }
    YV_LAUNCH_CHECK("fp8 swiglu");
    return YVMOE_OK;
}

}  // namespace yvmoe
