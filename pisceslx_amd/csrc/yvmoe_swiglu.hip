// Gated feed-forward block on full-precision weights, forward and backward, for gfx950:
//
//   g = x Wgᵀ, u = x Wuᵀ, h = silu(g) u, y = h Wdᵀ
//   dh = dy Wd, s = 1 / (1 + exp(-g)), du = dh g s, dg = dh u s (1 + g (1 - s))
//   dx = dg Wg + du Wu, dWg = dgᵀ x, dWu = duᵀ x, dWd = dyᵀ h
//
// (the expert of model/moe/expert.py:475-489 and its gradients).
//
// Products. Every product runs on v_mfma_f32_16x16x32_bf16 with fp32 sums. bf16 operands go in as they are.
// An fp32 operand is the sum of three bf16 terms (24 bits), and a product the six of the nine term products
// that reach fp32's last bits, the smallest first, so that the running sum is small while they are added.
// Roundings of the bf16 form: h, dg and du once each, where they become operands, and the outputs; g and u are
// kept for the backward pass in fp32 (in bf16 the gradients of the gate and up weights would be twice as far
// from the exact ones: 3.7e-3 relative instead of 2.4e-3). The fp32 form rounds h, dg and du to their 24 bits.
#include <algorithm>

#include "yvmoe_frag.h"
#include "yvmoe_internal.h"

namespace yvmoe {
namespace {

typedef __attribute__((address_space(3))) void* lds_ptr_t;
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4* lds_s16x4_t;

constexpr int kSeg = 12;      // operand pairs of a launch: 6 term products x 2 matrices
constexpr int kChunk = 64;    // contraction elements per LDS stage

constexpr int kBand = 8;      // row blocks that neighbouring tiles share columns over

// Term products of an fp32 product, smallest first: (term of A, term of B).
constexpr int kTermA[6] = {2, 0, 1, 1, 0, 0};
constexpr int kTermB[6] = {0, 2, 1, 0, 1, 0};

enum Epi { kOut, kSwiGLU, kGrad };

// What becomes of a product's sums.
struct Finish {
    int M, N;            // output rows and columns (kSwiGLU: columns of h)
    float* part;         // with several splits their sums [split][M][ldp], kSwiGLU [split][2][M][ldp]
    int ldp;
    // kOut: rows [0, split) to out, rows [split_at, ...) to out1 at row - split_at (split_at >= split)
    void* out;
    void* out1;
    int ldo, split, split_at, f32;
    // kSwiGLU, kGrad: h [M][ldh] and d = dg, du [M][2 ldh] (Planes; elements between them), and g and u, which kSwiGLU
    // may not have to keep
    long long plane_h, plane_d;
    char* h;
    char* d;
    float* gu;           // [2][M][ldh]
    int ldh;
};
// Operands in memory: rows by contraction ("KC": the contraction index is contiguous) or contraction by rows ("MC").
struct TileArgs : Finish {
    int ka, kb;          // contraction elements of A and of B; beyond them both count as zero
    int lda, ldb;        // elements between rows in memory
    int nseg;
    int ncb, tiles, total;  // column blocks, tiles, tiles x splits
    int split_chunks;       // chunks of a split of the contraction (all of them: one split)
    const char* a[kSeg];
    const char* b[kSeg];
    const char* b1[kSeg];  // kSwiGLU: the up matrix
};

// s_waitcnt immediates (gfx9 encoding)
constexpr int vm_only(int n) { return (n & 0xf) | ((n >> 4) << 14) | (0x7 << 4) | (0xf << 8); }
constexpr int lgkm0() { return 0xf | (0x3 << 14) | (0x7 << 4); }
constexpr int all_done() { return vm_only(0) & lgkm0(); }  // loads from memory and reads of LDS

// 16 bytes per lane from base + off to LDS at m0 + 16 lane; an offset of kNone reads zeros: the buffer's
// bounds are 2^31 bytes, which no other offset reaches (the host checks), and no lane reads behind a tensor.
constexpr unsigned kNone = 0xfffffff0u;
typedef int i32x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ void load_lds(const char* base, unsigned off, unsigned m0) {
    const unsigned long long p = (unsigned long long)base;
    const i32x4 rsrc = {(int)(unsigned)p, (int)(unsigned)(p >> 32) & 0xffff, (int)0x80000000u, 0x00020000};
    asm volatile("buffer_load_dwordx4 %0, %1, 0 offen lds" : : "v"(off), "s"(rsrc), "{m0}"(m0) : "memory");
}
__device__ __forceinline__ void mfma_acc(f32x4& acc, const bf16x8& a, const bf16x8& b) {
    asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(acc) : "v"(a), "v"(b));
}

// How many of n instructions go before MFMA i of t, spread over the first 4 / q of them.
constexpr int among(int i, int n, int t, int q) { return i * n * q / (4 * t) < n ? i * n * q / (4 * t) : n; }

// How h and d are stored: one bf16 plane (rounded), three (a value is the sum of three bf16 numbers), or fp32; kAlone: one
// plane of h, and neither g and u nor sums of splits. kOut: kFar, results that are read long after (past()).
enum Planes { kOne = 1, kAlone = 2, kThree = 3, kFp32 = 0, kFar = 4 };
// Four values to element e of h or d.
template <int PL>
__device__ __forceinline__ void put(char* base, long long e, long long plane, const float (&v)[4]) {
    if (PL == kFp32) {
        *(f32x4*)((float*)base + e) = f32x4{v[0], v[1], v[2], v[3]};
        return;
    }
    unsigned short* p = (unsigned short*)base + e;
    float r[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
    for (int t = 0; t < (PL == kThree ? 3 : 1); ++t) {
        const unsigned lo = pack_bf16(r[0], r[1]), hi = pack_bf16(r[2], r[3]);
        *(uint2*)(p + t * plane) = make_uint2(lo, hi);
        r[0] -= bf16_to_f32((unsigned short)(lo & 0xffff)), r[1] -= bf16_to_f32((unsigned short)(lo >> 16));
        r[2] -= bf16_to_f32((unsigned short)(hi & 0xffff)), r[3] -= bf16_to_f32((unsigned short)(hi >> 16));
    }
}

// What is not read before much else has been goes past the caches, which hold what the next products read: g and u, and
// the gradients of the weights (steps of 8192 x 1024 x 2816 644 -> 603 us with g and u, of 2000 x 5120 x 1536 388 -> 351
// to 372 with the gradients, of 4096 x 4096 x 11264 2937 -> 2885 with both).
template <class V>
__device__ __forceinline__ void past(void* at, V v) {
    __builtin_nontemporal_store(v, (V*)at);
}
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

// What becomes of four sums of row m, columns n .. n + 3.
template <int PL>
__device__ __forceinline__ void finish_out(const Finish& p, int m, int n, f32x4 v) {
    const bool first = m < p.split;
    if ((!first && m < p.split_at) || m >= p.M || n >= p.N) return;
    void* o = first ? p.out : p.out1;
    const long long e = (long long)(first ? m : m - p.split_at) * p.ldo + n;
    if (n + 4 <= p.N && p.ldo % 4 == 0) {
        const u32x2 b = {pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3])};
        if constexpr (PL == kFar) {
            if (p.f32) past((float*)o + e, v);
            else past((unsigned short*)o + e, b);
        } else {
            if (p.f32) *(f32x4*)((float*)o + e) = v;
            else *(u32x2*)((unsigned short*)o + e) = b;
        }
    } else {
#pragma unroll
        for (int q = 0; q < 4; ++q)
            if (n + q < p.N) {
                if (p.f32) ((float*)o)[e + q] = v[q];
                else ((unsigned short*)o)[e + q] = f32_to_bf16_rne(v[q]);
            }
    }
}
// Columns from N to ldh are sums of zeros and written as such: they are operands of products.
template <int PL>
__device__ __forceinline__ void finish_swiglu(const Finish& p, int m, int n, f32x4 g, f32x4 u) {
    if (m >= p.M || n >= p.ldh) return;
    const long long e = (long long)m * p.ldh + n;
    if (PL != kAlone && p.gu != nullptr) {
        past(p.gu + e, g);
        past(p.gu + (long long)p.M * p.ldh + e, u);
    }
    float h[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) h[q] = silu_fast(g[q]) * u[q];
    put<PL>(p.h, e, p.plane_h, h);
}
template <int PL>
__device__ __forceinline__ void finish_grad(const Finish& p, int m, int n, f32x4 dh) {
    if (m >= p.M || n >= p.ldh) return;
    const long long e = (long long)m * p.ldh + n;
    const f32x4 g = __builtin_nontemporal_load((const f32x4*)(p.gu + e)),
                u = __builtin_nontemporal_load((const f32x4*)(p.gu + (long long)p.M * p.ldh + e));
    float dg[4], du[4], h[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const float s = sigmoid_fast(g[q]), a = g[q] * s;
        h[q] = a * u[q];
        du[q] = dh[q] * a;
        dg[q] = dh[q] * u[q] * (s + a * (1.0f - s));
    }
    const long long ed = (long long)m * 2 * p.ldh + n;
    put<PL>(p.d, ed, p.plane_d, dg);
    put<PL>(p.d, ed + p.ldh, p.plane_d, du);
    put<PL>(p.h, e, p.plane_h, h);
}
// Blocks of 16 rows that a wavefront moves through LDS at a time, and their 16-byte quads: 4 x 4 NB KB fit the stages.
constexpr int finish_rows(int mb) { return mb < 4 ? mb : 4; }
constexpr int finish_quads(int mb, int nb) { return finish_rows(mb) * nb * 64; }
template <int EPI, int PL>
__device__ __forceinline__ void finish_quad(const Finish& p, int m, int n, f32x4 v, f32x4 u, int split) {
    if (p.part != nullptr) {
        if (m >= p.M || n >= p.ldp) return;
        float* to = p.part + ((long long)split * (EPI == kSwiGLU ? 2 : 1) * p.M + m) * p.ldp + n;
        *(f32x4*)to = v;
        if (EPI == kSwiGLU) *(f32x4*)(to + (long long)p.M * p.ldp) = u;
    } else if constexpr (EPI == kOut) {
        finish_out<PL>(p, m, n, v);
    } else if constexpr (EPI == kGrad) {
        finish_grad<PL>(p, m, n, v);
    } else {
        finish_swiglu<PL>(p, m, n, v, u);
    }
}
// h of the wavefront's block AT and of those after it. Written out by recursion: `#pragma unroll` gives up on bodies as
// long as these, and the sums would then go through memory.
template <int MB, int NB, int AT = 0>
__device__ __forceinline__ void finish_blocks(const Finish& p, const f32x4 (&acc)[MB][NB], int m, int n) {
    constexpr int NH = NB / 2, i = AT / NH, j = AT % NH;
    finish_swiglu<kAlone>(p, m + 16 * i, n + 16 * j, acc[i][j], acc[i][j + NH]);
    asm volatile("" ::: "memory");  // one block's addresses at a time
    if constexpr (AT + 1 < MB * NH) finish_blocks<MB, NB, AT + 1>(p, acc, m, n);
}
// A wavefront's blocks, from row m and column n on: lane 16 g + r of block (i, j) holds row 16 i + r, columns 16 j + 4 g
// .. + 3 (kSwiGLU: of gate, then of up). They go through LDS, B blocks of rows at a time, so that the lanes then hold
// whole rows and what they write and read is whole lines, not quarters of 16 (a training step of
// 4096 x 4096 x 11264 3008 us, so 2940; fp32, 2052 x 1024 x 2816, 787 and 760). Quad c of row r lies at c ^ r. The
// loop over the quads stays one: written out, the code would come from memory more slowly than it runs.
template <int EPI, int PL, int MB, int NB>
__device__ __forceinline__ void finish(const Finish& p, const f32x4 (&acc)[MB][NB], f32x4* mine, int m, int n, int split) {
    constexpr int NH = EPI == kSwiGLU ? NB / 2 : NB, Q = 4 * NH, B = finish_rows(MB), G = B * NH < 4 ? B * NH : 4;
    const int lane = threadIdx.x & 63;
    // bf16 h alone: 8 bytes for 32 that LDS would move (8192 x 1024 x 2816: 149 us a block, through LDS 159)
    if constexpr (PL == kAlone) return finish_blocks(p, acc, m + (lane & 15), n + 4 * (lane >> 4));
    auto quad = [&](int mat, int r, int c) { return mine + (mat * 16 * B + r) * Q + (c ^ (r & 15 & (Q - 1))); };
#pragma unroll
    for (int i0 = 0; i0 < MB; i0 += B) {
#pragma unroll
        for (int i = 0; i < B; ++i)
#pragma unroll
            for (int j = 0; j < NB; ++j)
                *quad(j / NH, 16 * i + (lane & 15), 4 * (j % NH) + (lane >> 4)) = acc[i0 + i][j];
        wave_order();
#pragma unroll 1
        for (int t = 0; t < B * NH; t += G) {
            f32x4 v[G], u[G];
#pragma unroll
            for (int k = 0; k < G; ++k) {
                const int r = (64 * (t + k) + lane) / Q, c = lane % Q;
                v[k] = *quad(0, r, c), u[k] = *quad(NB / NH - 1, r, c);
            }
#pragma unroll
            for (int k = 0; k < G; ++k)
                finish_quad<EPI, PL>(p, m + 16 * i0 + (64 * (t + k) + lane) / Q, n + 4 * (lane % Q), v[k], u[k], split);
        }
        wave_order();
    }
}

// Of bf16, whose lane groups g read pieces g, and of fp32, where they read pieces 2 g.
template <bool F32>
__device__ __forceinline__ int swizzle(int r) {
    return F32 ? (r ^ r >> 3 & 1) & 7 : (r >> 1 & 3) | ((r ^ r >> 3) & 1) << 2;
}

// One operand's part of a stage: TW rows (or columns) of a chunk, 64 contraction elements of bf16 or 32 of fp32.
// KC: 128-byte rows in 16-byte pieces, piece c of row r at c ^ swizzle(r): the 16 lanes that read together, of two
//     neighbouring lane groups and 16 rows, then lie in different banks.
// MC: rows of TW elements, in groups of 16 elements (bf16: pairs of pieces, fp32: four), group p of row k at p ^ f(k).
//     bf16: f(k) = (k & 3) | (k >> 1 & 4) (64 wide: k & 3), so that the four rows that 16 lanes read together lie in
//     different banks; fp32: f(k) = k >> 3 & 3, the four lane groups' rows.
template <bool MC, int TW, bool F32 = false>
struct Stage {
    static constexpr int BYTES = TW * 128;
    static constexpr int LOADS = BYTES / 1024 / 4;  // of a wavefront
    static constexpr int ES = F32 ? 4 : 2, CHUNK = 128 / ES, PE = 16 / ES;
    static constexpr int ROW = TW * ES;             // MC: bytes of a row, pieces of a load's rows
    static constexpr int RPL = ROW > 1024 ? 1 : 1024 / ROW, PPR = ROW / 16;
    static_assert(ROW <= 1024, "a load holds whole rows");
    unsigned off[LOADS];
    long long step;  // bytes per chunk

    __device__ __forceinline__ static int f(int k) {
        return F32 ? k >> 3 & 3 : ((k & 3) | (k >> 1 & 4)) & (TW >= 128 ? 7 : 3);
    }
    // the first of the lane's elements in load j of a wavefront: row of the tile and contraction element
    __device__ __forceinline__ static void place(int wave, int lane, int j, int& m, int& k) {
        const int blk = wave * LOADS + j;
        if (MC) {
            constexpr int GP = 16 / PE;  // pieces of a group
            const int piece = lane % PPR;
            k = blk * RPL + lane / PPR;
            m = ((piece / GP ^ f(k)) * GP + piece % GP) * PE;
        } else {
            m = blk * 8 + lane / 8;
            k = ((lane % 8) ^ swizzle<F32>(m)) * PE;
        }
    }
    // row0: first row of the tile in the operand, rows: how many the operand has
    __device__ __forceinline__ void init(int wave, int lane, int row0, int rows, int ld) {
#pragma unroll
        for (int j = 0; j < LOADS; ++j) {
            int m, k;
            place(wave, lane, j, m, k);
            // KC offsets count rows from the tile, MC offsets columns from the matrix
            const long long e = MC ? (long long)k * ld + row0 + m : (long long)m * ld + k;
            off[j] = row0 + m < rows ? (unsigned)(e * ES) : kNone;
        }
        step = MC ? (long long)CHUNK * ld * ES : 128;
    }
    // load j of the chunk that starts `left` elements before the operand's end; `as`: the wavefront whose rows it takes
    __device__ __forceinline__ void load(int wave, int as, int lane, int j, const char* at, int left, unsigned lds) const {
        unsigned o = off[j];
        if (left < CHUNK) {
            int m, k;
            place(as, lane, j, m, k);
            o = k < left ? o : kNone;
        }
        load_lds(at, o, lds + (wave * LOADS + j) * 1024);
    }
};

// Fragment of the MFMA step s (32 contraction elements) for the 16 rows from r0: lane 16 g + r gets row r0 + r,
// elements 8 g .. 8 g + 7 of the step.
template <bool MC, int TW>
struct Reader {
    int at;  // lane's byte for r0 = the wavefront's first row, s = 0
    __device__ __forceinline__ void init(int lane, int r0) {
        const int g = lane >> 4, i = lane & 15;
        if (MC) {
            const int k = 8 * g + (i >> 2);
            at = k * TW * 2 + (((r0 >> 4) ^ Stage<MC, TW>::f(k)) << 5) + (i & 3) * 8;
        } else {
            const int r = r0 + i;
            at = r * 128 + ((g ^ swizzle<false>(r)) << 4);
        }
    }
    // blocks of 16 rows are counted from the wavefront's first, which is a multiple of their number
    __device__ __forceinline__ bf16x8 read(const unsigned char* stage, int s, int blk) const {
        if (MC) {
            const unsigned char* p = stage + (at ^ blk << 5) + s * 32 * TW * 2;
            union { s16x4 h[2]; bf16x8 v; } f;
            f.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t)p);
            f.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t)(p + 4 * TW * 2));
            return f.v;
        }
        return *(const bf16x8*)(stage + (at ^ s << 6) + blk * 2048);
    }
};
// The same of fp32, whose chunk is one step, as three bf16 terms: cut off, not rounded, so that two take a mask and a
// subtraction each, and all 24 bits are kept.
template <bool MC, int TW>
struct Reader32 {
    int at;
    __device__ __forceinline__ void init(int lane, int r0) {
        const int g = lane >> 4, i = lane & 15;
        if (MC) {
            at = 8 * g * TW * 4 + (((r0 >> 4) ^ Stage<MC, TW, true>::f(8 * g)) << 6) + i * 4;
        } else {
            const int r = r0 + i;
            at = r * 128 + (((2 * g) ^ swizzle<true>(r)) << 4);
        }
    }
    __device__ __forceinline__ void read(const unsigned char* stage, int blk, float (&v)[8]) const {
        if (MC) {
            const unsigned char* p = stage + (at ^ blk << 6);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = *(const float*)(p + e * TW * 4);
        } else {
            const float4 lo = *(const float4*)(stage + at + blk * 2048), hi = *(const float4*)(stage + (at ^ 16) + blk * 2048);
            v[0] = lo.x, v[1] = lo.y, v[2] = lo.z, v[3] = lo.w, v[4] = hi.x, v[5] = hi.y, v[6] = hi.z, v[7] = hi.w;
        }
    }
    __device__ __forceinline__ static void terms(const float (&v)[8], bf16x8 (&t)[3]) {
        union { unsigned u[4]; bf16x8 b; } f;
        float r[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) r[e] = v[e];
#pragma unroll
        for (int k = 0; k < 3; ++k) {
#pragma unroll
            for (int e = 0; e < 4; ++e)  // the upper halves of two values
                f.u[e] = __builtin_amdgcn_perm(__float_as_uint(r[2 * e + 1]), __float_as_uint(r[2 * e]), 0x07060302u);
            t[k] = f.b;
            if (k < 2) {
#pragma unroll
                for (int e = 0; e < 8; ++e) r[e] -= __uint_as_float(__float_as_uint(r[e]) & 0xffff0000u);
            }
        }
    }
};

// One tile of 32 MB rows x 32 NB columns (kSwiGLU: 16 NB columns of h, gate and up) by four wavefronts in a
// 2 x 2 grid, each 16 MB x 16 NB: MB x NB blocks of 16 x 16, fp32 sums in AGPRs (an MFMA in inline assembly
// with the sum as one tied AGPR operand, so that the register allocator copies none). Chunks of 64
// contraction elements move to LDS by direct loads through two stages; the MFMAs of a chunk run in two
// halves with the next half's fragment reads (in the first four fifths of them) and the loads of the chunk after next
// among them, one barrier between the halves. The columns' operand is the MFMA's first, so that a lane holds four
// consecutive columns of one row. Bound by the matrix unit, whose operands LDS must bring (1536 of 2048 cycles a chunk):
// 4096 x 4096 x 11264, bf16: gate and up 643 us (1.18 PFLOP/s), down 285 (1.33, without the loads from memory 1.68), dx
// 566 (1.34), weights' gradients 665 and 332 (1.14); dh 459, 120 of which read g and u and write d and h. The 256 x 256 form
// of kAlone spills one register.
template <int EPI, int PL, bool AMC, bool BMC, int MB, int NB>
__global__ __launch_bounds__(256) void swiglu_tile_kernel(TileArgs p) {
    constexpr int TM = 32 * MB, TN = 32 * NB;
    constexpr int T = MB * NB, R = MB + NB;
    constexpr bool DUAL = EPI == kSwiGLU;
    typedef Stage<AMC, TM> SA;
    typedef Stage<BMC, TN> SB;
    constexpr int DA = SA::LOADS, D = SA::LOADS + SB::LOADS;
    __shared__ __attribute__((aligned(1024))) unsigned char lds[2][SA::BYTES + SB::BYTES];
    static_assert(4 * 16 * finish_quads(MB, NB) <= 2 * (SA::BYTES + SB::BYTES), "the sums in LDS");
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wr = wave >> 1, wc = wave & 1;
    // tiles in 8 contiguous ranges (one per XCD)
    const int per = (p.total + 7) / 8;
    const int local = blockIdx.x / 8;
    const int item = (blockIdx.x % 8) * per + local;
    if (local >= per || item >= p.total) return;
    // splits slowest: tiles of one split, which run together, share their operands
    const int split = item / p.tiles, tile = item - split * p.tiles;
    // eight row blocks and all columns, row block fastest, then the next eight: the tiles that an XCD works on at a
    // time (32 in a row) share 8 panels of rows and 4 of columns, not one and 32
    const int band = tile / (kBand * p.ncb), in = tile - band * kBand * p.ncb;
    const int height = min(kBand, (p.M + TM - 1) / TM - band * kBand);
    const int m0 = (band * kBand + in % height) * TM;
    const int n0 = (in / height) * (DUAL ? TN / 2 : TN);

    SA sa;
    SB sb;
    sa.init(wave, lane, m0, p.M, p.lda);
    // kSwiGLU: tile columns 0 .. TN / 2 - 1 are gate rows, the others the same up rows: wavefronts 0 and 1 load
    // the gate's half, 2 and 3 the up's
    sb.init(DUAL ? wave & 1 : wave, lane, n0, p.N, p.ldb);
    static_assert(!DUAL || !BMC, "the forward pass reads weights row by row");
    const long long a_tile = AMC ? (long long)m0 * 2 : (long long)m0 * p.lda * 2;
    const long long b_tile = BMC ? (long long)n0 * 2 : (long long)n0 * p.ldb * 2;
    const unsigned lds0 = (unsigned)(size_t)(lds_ptr_t)&lds[0][0];
    const int cps = (max(p.ka, p.kb) + kChunk - 1) / kChunk;  // chunks per segment
    int chunks = cps * p.nseg;

    // the next chunk to load: segment and place in it
    int seg = 0, at = 0;
    const int first = split * p.split_chunks;
    chunks = min(p.split_chunks, chunks - first);
    if (first > 0) seg = first / cps, at = (first - seg * cps) * kChunk;
    const char *pa = p.a[seg] + (AMC ? 0 : a_tile) + (at / kChunk) * sa.step,
               *pb = (DUAL && wave >= 2 ? p.b1[seg] : p.b[seg]) + (BMC ? 0 : b_tile) + (at / kChunk) * sb.step;
    auto load = [&](int st, int j) {
        const unsigned base = lds0 + st * (SA::BYTES + SB::BYTES);
        if (j < DA) {
            sa.load(wave, wave, lane, j, pa, p.ka - at, base);
        } else {
            sb.load(wave, DUAL ? wave & 1 : wave, lane, j - DA, pb, p.kb - at, base + SA::BYTES);
        }
    };
    auto advance = [&]() {
        at += kChunk;
        pa += sa.step;
        pb += sb.step;
        if (at >= cps * kChunk && seg + 1 < p.nseg) {
            ++seg;
            at = 0;
            pa = p.a[seg] + (AMC ? 0 : a_tile);
            pb = (DUAL && wave >= 2 ? p.b1[seg] : p.b[seg]) + (BMC ? 0 : b_tile);
        }
    };

    Reader<AMC, TM> ra;
    Reader<BMC, TN> rb;
    ra.init(lane, wr * 16 * MB);
    // kSwiGLU: the wavefront's first NB / 2 blocks are gate columns, the others the up columns of the same
    rb.init(lane, DUAL ? wc * 8 * NB : wc * 16 * NB);
    f32x4 acc[MB][NB];
#pragma unroll
    for (int i = 0; i < MB; ++i)
#pragma unroll
        for (int j = 0; j < NB; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    bf16x8 fa[2][MB], fb[2][NB];
    auto read = [&](int st, int s, int q) {
        // in the order of use: the first column block, all row blocks, the other column blocks
        if (q >= 1 && q <= MB) {
            fa[s][q - 1] = ra.read(&lds[st][0], s, q - 1);
        } else {
            const int j = q == 0 ? 0 : q - MB;
            fb[s][j] = rb.read(&lds[st][SA::BYTES], s, DUAL && j >= NB / 2 ? j - NB / 2 + NB : j);
        }
    };
    if (chunks > 0) {
#pragma unroll
        for (int j = 0; j < D; ++j) load(0, j);
        if (chunks > 1) advance();
#pragma unroll
        for (int j = 0; j < D; ++j) load(1, j);
        __builtin_amdgcn_s_waitcnt(vm_only(D));  // nothing has been read from LDS yet
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
#pragma unroll
        for (int q = 0; q < R; ++q) read(0, 0, q);
        for (int c = 0; c < chunks; ++c) {
            const int st = c & 1;
#pragma unroll
            for (int i = 0; i < T; ++i) {
                mfma_acc(acc[i % MB][i / MB], fb[0][i / MB], fa[0][i % MB]);
#pragma unroll
                for (int q = among(i, R, T, 5); q < among(i + 1, R, T, 5); ++q) read(st, 1, q);
            }
            // this wavefront has read chunk c and holds its loads of chunk c + 1: the barrier frees the stage
            // for chunk c + 2 and publishes chunk c + 1
            __builtin_amdgcn_s_waitcnt(vm_only(0));
            __builtin_amdgcn_s_waitcnt(lgkm0());
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            // past the last chunk the loads repeat it and the reads see an idle stage; neither is used
            if (c + 2 < chunks) advance();
#pragma unroll
            for (int i = 0; i < T; ++i) {
                mfma_acc(acc[i % MB][i / MB], fb[1][i / MB], fa[1][i % MB]);
#pragma unroll
                for (int j = among(i, D, T, 4); j < among(i + 1, D, T, 4); ++j) load(st, j);
#pragma unroll
                for (int q = among(i, R, T, 5); q < among(i + 1, R, T, 5); ++q) read(st ^ 1, 0, q);
            }
        }
        // the repeated loads land before the work-group ends; wait states between the last MFMAs and the
        // reads of their sums
        __builtin_amdgcn_s_waitcnt(vm_only(0));
    }
    asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 7" ::: "memory");

    const Finish fin = p;  // apart from the arguments that the loop indexes
    __syncthreads();
    finish<EPI, PL>(fin, acc, (f32x4*)&lds[0][0] + wave * finish_quads(MB, NB), m0 + wr * 16 * MB,
                    n0 + wc * 16 * (DUAL ? NB / 2 : NB), split);
}

// fp32 operands as they lie, where they are too few products to pay for packing: a tile of 64 rows x 128 columns
// (kSwiGLU: 64 columns of h), four wavefronts in a 2 x 2 grid of 32 rows x 64 columns, chunks of 32 contraction
// elements in two stages. A fragment becomes three bf16 terms in registers (44 instructions of the VALU beside the 6
// MFMAs that each pair of fragments takes), the small term products and the large ones have sums of their own. Three
// work-groups share a CU, so one's conversion runs beside another's products and loads.
template <int EPI, bool BMC>
__global__ __launch_bounds__(256) void swiglu_f32_kernel(TileArgs p) {
    constexpr int MB = 2, NB = 4, TM = 64, TN = 128;
    constexpr bool DUAL = EPI == kSwiGLU;
    typedef Stage<false, TM, true> SA;
    typedef Stage<BMC, TN, true> SB;
    __shared__ __attribute__((aligned(1024))) unsigned char lds[2][SA::BYTES + SB::BYTES];
    static_assert(4 * 16 * finish_quads(MB, NB) <= 2 * (SA::BYTES + SB::BYTES), "the sums in LDS");
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wr = wave >> 1, wc = wave & 1;
    const int per = (p.total + 7) / 8;
    const int local = blockIdx.x / 8;
    const int item = (blockIdx.x % 8) * per + local;
    if (local >= per || item >= p.total) return;
    const int split = item / p.tiles, tile = item - split * p.tiles;
    const int band = tile / (kBand * p.ncb), in = tile - band * kBand * p.ncb;
    const int height = min(kBand, (p.M + TM - 1) / TM - band * kBand);
    const int m0 = (band * kBand + in % height) * TM;
    const int n0 = (in / height) * (DUAL ? TN / 2 : TN);
    SA sa;
    SB sb;
    sa.init(wave, lane, m0, p.M, p.lda);
    sb.init(DUAL ? wave & 1 : wave, lane, n0, p.N, p.ldb);  // kSwiGLU: as in swiglu_tile_kernel
    const long long a_tile = (long long)m0 * p.lda * 4, b_tile = BMC ? 0 : (long long)n0 * p.ldb * 4;
    const unsigned lds0 = (unsigned)(size_t)(lds_ptr_t)&lds[0][0];
    const int cps = (max(p.ka, p.kb) + SA::CHUNK - 1) / SA::CHUNK;
    const int first = split * p.split_chunks;
    const int chunks = min(p.split_chunks, cps * p.nseg - first);
    int seg = first / cps, c0 = first - seg * cps;  // segment and chunk of it to load next
    auto load = [&](int st) {
        const char* pa = p.a[seg] + a_tile + c0 * sa.step;
        const char* pb = (DUAL && wave >= 2 ? p.b1[seg] : p.b[seg]) + b_tile + c0 * sb.step;
        const unsigned base = lds0 + st * (SA::BYTES + SB::BYTES);
        const int left = SA::CHUNK * c0;
#pragma unroll
        for (int j = 0; j < SA::LOADS; ++j) sa.load(wave, wave, lane, j, pa, p.ka - left, base);
#pragma unroll
        for (int j = 0; j < SB::LOADS; ++j)
            sb.load(wave, DUAL ? wave & 1 : wave, lane, j, pb, p.kb - left, base + SA::BYTES);
        if (++c0 == cps) c0 = 0, ++seg;
    };
    Reader32<false, TM> ra;
    Reader32<BMC, TN> rb;
    ra.init(lane, wr * 16 * MB);
    rb.init(lane, DUAL ? wc * 8 * NB : wc * 16 * NB);
    f32x4 large[MB][NB], small[MB][NB];
#pragma unroll
    for (int i = 0; i < MB; ++i)
#pragma unroll
        for (int j = 0; j < NB; ++j) large[i][j] = small[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (chunks > 0) load(0);
    for (int c = 0; c < chunks; ++c) {
        const int st = c & 1;
        // this wavefront's loads of chunk c have landed and its reads of chunk c - 1 are over, and after the barrier
        // everybody's
        __builtin_amdgcn_s_waitcnt(all_done());
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        if (c + 1 < chunks) load(st ^ 1);
        bf16x8 a[MB][3];
#pragma unroll
        for (int i = 0; i < MB; ++i) {
            float v[8];
            ra.read(&lds[st][0], i, v);
            ra.terms(v, a[i]);
        }
#pragma unroll
        for (int j = 0; j < NB; ++j) {
            float v[8];
            bf16x8 b[3];
            rb.read(&lds[st][SA::BYTES], DUAL && j >= NB / 2 ? j - NB / 2 + NB : j, v);
            rb.terms(v, b);
#pragma unroll
            for (int i = 0; i < MB; ++i) {
#pragma unroll
                for (int t = 0; t < 5; ++t)
                    small[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b[kTermB[t]], a[i][kTermA[t]], small[i][j], 0, 0, 0);
                large[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b[0], a[i][0], large[i][j], 0, 0, 0);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < MB; ++i)
#pragma unroll
        for (int j = 0; j < NB; ++j) large[i][j] = large[i][j] + small[i][j];
    const Finish fin = p;
    __syncthreads();
    finish<EPI, kFp32>(fin, large, (f32x4*)&lds[0][0] + wave * finish_quads(MB, NB), m0 + wr * 16 * MB,
                       n0 + wc * 16 * (DUAL ? NB / 2 : NB), split);
}

// ------------------------------------------------------------------ few rows
// Up to 64 rows of the forward pass: bound by the stream of the weights, which are read as they lie. A work-group of
// eight wavefronts owns 16 columns (kSwiGLU: gate and up), the wavefronts deal out the contraction in spans of SPAN
// steps and add their sums in LDS, in order. Lane 16 g + r reads 16 bytes of weight row r and of row r of x, so a
// step is 32 (fp32: 16) elements and a span of four 256 consecutive bytes of every weight row; any alignment. fp32 runs
// on the fp32 MFMAs: four a step, each on one element of the lanes' four.
struct FewArgs {
    const void* x;
    int N, K, ldx;
    const void* w[2];       // [O][K]
    int O;
    void* out;              // kOut: [N][O]; kSwiGLU: h [N][ldh], in x's type
    float* gu;              // kSwiGLU: [2][N][ldh] or none
    int ldh;
};

struct __attribute__((packed, aligned(2))) Any16 {
    unsigned v[4];
};
template <bool F32>
struct Piece {  // 16 bytes of a row
    union {
        uint4 u;
        bf16x8 b;
        float f[4];
        unsigned short s[8];
    };
    static constexpr int E = F32 ? 4 : 8, STEP = 4 * E;
    __device__ __forceinline__ void load(const void* p, size_t at) {
        const Any16 a = *(const Any16*)((const char*)p + at * (F32 ? 4 : 2));
        u = make_uint4(a.v[0], a.v[1], a.v[2], a.v[3]);
    }
    // the first `left` elements, zeros behind them
    __device__ __forceinline__ void load_end(const void* p, size_t at, int left) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
            if (F32) f[e] = e < left ? ((const float*)p)[at + e] : 0.0f;
            else s[e] = e < left ? ((const unsigned short*)p)[at + e] : 0;
        }
    }
};
template <bool F32>
__device__ __forceinline__ f32x4 few_mfma(const Piece<F32>& a, const Piece<F32>& b, f32x4 c) {
    if constexpr (F32) {
#pragma unroll
        for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.f[e], b.f[e], c, 0, 0, 0);
        return c;
    } else {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.b, b.b, c, 0, 0, 0);
    }
}

template <int EPI, bool F32, int MR>
__global__ __launch_bounds__(512) void swiglu_few_kernel(FewArgs p) {
    constexpr int NM = EPI == kSwiGLU ? 2 : 1;
    constexpr int SPAN = F32 && MR == 4 ? 2 : 4;  // as many as registers hold
    typedef Piece<F32> P;
    __shared__ f32x4 part[8][NM * MR][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = lane >> 4, r = lane & 15;
    // rows past the last one read it again: their sums are not stored
    const size_t wrow = (size_t)min((int)blockIdx.x * 16 + r, p.O - 1) * p.K;
    size_t xrow[MR];
#pragma unroll
    for (int i = 0; i < MR; ++i) xrow[i] = (size_t)min(16 * i + r, p.N - 1) * p.ldx;
    f32x4 acc[NM][MR];
#pragma unroll
    for (int m = 0; m < NM; ++m)
#pragma unroll
        for (int i = 0; i < MR; ++i) acc[m][i] = f32x4{0.f, 0.f, 0.f, 0.f};
    const int steps = p.K / P::STEP, spans = (steps + SPAN - 1) / SPAN;
    for (int sp = wave; sp < spans; sp += 8) {
        const int s0 = sp * SPAN;
        P w[NM][SPAN], x[MR][SPAN];
        if (s0 + SPAN <= steps) {
#pragma unroll
            for (int s = 0; s < SPAN; ++s) {
                const size_t k = (size_t)(s0 + s) * P::STEP + g * P::E;
#pragma unroll
                for (int m = 0; m < NM; ++m) w[m][s].load(p.w[m], wrow + k);
#pragma unroll
                for (int i = 0; i < MR; ++i) x[i][s].load(p.x, xrow[i] + k);
            }
            __builtin_amdgcn_sched_barrier(0);  // all of the span's loads in flight
#pragma unroll
            for (int s = 0; s < SPAN; ++s)
#pragma unroll
                for (int m = 0; m < NM; ++m)
#pragma unroll
                    for (int i = 0; i < MR; ++i) acc[m][i] = few_mfma<F32>(w[m][s], x[i][s], acc[m][i]);
        } else {
            for (int s = s0; s < steps; ++s) {
                const size_t k = (size_t)s * P::STEP + g * P::E;
#pragma unroll
                for (int m = 0; m < NM; ++m) w[m][0].load(p.w[m], wrow + k);
#pragma unroll
                for (int i = 0; i < MR; ++i) x[i][0].load(p.x, xrow[i] + k);
#pragma unroll
                for (int m = 0; m < NM; ++m)
#pragma unroll
                    for (int i = 0; i < MR; ++i) acc[m][i] = few_mfma<F32>(w[m][0], x[i][0], acc[m][i]);
            }
        }
    }
    if (steps * P::STEP < p.K && wave == spans % 8) {
        // the rest of the rows, less than a step
        const size_t k = (size_t)steps * P::STEP + g * P::E;
        const int left = p.K - (int)k;
        P w[NM], x[MR];
#pragma unroll
        for (int m = 0; m < NM; ++m) w[m].load_end(p.w[m], wrow + k, left);
#pragma unroll
        for (int i = 0; i < MR; ++i) x[i].load_end(p.x, xrow[i] + k, left);
#pragma unroll
        for (int m = 0; m < NM; ++m)
#pragma unroll
            for (int i = 0; i < MR; ++i) acc[m][i] = few_mfma<F32>(w[m], x[i], acc[m][i]);
    }
#pragma unroll
    for (int m = 0; m < NM; ++m)
#pragma unroll
        for (int i = 0; i < MR; ++i) part[wave][m * MR + i][lane] = acc[m][i];
    __syncthreads();
    if (wave >= MR) return;  // wavefront i finishes rows 16 i .. + 15
    f32x4 v[NM];
#pragma unroll
    for (int m = 0; m < NM; ++m) {
        v[m] = part[0][m * MR + wave][lane];
#pragma unroll
        for (int k = 1; k < 8; ++k) v[m] = v[m] + part[k][m * MR + wave][lane];
    }
    const int n = 16 * wave + r, o = blockIdx.x * 16 + 4 * g;
    if (n >= p.N) return;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if constexpr (EPI == kSwiGLU) {
            const size_t at = (size_t)n * p.ldh + o + e;
            const bool in = o + e < p.O;
            if (o + e >= p.ldh) continue;
            // behind the last column: zeros, as the tiles write them
            const float a = in ? v[0][e] : 0.0f, u = in ? v[NM - 1][e] : 0.0f, h = silu_fast(a) * u;
            if (p.gu != nullptr) p.gu[at] = a, p.gu[(size_t)p.N * p.ldh + at] = u;
            if (F32) ((float*)p.out)[at] = h;
            else ((unsigned short*)p.out)[at] = f32_to_bf16_rne(h);
        } else if (o + e < p.O) {
            const size_t at = (size_t)n * p.O + o + e;
            if (F32) ((float*)p.out)[at] = v[0][e];
            else ((unsigned short*)p.out)[at] = f32_to_bf16_rne(v[0][e]);
        }
    }
}

// Sums of the splits, in order, and what becomes of them.
template <int EPI, int PL>
__global__ __launch_bounds__(256) void swiglu_sum_kernel(Finish p, int splits) {
    constexpr int NM = EPI == kSwiGLU ? 2 : 1;
    const int per = p.ldp / 4;
    const long long total = (long long)p.M * per, plane = (long long)p.M * p.ldp;
    for (long long e = (long long)blockIdx.x * 256 + threadIdx.x; e < total; e += (long long)gridDim.x * 256) {
        const int m = (int)(e / per), n = (int)(e - (long long)m * per) * 4;
        const float* at = p.part + (long long)m * p.ldp + n;
        f32x4 v[NM];
#pragma unroll
        for (int k = 0; k < NM; ++k) v[k] = *(const f32x4*)(at + k * plane);
        for (int s = 1; s < splits; ++s)
#pragma unroll
            for (int k = 0; k < NM; ++k) v[k] = v[k] + *(const f32x4*)(at + (s * NM + k) * plane);
        if constexpr (EPI == kOut) finish_out<PL>(p, m, n, v[0]);
        else if constexpr (EPI == kGrad) finish_grad<PL>(p, m, n, v[0]);
        else finish_swiglu<PL>(p, m, n, v[0], v[NM - 1]);
    }
}

// Tensors of rows of any width to planes of bf16 terms whose rows are a multiple of 8 wide, zeros behind the last
// column: up to five tensors a launch, 8 values a thread.
struct PackArgs {
    int n;
    long long pieces;  // of all tensors
    struct {
        const void* src;
        unsigned short* dst;
        long long end, plane;  // pieces up to this tensor's last one, elements between planes
        int cols, ld;
    } t[5];
};
template <bool F32>
__global__ __launch_bounds__(256) void swiglu_pack_kernel(PackArgs a) {
    for (long long e = (long long)blockIdx.x * 256 + threadIdx.x; e < a.pieces; e += (long long)gridDim.x * 256) {
        int k = 0;
        while (e >= a.t[k].end) ++k;
        const auto& t = a.t[k];
        const long long i = e - (k > 0 ? a.t[k - 1].end : 0);
        const int per = t.ld / 8;
        const long long row = i / per;
        const int c = (int)(i - row * per) * 8;
        const size_t at = (size_t)row * t.cols + c;
        Piece<F32> v[F32 ? 2 : 1];
#pragma unroll
        for (int q = 0; q < (F32 ? 2 : 1); ++q) {
            if (c + 8 <= t.cols) v[q].load(t.src, at + 4 * q);
            else v[q].load_end(t.src, at + 4 * q, t.cols - c - 4 * q);
        }
        unsigned short* dst = t.dst + row * t.ld + c;
        if constexpr (F32) {
            // the terms of eight values, a plane's 16 bytes at a time
            float r[8];
#pragma unroll
            for (int q = 0; q < 8; ++q) r[q] = v[q / 4].f[q % 4];
#pragma unroll
            for (int p = 0; p < 3; ++p) {
                unsigned d[4];
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    d[q] = pack_bf16(r[2 * q], r[2 * q + 1]);
                    r[2 * q] -= bf16_to_f32((unsigned short)(d[q] & 0xffff));
                    r[2 * q + 1] -= bf16_to_f32((unsigned short)(d[q] >> 16));
                }
                *(uint4*)(dst + p * t.plane) = make_uint4(d[0], d[1], d[2], d[3]);
            }
        } else {
            *(uint4*)dst = v[0].u;
        }
    }
}

// ------------------------------------------------------------------ host
inline int up8(int v) { return (v + 7) / 8 * 8; }
inline int up4(int v) { return (v + 3) / 4 * 4; }

// An operand as planes of bf16 terms.
struct Operand {
    const char* p;
    int ld;
    long long plane;  // bytes
};

// Parts of a workspace, and the tensors to be packed into them; dry: sizes only, nothing is launched.
struct Carve {
    char* base;
    bool dry;
    int act;
    size_t used = 0;  // where it starts in the workspace, and what is taken
    PackArgs packs{};
    char* take(size_t bytes) {
        char* r = dry ? nullptr : base + used;
        used += align_up(bytes, 256);
        return r;
    }
    // rows x cols as an operand: itself, where a row is whole 16-byte pieces of bf16
    Operand operand(const void* t, long long rows, int cols) {
        if (act == YVMOE_ACT_BF16 && cols % 8 == 0) return {(const char*)t, cols, 0};
        const int ld = up8(cols);
        char* dst = take((size_t)rows * ld * 2 * (act == YVMOE_ACT_F32 ? 3 : 1));
        const long long pieces = rows * (ld / 8);
        packs.pieces += pieces;
        packs.t[packs.n++] = {t, (unsigned short*)dst, packs.pieces, rows * ld, cols, ld};
        return {dst, ld, rows * ld * 2};
    }
    void pack(hipStream_t st) const {
        if (packs.pieces == 0) return;
        const unsigned blocks = (unsigned)std::min<long long>((packs.pieces + 255) / 256, 1 << 16);
        if (act == YVMOE_ACT_F32) swiglu_pack_kernel<true><<<blocks, 256, 0, st>>>(packs);
        else swiglu_pack_kernel<false><<<blocks, 256, 0, st>>>(packs);
    }
};

// Adds the n = 1 or 6 operand pairs of A · Bᵀ (with b1: gate and up) to a launch.
void add_product(TileArgs& p, int n, const Operand& a, const Operand& b, const Operand* b1 = nullptr) {
    for (int t = 0; t < n; ++t) {
        const int ta = n == 1 ? 0 : kTermA[t], tb = n == 1 ? 0 : kTermB[t];
        p.a[p.nseg] = a.p + ta * a.plane;
        p.b[p.nseg] = b.p + tb * b.plane;
        if (b1 != nullptr) p.b1[t] = b1->p + tb * b1->plane;
        ++p.nseg;
    }
    p.lda = a.ld;
    p.ldb = b.ld;
}

// Tile and number of splits of the contraction for M x N outputs (kSwiGLU: N twice the columns of h) of `chunks`
// chunks: the least of an estimate. A CU's work-group takes `alone` us a chunk when it runs by itself and `shared` us of
// the CU's time beside others (measured: 256 1.45 and 1.79 under full load, 128 0.84 and 0.42 to 0.60, 64 0.63 and
// 0.28 to 0.34); splits cost a launch and their sums' traffic. direct: the fp32 form, 64 x 128 and chunks of 32.
struct Plan {
    int tile, splits, len;  // len: chunks of a split
};
Plan plan_of(int M, int N, int chunks, bool direct) {
    static const struct { int rows, cols; float alone, shared; } kinds[4] = {
        {256, 256, 1.5f, 1.7f}, {128, 128, 0.84f, 0.58f}, {64, 64, 0.63f, 0.3f}, {64, 128, 0.9f, 0.5f}};
    Plan best{256, 1, std::max(chunks, 1)};
    float least = 1e30f;
    for (int i = direct ? 3 : 0; i < (direct ? 4 : 3); ++i) {
        const auto& k = kinds[i];
        const long long tiles = (long long)((M + k.rows - 1) / k.rows) * ((N + k.cols - 1) / k.cols);
        for (int s = 1; s <= 16 && (s == 1 || chunks / s >= 4); ++s) {
            const float per_cu = (float)((tiles * s + 255) / 256);
            const int len = (chunks + s - 1) / s;
            float us = std::max(k.alone, per_cu * k.shared) * len;
            if (s > 1) us += 4.0f + (float)s * M * N * 8.0f / 4e6f;
            if (us < least) least = us, best = {k.rows, ceil_div(chunks, std::max(len, 1)), std::max(len, 1)};
        }
    }
    best.splits = std::max(best.splits, 1);
    return best;
}

inline int chunks_of(int k, int nseg, bool direct) { return ceil_div(k, direct ? 32 : kChunk) * nseg; }
// Bytes of the partial sums of an M x N product (N as in plan_of).
size_t part_bytes(int M, int N, int k, int nseg, bool direct) {
    const Plan q = plan_of(M, N, chunks_of(k, nseg, direct), direct);
    return q.splits > 1 ? (size_t)q.splits * M * (N + 16) * 4 : 0;
}

template <int EPI, int PL, bool AMC, bool BMC, int MB, int NB>
void tile_grid(TileArgs p, int splits, hipStream_t st) {
    const int cols = EPI == kSwiGLU ? 16 * NB : 32 * NB;
    p.ncb = ceil_div(p.N, cols);
    p.tiles = ceil_div(p.M, 32 * MB) * p.ncb;
    p.total = p.tiles * splits;
    swiglu_tile_kernel<EPI, PL, AMC, BMC, MB, NB><<<(unsigned)(ceil_div(p.total, 8) * 8), 256, 0, st>>>(p);
}

template <int EPI, int PL, bool AMC, bool BMC>
void tiles_of(const TileArgs& p, const Plan& q, hipStream_t st) {
    if (q.tile == 256) tile_grid<EPI, PL, AMC, BMC, 8, 8>(p, q.splits, st);
    else if (q.tile == 128) tile_grid<EPI, PL, AMC, BMC, 4, 4>(p, q.splits, st);
    else tile_grid<EPI, PL, AMC, BMC, 2, 2>(p, q.splits, st);
}

// PL: kSwiGLU, kGrad, how h and d are stored; kOut with kFp32: the fp32 form on operands as they lie.
template <int EPI, int PL, bool AMC, bool BMC>
void tile_launch(TileArgs p, float* part, hipStream_t st) {
    if (p.M <= 0 || p.N <= 0) return;
    constexpr bool DIRECT = PL == kFp32;
    const Plan q = plan_of(p.M, EPI == kSwiGLU ? 2 * p.N : p.N, chunks_of(std::max(p.ka, p.kb), p.nseg, DIRECT), DIRECT);
    p.split_chunks = q.len;
    if (q.splits > 1) {
        p.part = part;
        p.ldp = EPI == kOut ? up4(p.N) : p.ldh;
    }
    if constexpr (DIRECT) {
        p.ncb = ceil_div(p.N, EPI == kSwiGLU ? 64 : 128);
        p.tiles = ceil_div(p.M, 64) * p.ncb;
        p.total = p.tiles * q.splits;
        swiglu_f32_kernel<EPI, BMC><<<(unsigned)(ceil_div(p.total, 8) * 8), 256, 0, st>>>(p);
    } else if constexpr (EPI == kSwiGLU && PL == kOne) {
        if (p.gu == nullptr && q.splits == 1) tiles_of<EPI, kAlone, AMC, BMC>(p, q, st);
        else tiles_of<EPI, PL, AMC, BMC>(p, q, st);
    } else {
        tiles_of<EPI, PL, AMC, BMC>(p, q, st);
    }
    if (q.splits > 1) {
        const long long quads = (long long)p.M * (p.ldp / 4);
        swiglu_sum_kernel<EPI, PL><<<(unsigned)std::min<long long>((quads + 255) / 256, 8192), 256, 0, st>>>(p, q.splits);
    }
}

// Whether fp32 operands can go into the products as they lie: rows of whole 16-byte pieces.
inline bool direct_f32(int act, int H, int F) { return act == YVMOE_ACT_F32 && H % 4 == 0 && F % 4 == 0; }
// And whether they do: packing reads and writes 10 bytes for each of (N + 3 F) H values, at 3.5 TB/s, and takes the
// 36 N H F operations of the term products from about 1.0 to 1.3 PFLOP/s (4096 x 11264, forward: 800 rows direct
// 1340 us, 1200 packed 1856).
inline bool goes_direct(int act, int N, int H, int F) {
    return direct_f32(act, H, F) && (double)N * F < 344.0 * ((double)N + 3.0 * F);
}

// Each block of 16 columns reads all rows from L2: with many blocks, tiles take over from 33 rows on (4096 x 11264, bf16,
// forward: 33 rows 101 us against about 95, 64 rows 137 against 98; 5120 x 1536: 64 rows 47 against 56).
// fp32, where it has tiles without packing, from 33 on (1024 x 2816: 33 rows 57 us against 33, 17 rows 26 against 33), and
// on large weights from 17 (4096 x 11264: 17 rows 179 us against 145).
inline bool few_rows(int act, int N, int H, int F) {
    if (direct_f32(act, H, F)) return N <= ((long long)H * F >= 1 << 22 ? 16 : 32);
    return N <= (F >= 8192 ? 32 : 64);
}

template <int EPI, bool F32>
void few_launch(const FewArgs& p, hipStream_t st) {
    const unsigned blocks = (unsigned)ceil_div(p.O, 16);
    if (p.N <= 16) swiglu_few_kernel<EPI, F32, 1><<<blocks, 512, 0, st>>>(p);
    else if (p.N <= 32) swiglu_few_kernel<EPI, F32, 2><<<blocks, 512, 0, st>>>(p);
    else swiglu_few_kernel<EPI, F32, 4><<<blocks, 512, 0, st>>>(p);
}

}  // namespace

size_t swiglu_saved_bytes(int N, int F) { return (size_t)2 * N * up8(F) * 4; }

// With bytes nothing is launched: *bytes is the size of the workspace.
int swiglu_forward_launch(const void* x, int act, int N, const yvmoe_swiglu_weights* w, float* saved, void* out,
                          char* ws, size_t* bytes, hipStream_t st) {
    const int H = w->hidden, F = w->ffn, F8 = up8(F), planes = act == YVMOE_ACT_F32 ? 3 : 1;
    Carve c{ws, bytes != nullptr, act};
    if (few_rows(act, N, H, F)) {
        const bool f32 = act == YVMOE_ACT_F32;
        void* h = c.take((size_t)N * F8 * (f32 ? 4 : 2));
        if (bytes != nullptr) *bytes = c.used;
        if (c.dry || N == 0) return YVMOE_OK;
        const FewArgs p{x, N, H, H, {w->w_gate, w->w_up}, F, h, saved, F8};
        const FewArgs q{h, N, F, F8, {w->w_down, nullptr}, H, out, nullptr, 0};
        if (f32) few_launch<kSwiGLU, true>(p, st), few_launch<kOut, true>(q, st);
        else few_launch<kSwiGLU, false>(p, st), few_launch<kOut, false>(q, st);
        YV_LAUNCH_CHECK("swiglu_forward");
        return YVMOE_OK;
    }
    const bool direct = goes_direct(act, N, H, F);
    const long long plane = (long long)N * F8;
    Operand ox{(const char*)x, H, 0}, og{(const char*)w->w_gate, H, 0}, ou{(const char*)w->w_up, H, 0},
        od{(const char*)w->w_down, F, 0};
    if (!direct) {
        ox = c.operand(x, N, H);
        og = c.operand(w->w_gate, F, H);
        ou = c.operand(w->w_up, F, H);
        od = c.operand(w->w_down, H, F);
    }
    const int terms = act == YVMOE_ACT_F32 && !direct ? 6 : 1;
    char* h = c.take((size_t)plane * (direct ? 4 : 2 * planes));
    float* part = (float*)c.take(std::max(part_bytes(N, 2 * F, H, terms, direct), part_bytes(N, H, F8, terms, direct)));
    if (bytes != nullptr) *bytes = c.used;
    if (c.dry || N == 0) return YVMOE_OK;
    c.pack(st);
    TileArgs p{};
    p.M = N;
    p.N = F;
    p.ka = p.kb = ox.ld;
    add_product(p, terms, ox, og, &ou);
    p.h = h;
    p.plane_h = plane;
    p.gu = saved;
    p.ldh = F8;
    TileArgs q{};
    q.M = N;
    q.N = H;
    q.ka = F8;
    q.kb = direct ? F : F8;
    add_product(q, terms, Operand{h, F8, plane * 2}, od);
    q.out = out;
    q.ldo = H;
    q.split = q.split_at = N;
    q.f32 = act == YVMOE_ACT_F32;
    if (direct) tile_launch<kSwiGLU, kFp32, false, false>(p, part, st);
    else if (planes == 3) tile_launch<kSwiGLU, kThree, false, false>(p, part, st);
    else tile_launch<kSwiGLU, kOne, false, false>(p, part, st);
    if (direct) tile_launch<kOut, kFp32, false, false>(q, part, st);
    else tile_launch<kOut, kOne, false, false>(q, part, st);
    YV_LAUNCH_CHECK("swiglu_forward");
    return YVMOE_OK;
}

int swiglu_backward_launch(const void* dy, const void* x, const float* saved, int act, int N,
                           const yvmoe_swiglu_weights* w, void* dx, void* dwg, void* dwu, void* dwd, char* ws,
                           size_t* bytes, hipStream_t st) {
    const int H = w->hidden, F = w->ffn, F8 = up8(F);
    const int f32 = act == YVMOE_ACT_F32, planes = f32 ? 3 : 1, terms = f32 ? 6 : 1;
    const bool direct = goes_direct(act, N, H, F);
    Carve c{ws, bytes != nullptr, act};
    const long long plane = (long long)N * F8;
    // dy and x as operands of the weights' gradients, weights and dy of dh and dx
    const bool wgrad = c.dry || dwg != nullptr || dwu != nullptr || dwd != nullptr;
    Operand ody{(const char*)dy, H, 0}, ox{(const char*)x, H, 0}, og{(const char*)w->w_gate, H, 0},
        ou{(const char*)w->w_up, H, 0}, od{(const char*)w->w_down, F, 0};
    Operand pdy = ody, oh{}, odd{};
    if (!direct || wgrad) pdy = c.operand(dy, N, H);
    if (!direct) {
        ody = pdy;
        od = c.operand(w->w_down, H, F);
        if (c.dry || dx != nullptr) {
            og = c.operand(w->w_gate, F, H);
            ou = c.operand(w->w_up, F, H);
        }
    }
    if (c.dry || dwg != nullptr || dwu != nullptr) ox = c.operand(x, N, H);
    // h, dg and du: planes of terms, or fp32 first and packed for the weights' gradients
    char* h = c.take((size_t)plane * (direct ? 4 : 2 * planes));
    char* d = c.take((size_t)plane * 2 * (direct ? 4 : 2 * planes));
    oh = Operand{h, F8, plane * 2};
    odd = Operand{d, 2 * F8, plane * 4};
    Carve late{c.base, c.dry, act, c.used};
    if (direct && wgrad) {
        oh = late.operand(h, N, F8);
        odd = late.operand(d, N, 2 * F8);
        c.used = late.used;
    }
    float* part = (float*)c.take(std::max({part_bytes(N, F, H, direct ? 1 : terms, direct),
                                           part_bytes(N, H, F8, direct ? 2 : 2 * terms, direct),
                                           part_bytes(F8 + F, H, N, terms, false), part_bytes(F, H, N, terms, false),
                                           part_bytes(H, F, N, terms, false)}));
    if (bytes != nullptr) *bytes = c.used;
    if (c.dry) return YVMOE_OK;
    c.pack(st);
    TileArgs p{};
    p.M = N;
    p.N = F;
    p.ka = ody.ld;
    p.kb = H;
    add_product(p, direct ? 1 : terms, ody, od);
    p.h = h;
    p.plane_h = plane;
    p.d = d;
    p.plane_d = plane * 2;
    p.gu = const_cast<float*>(saved);
    p.ldh = F8;
    if (direct) tile_launch<kGrad, kFp32, false, true>(p, part, st);
    else if (planes == 3) tile_launch<kGrad, kThree, false, true>(p, part, st);
    else tile_launch<kGrad, kOne, false, true>(p, part, st);
    if (dx != nullptr) {
        TileArgs q{};
        q.M = N;
        q.N = H;
        q.ka = F8;
        q.kb = F;
        const int e = direct ? 4 : 2;
        const Operand dg{d, 2 * F8, plane * 4}, du{d + (size_t)F8 * e, 2 * F8, plane * 4};
        add_product(q, direct ? 1 : terms, dg, og);
        add_product(q, direct ? 1 : terms, du, ou);
        if (terms > 1 && !direct) {  // both matrices' smallest terms first
            const TileArgs in = q;
            for (int t = 0; t < 12; ++t) {
                q.a[t] = in.a[t / 2 + 6 * (t & 1)];
                q.b[t] = in.b[t / 2 + 6 * (t & 1)];
            }
        }
        q.out = dx;
        q.ldo = H;
        q.split = q.split_at = N;
        q.f32 = f32;
        if (direct) tile_launch<kOut, kFp32, false, true>(q, part, st);
        else tile_launch<kOut, kOne, false, true>(q, part, st);
    }
    late.pack(st);
    if (dwg != nullptr || dwu != nullptr) {
        const bool both = dwg != nullptr && dwu != nullptr;
        TileArgs q{};
        q.M = both ? F8 + F : F;
        q.N = H;
        q.ka = q.kb = N;
        add_product(q, terms, dwg != nullptr ? odd : Operand{odd.p + 2 * (size_t)F8, odd.ld, odd.plane}, ox);
        q.out = dwg != nullptr ? dwg : dwu;
        q.out1 = dwu;
        q.ldo = H;
        q.split = F;
        q.split_at = both ? F8 : F;
        q.f32 = f32;
        tile_launch<kOut, kFar, true, true>(q, part, st);
    }
    if (dwd != nullptr) {
        TileArgs q{};
        q.M = H;
        q.N = F;
        q.ka = q.kb = N;
        add_product(q, terms, pdy, oh);
        q.out = dwd;
        q.ldo = F;
        q.split = q.split_at = H;
        q.f32 = f32;
        tile_launch<kOut, kFar, true, true>(q, part, st);
    }
    YV_LAUNCH_CHECK("swiglu_backward");
    return YVMOE_OK;
}

}  // namespace yvmoe
