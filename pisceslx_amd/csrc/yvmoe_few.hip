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
//    slots in LDS; cheaper than another launch), then the gate/up products of the routed experts as
//    (tile, 16 columns of F) items, and once all of them are there each work-group takes 16
//    columns of H of *all* tiles, so that the weighted sum, the shared mixture and the skip residual
//    end in its LDS: no expert output leaves the chip. Where H gives too few work-groups, up to eight
//    share 16 columns, and the last one to finish adds up their sums, in their order.
//
// Between the two halves of 2 work-groups wait for each other's h. A work-group's first five items are
// its own, and it marks them when they are done; the rest are handed out by a counter, which evens out
// the work-groups, and those done are counted. Items of the second kind are held by work-groups that
// run and wait for nothing; those of the first kind are computed by a work-group that has waited long
// for their mark (the same bits, so doing them twice is harmless). So the wait ends whichever part of
// the grid is resident, also beside other kernels that wait. What work-groups hand to each other is
// written through and read past the caches (sc1): an acquire in every wavefront would invalidate the L2s each
// time, which cost 30 us in a form of 4,096 wavefronts. A wait that nothing ends is given up after seconds, and
// the columns of that work-group are NaN.
//
// Rounding: weights enter exactly (codes as bf16, scales on the fp32 sums), h as two bf16 terms (16 bits) for
// the second product's MFMAs; the outputs are rounded once at the end.
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "yvmoe_frag.h"
#include "yvmoe_internal.h"
#include "yvmoe_topk.h"

namespace yvmoe {
namespace {

// k-steps per chunk and chunks held for two matrices and for one, without and with activations in LDS. As
// many bytes in flight as the 168 registers of nine wavefronts hold without spilling in a loop (which cost
// bf16 a half); longer chunks make the last one of a short K emptier (fp32 with two k-steps: 56 -> 70 us at one
// token, 1024 -> 2816; bf16 with two: 2 to 5 % more from 1088 to 4096). More and thinner wavefronts do not
// help: with 11 one int8 token takes 48 us, with 15 61, with 8 44.
struct Depth {
    int u2, r2, u1, r1, lu2, lr2, lu1, lr1;
    constexpr int unit(int nm, bool lds) const { return nm == 2 ? (lds ? lu2 : u2) : (lds ? lu1 : u1); }
    constexpr int ring(int nm, bool lds) const { return nm == 2 ? (lds ? lr2 : r2) : (lds ? lr1 : r1); }
};

constexpr int kFewSlots = kFewTokens * YVMOE_MAX_TOPK;
constexpr int kFewTiles = kFewSlots + 2 * YVMOE_MAX_SHARED;
// Wavefronts that stream weights; one more sums their products, stores h, takes items and waits, so that
// the streams never wait for a store or an atomic (which answer after microseconds, and in the order
// of the loads round them).
constexpr int kWaves = 8, kThreads = 64 * kWaves, kAllThreads = kThreads + 64;
constexpr int kYRows = 512;            // rows of partial expert outputs that a work-group holds
constexpr int kGrid = kFewGrid;  // most work-groups of the second kernel: one per CU
// Looks at a signal, between half and one microsecond each, before helping, and rounds of them after which a wait
// with nothing to help with is given up (seconds).
constexpr int kPatience = 1024, kMostRounds = 1 << 11;
enum Waited { WAIT_DONE = -1, WAIT_GIVEN_UP = -2 };
// What a SIG_GO word holds: GO_DONE once all is done, before that 0 or how a test wants the wait.
enum Go { GO_DONE = 1, GO_ONE_LOOK = 2, GO_NO_WAIT = 4 };
std::atomic<int> wait_mode{0};

constexpr int kOwnItems = 5;  // gate/up items that a work-group takes without asking (GateUpItems)
constexpr int kMarkWords = kGrid / 32, kGoLines = 32;
// Words that work-groups signal with, each on a line of its own: an address serves some 50 accesses a
// microsecond, and all work-groups come at about the same time.
enum Signal {
    SIG_MARKS = 0,               // kMarkWords words of 32 bits: the work-group's own items are done
    SIG_FINISHED = kMarkWords,   // items handed out that are done
    SIG_ROOT,                    // of the above, how many are complete
    SIG_TICKET,                  // items handed out
    SIG_GO,                      // kGoLines words: all is done (Go)
    SIG_COUNT = SIG_GO + kGoLines
};
constexpr int kSignalBytes = SIG_COUNT * 128;
static_assert(kSignalBytes <= kFewSignalBytes, "workspace layout");

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
    const void* xo; // x, for int4 in its order of columns
    void* h;        // [terms][N k + S N][F], routed rows by expert, then the shared experts' tokens
    unsigned* signals;  // Signal words, 32 apart
    int hparts;       // work-groups per 16 columns of H
    int parts;        // parts of a work-group's share of K
    int* hcount;      // [H / 16]: those of them that are done
    float* hsum;      // [hparts][2][N][H]: their sums of the routed and of the shared experts
    int wait_mode;    // what the first kernel puts into the SIG_GO words
};

// ---------------------------------------------------------------- weights and activations
// A wavefront multiplies 16 activation rows (the first MFMA operand) with 16 rows of a weight matrix
// over 64-wide k-steps. Lane l = 16 g + r holds columns 16 g .. 16 g + 15 of activation row r and of
// weight row r; the accumulator holds activation rows 4 g + i of weight row r, so that a row's scale
// stays in the lanes that hold its codes.
//
// Raw: a k-step's weights as stored. Act: a k-step's activations. DEPTH: k-steps per chunk, and
// chunks that the registers hold, all but one of them in flight.
// GROUPED: the scale belongs to a row (int4) or 128 rows (fp8) and 128 columns, that is two k-steps.
template <int WF>
struct Wt;

// h in two bf16 terms (16 bits), so that its rounding does not add to the outputs' own (with one term errors
// against 64 bits are 1.4 times as large): both are rows of one operand, so that they cost no instruction. A tile
// of the second kernel has eight rows therefore, and more of one expert's read its weights again.
template <int WF>
constexpr int kTerms = WF == YVMOE_W_F32 ? 1 : 2;
template <int WF>
constexpr int kTileRows = 16 / kTerms<WF>;

// 16 bytes at an offset (none, and nothing read, past the buffer's end). FRESH: read past the caches (h,
// which other work-groups of the launch have written).
template <bool FRESH>
__device__ __forceinline__ uint4 act_load16(__amdgpu_buffer_rsrc_t b, unsigned offset) {
    const u32x4 v = __builtin_amdgcn_raw_buffer_load_b128(b, offset, 0, FRESH ? 16 : 0);
    return make_uint4(v.x, v.y, v.z, v.w);
}

struct ActB16 {
    Frag16 f;
    static constexpr int BYTES = 2, LANE = 16;  // of an element; columns between lane groups
    template <bool FRESH>
    __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t b, unsigned row, int ks) {
        f.u[0] = act_load16<FRESH>(b, row + ks * 128);
        f.u[1] = act_load16<FRESH>(b, row + ks * 128 + 16);
    }
    __device__ __forceinline__ void read(const char* row, int ks) {
        f.u[0] = *(const uint4*)(row + ks * 128);
        f.u[1] = *(const uint4*)(row + ks * 128 + 16);
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
    static constexpr Depth DEPTH = {1, 3, 1, 4, 1, 4, 1, 4};
    static constexpr bool GROUPED = false;
    static __device__ __forceinline__ const char* ptr(const void* b, long long e, int n0, int K, int lane) {
        return block_ptr(b, e * 2, n0, K, 2048, 16, lane);
    }
    static __device__ __forceinline__ void load(Raw& r, const char* p, int ks) {
        r.u[0] = nt_load16(p + (size_t)ks * 2048);
        r.u[1] = nt_load16(p + (size_t)ks * 2048 + 1024);
    }
    static __device__ __forceinline__ const Frag16& frag(const Raw& w) { return w; }
};

template <>
struct Wt<YVMOE_W_INT8> {
    typedef uint4 Raw;
    typedef ActB16 Act;
    static constexpr Depth DEPTH = {2, 2, 4, 2, 2, 3, 4, 3};
    static constexpr bool GROUPED = false;
    static __device__ __forceinline__ const char* ptr(const void* b, long long e, int n0, int K, int lane) {
        return block_ptr(b, e, n0, K, 1024, 16, lane);
    }
    static __device__ __forceinline__ void load(Raw& r, const char* p, int ks) {
        r = nt_load16(p + (size_t)ks * 1024);
    }
    static __device__ __forceinline__ Frag16 frag(const Raw& r) {
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
        return f;
    }
};

template <>
struct Wt<YVMOE_W_FP8> {
    typedef uint4 Raw;
    typedef ActB16 Act;
    static constexpr Depth DEPTH = {2, 2, 4, 2, 2, 3, 4, 3};
    static constexpr bool GROUPED = true;
    static __device__ __forceinline__ const char* ptr(const void* b, long long e, int n0, int K, int lane) {
        return block_ptr(b, e, n0, K, 1024, 16, lane);
    }
    static __device__ __forceinline__ void load(Raw& r, const char* p, int ks) {
        r = nt_load16(p + (size_t)ks * 1024);
    }
    static __device__ __forceinline__ Frag16 frag(const Raw& r) {
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
        return f;
    }
};

// int4: a byte of value q < 16 is the e4m3 number q / 512, so two codes cost a conversion to bf16 and a
// share of the masks; the products' sum is Σ x q / 512, and one more MFMA with a constant operand gives
// -8 / 512 Σ x for the group, which makes it Σ x (q - 8) / 512. All are fp32 sums of exact products. The
// operand's columns then are 0, 2, 4, 6, 1, 3, 5, 7 of eight, and activations are kept in that order.
template <>
struct Wt<YVMOE_W_INT4> {
    typedef uint2 Raw;
    typedef ActB16 Act;
    static constexpr Depth DEPTH = {2, 3, 4, 4, 4, 3, 8, 3};
    static constexpr bool GROUPED = true;
    static __device__ __forceinline__ const char* ptr(const void* b, long long e, int n0, int K, int lane) {
        return block_ptr(b, e / 2, n0, K, 512, 8, lane);
    }
    static __device__ __forceinline__ void load(Raw& r, const char* p, int ks) {
        r = nt_load8(p + (size_t)ks * 512);
    }
    static __device__ __forceinline__ uint4 codes(unsigned w) {
        const int lo = (int)(w & 0x0F0F0F0Fu), hi = (int)(w >> 4 & 0x0F0F0F0Fu);
        return make_uint4(__builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false)),
                          __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true)),
                          __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false)),
                          __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true)));
    }
    static __device__ __forceinline__ void offset(const Act& a, f32x4& corr) {
        Frag16 c;
        c.u[0] = make_uint4(0xBC80BC80u, 0xBC80BC80u, 0xBC80BC80u, 0xBC80BC80u);  // -8 / 512
        corr = mfma16(a.f.v[0], c.v[0], corr);
        corr = mfma16(a.f.v[1], c.v[0], corr);
    }
    static __device__ __forceinline__ Frag16 frag(const Raw& r) {
        Frag16 f;
        f.u[0] = codes(r.x);
        f.u[1] = codes(r.y);
        return f;
    }
};
// Eight columns of bf16 activations in int4's order; its inverse place of a column is int4_place.
__device__ __forceinline__ uint4 int4_order(const uint4& v) {
    return make_uint4(__builtin_amdgcn_perm(v.y, v.x, 0x05040100u), __builtin_amdgcn_perm(v.w, v.z, 0x05040100u),
                      __builtin_amdgcn_perm(v.y, v.x, 0x07060302u), __builtin_amdgcn_perm(v.w, v.z, 0x07060302u));
}
__device__ __forceinline__ int int4_place(int col) { return (col & ~7) | (col & 7) >> 1 | (col & 1) << 2; }

// fp32: rows as they are, on the fp32 MFMAs. Lane group g holds columns 16 i + 4 g .. 16 i + 4 g + 3 for
// i = 0..3, so that a load of 16 bytes takes 64 of a row.
template <>
struct Wt<YVMOE_W_F32> {
    struct Raw {
        uint4 v[4];
    };
    struct Act {
        uint4 v[4];
        static constexpr int BYTES = 4, LANE = 4;
        template <bool FRESH>
        __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t b, unsigned row, int ks) {
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = act_load16<FRESH>(b, row + ks * 256 + 64 * i);
        }
        __device__ __forceinline__ void read(const char* row, int ks) {
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = *(const uint4*)(row + ks * 256 + 64 * i);
        }
    };
    static constexpr Depth DEPTH = {1, 2, 1, 3, 1, 3, 2, 3};
    static constexpr bool GROUPED = false;
    static __device__ __forceinline__ const char* ptr(const void* b, long long e, int n0, int K, int lane) {
        return (const char*)b + (e + (long long)(n0 + (lane & 15)) * K + 4 * (lane >> 4)) * 4;
    }
    static __device__ __forceinline__ void load(Raw& r, const char* p, int ks) {
#pragma unroll
        for (int i = 0; i < 4; ++i) r.v[i] = nt_load16(p + (size_t)ks * 256 + 64 * i);
    }
    static __device__ __forceinline__ void mma(const Raw& w, const Act& a, f32x4& acc) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            acc = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a.v[i].x), __uint_as_float(w.v[i].x), acc, 0, 0, 0);
            acc = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a.v[i].y), __uint_as_float(w.v[i].y), acc, 0, 0, 0);
            acc = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a.v[i].z), __uint_as_float(w.v[i].z), acc, 0, 0, 0);
            acc = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a.v[i].w), __uint_as_float(w.v[i].w), acc, 0, 0, 0);
        }
    }
};

// Activation rows that fit are kept in LDS, padded so that 16 rows' pieces fall on different banks. (int4 reads
// two bytes of activations for one of weights: with x in LDS 4 tokens of 5120 -> 1536 take 122 us, not 140.) One
// room for all: x from its start and the router's logits, then the wavefronts' sums at its end; for the down
// product h from its start, then the partial outputs.
constexpr int kPoolBytes = 151296, kEndBytes = 32768, kRowPad = 16;
typedef __attribute__((address_space(3))) void* lds_ptr_t;
typedef const __attribute__((address_space(1))) void* gbl_ptr_t;

// Loads nrows rows of bytes (a multiple of 128) straight into LDS; done when the loads are. FRESH as above.
template <bool FRESH>
__device__ __forceinline__ void stage_rows(const void* src, int nrows, int bytes, char* lds, int wave, int lane) {
    const int pieces = (bytes + 1023) / 1024;  // of a row, 16 bytes per lane
    for (int i = wave; i < nrows * pieces; i += kWaves + 1) {
        const int row = i / pieces, at = (i - row * pieces) * 1024;
        if (at + 16 * lane < bytes)
            __builtin_amdgcn_global_load_lds((gbl_ptr_t)((const char*)src + (long long)row * bytes + at + 16 * lane),
                                             (lds_ptr_t)(lds + row * (bytes + kRowPad) + at), 16, 0, FRESH ? 16 : 0);
    }
}

// NM matrices' 16 rows from n0 against one set of activation rows.
template <int WF, int NM>
struct Operands {
    typedef typename Wt<WF>::Act Act;
    const char* w[NM];
    const void* s[NM];  // the scales: int8, int4 of the lane's row, fp8 of these rows
    int left[NM];       // int4: scales from there to the end of all
    __amdgpu_buffer_rsrc_t buf;  // the activations, and the lane's row in them at its columns
    unsigned off;

    __device__ __forceinline__ void set(int m, const void* base, const void* scales, long long e, int total, int out,
                                        int K, int n0, int lane) {
        w[m] = Wt<WF>::ptr(base, e * out * K, n0, K, lane);
        if constexpr (WF == YVMOE_W_INT4) {
            const long long at = (e * out + n0 + (lane & 15)) * (K / 128);
            s[m] = (const unsigned short*)scales + at;
            left[m] = (int)min((long long)total * out * (K / 128) - at, 1ll << 20);
        }
        else if constexpr (WF == YVMOE_W_FP8)
            s[m] = (const float*)scales + (e * (out / 128) + n0 / 128) * (K / 128);
        else if constexpr (WF == YVMOE_W_INT8)
            s[m] = (const unsigned short*)scales + e * out + n0 + (lane & 15);
        else s[m] = nullptr;
    }
    // row < 0: a lane without a row, whose loads give zero and read nothing. LDS: where stage_rows puts
    // the rows (such a lane then reads some row; its products are not used).
    template <bool LDS>
    __device__ __forceinline__ void rows(const void* base, int nrows, int row, int K, int lane) {
        if constexpr (LDS) {
            off = (unsigned)((row < 0 ? 0 : row) * (K * Act::BYTES + kRowPad) + Act::LANE * (lane >> 4) * Act::BYTES);
            return;
        }
        buf = __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, nrows * K * Act::BYTES, 0x00027000);
        off = row < 0 ? 0x80000000u : (unsigned)(row * K + Act::LANE * (lane >> 4)) * Act::BYTES;
    }
};

// A chunk in flight: its weights with their scales, and where its activations are.
template <int WF, int NM, bool LDS>
struct Chunk {
    typedef Wt<WF> W;
    static constexpr int U = W::DEPTH.unit(NM, LDS);
    typename W::Raw w[U][NM];
    struct __attribute__((packed, aligned(2))) Scales {
        typename std::conditional<(U > 4), unsigned long long,
                                  typename std::conditional<(U > 2), unsigned, unsigned short>::type>::type v;
    };
    float s[WF == YVMOE_W_FP8 ? U / 2 : 1][NM];
    Scales sraw[NM];  // int4
    int sshift[NM];
    float rs[NM];  // int8: the row's scale
    int c;
    unsigned act;

    __device__ __forceinline__ float scale(int group, int m) const {
        if constexpr (WF == YVMOE_W_INT4)
            return 512.0f * bf16_to_f32((unsigned short)(sraw[m].v >> (sshift[m] + 16 * group)));
        return s[WF == YVMOE_W_FP8 ? group : 0][m];
    }

    // k-steps past the end: the last one again, not used. int8's scales with every chunk: loads on one
    // path only would make the compiler wait for them at once.
    template <class Ops>
    __device__ __forceinline__ void load_weights(const Ops& o, int chunk, int nks) {
        c = chunk;
        act = o.off;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int ks = min(c * U + u, nks - 1);
#pragma unroll
            for (int m = 0; m < NM; ++m) {
                W::load(w[u][m], o.w[m], ks);
                if constexpr (WF == YVMOE_W_FP8)
                    if (u % 2 == 0) s[u / 2][m] = ((const float*)o.s[m])[ks / 2];
            }
        }
        if constexpr (WF == YVMOE_W_INT4) {
            // a row's scales of the chunk in one load (each touches 16 rows' lines, whatever its width: 2 tokens of
            // 5120 -> 1536 take 79.9 us, 82.3 with a load a group), which starts early enough to end with the array
            const int start = min(c * (U / 2), (nks - 1) / 2);
#pragma unroll
            for (int m = 0; m < NM; ++m) {
                const int from = min(start, o.left[m] - U / 2);
                sraw[m] = *(const Scales*)((const unsigned short*)o.s[m] + from);
                sshift[m] = 16 * (start - from);
            }
        }
        if constexpr (WF == YVMOE_W_INT8)
#pragma unroll
            for (int m = 0; m < NM; ++m) rs[m] = bf16_to_f32(*(const unsigned short*)o.s[m]);
    }
};
template <int WF, int NM, bool LDS>
struct Acts {
    static constexpr int U = Wt<WF>::DEPTH.unit(NM, LDS);
    typename Wt<WF>::Act a[U];
    template <bool FRESH>
    __device__ __forceinline__ void load(const Chunk<WF, NM, LDS>& q, __amdgpu_buffer_rsrc_t buf, int nks) {
#pragma unroll
        for (int u = 0; u < U; ++u) a[u].template load<FRESH>(buf, q.act, min(q.c * U + u, nks - 1));
    }
    __device__ __forceinline__ void read(const Chunk<WF, NM, LDS>& q, const char* lds, int nks) {
#pragma unroll
        for (int u = 0; u < U; ++u) a[u].read(lds + q.act, min(q.c * U + u, nks - 1));
    }
};

// A k-step's products of a matrix.
template <int WF>
__device__ __forceinline__ void products(const typename Wt<WF>::Raw& w, const typename Wt<WF>::Act& a, f32x4& acc) {
    if constexpr (WF == YVMOE_W_F32) {
        Wt<WF>::mma(w, a, acc);
    } else {
        const Frag16 f = Wt<WF>::frag(w);
        acc = mfma16(a.f.v[0], f.v[0], acc);
        acc = mfma16(a.f.v[1], f.v[1], acc);
    }
}

// ORDER: the activations are as the caller has them, not in int4's order yet.
template <int WF, int NM, bool LDS, bool ORDER>
__device__ __forceinline__ void mma(const Chunk<WF, NM, LDS>& q, Acts<WF, NM, LDS>& x, int nks, f32x4 (&acc)[NM]) {
    typedef Wt<WF> W;
    const int c = q.c;
    constexpr int U = W::DEPTH.unit(NM, LDS);
    if constexpr (!W::GROUPED) {
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (c * U + u < nks)
#pragma unroll
                for (int m = 0; m < NM; ++m) products<WF>(q.w[u][m], x.a[u], acc[m]);
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
                    if constexpr (ORDER)
#pragma unroll
                        for (int h = 0; h < 2; ++h) x.a[u].f.u[h] = int4_order(x.a[u].f.u[h]);
                    W::offset(x.a[u], corr);
                }
#pragma unroll
                for (int m = 0; m < NM; ++m) products<WF>(q.w[u][m], x.a[u], part[m]);
            }
#pragma unroll
            for (int m = 0; m < NM; ++m) {
                const float s = q.scale(p / 2, m);
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    acc[m][i] = __builtin_fmaf(s, WF == YVMOE_W_INT4 ? part[m][i] + corr[i] : part[m][i], acc[m][i]);
            }
        }
    }
}

template <int WF, int NM, bool LDS>
__device__ __forceinline__ int chunks(int K) {
    constexpr int U = Wt<WF>::DEPTH.unit(NM, LDS);
    return (K / 64 + U - 1) / U;
}

// A wavefront's products along a walk. The walk stands at a chunk (o, c; c past the end: nothing) with
// its place(): whether the products up to it end there (ends) and whether they are all (all); next()
// moves it one on, after the end to lines that everyone reads. While a chunk is multiplied, the weights
// of the next ones and (without LDS) the activations of the next are in flight, across items too. The
// start is apart, so that the weights' part of it can come before a wait.
template <int WF, int NM, class Walk, bool LDS, bool FRESH = false, bool ORDER = false>
struct Ring {
    static constexpr int kRing = Wt<WF>::DEPTH.ring(NM, LDS);
    static_assert(kRing <= kOwnItems - 1, "what the streams look ahead");
    Chunk<WF, NM, LDS> q[kRing];
    Acts<WF, NM, LDS> x[LDS ? 1 : 2];
    typename Walk::Place place[kRing];

    __device__ __forceinline__ void start_weights(Walk& w, int nks) {
#pragma unroll
        for (int i = 0; i < kRing - 1; ++i) {
            q[i].load_weights(w.o, w.c, nks);
            place[i] = w.place();
            w.next();
        }
    }
    __device__ __forceinline__ void start_acts(Walk& w, int nks) {
        if constexpr (!LDS) x[0].template load<FRESH>(q[0], w.o.buf, nks);
    }

    template <class End>
    __device__ __forceinline__ void run(Walk& w, const char* lds, int nks, End end) {
        constexpr int STEPS = LDS || kRing % 2 == 0 ? kRing : 2 * kRing;
        f32x4 acc[NM];
#pragma unroll
        for (int m = 0; m < NM; ++m) acc[m] = f32x4{0.f, 0.f, 0.f, 0.f};
        while (true) {
#pragma unroll
            for (int i = 0; i < STEPS; ++i) {
                constexpr int AHEAD = kRing - 1;
                Chunk<WF, NM, LDS>&p = q[i % kRing], &n = q[(i + AHEAD) % kRing];
                if constexpr (!LDS && kRing > 2) x[(i + 1) % 2].template load<FRESH>(q[(i + 1) % kRing], w.o.buf, nks);
                n.load_weights(w.o, w.c, nks);
                if constexpr (!LDS && kRing == 2) x[(i + 1) % 2].template load<FRESH>(n, w.o.buf, nks);
                place[(i + AHEAD) % kRing] = w.place();
                w.next();
                __builtin_amdgcn_sched_barrier(0);
                if constexpr (LDS) x[0].read(p, lds, nks);
                mma<WF, NM, LDS, ORDER>(p, x[LDS ? 0 : i % 2], nks, acc);
                if (place[i % kRing].ends) {
                    if constexpr (WF == YVMOE_W_INT8)
#pragma unroll
                        for (int m = 0; m < NM; ++m)
#pragma unroll
                            for (int r = 0; r < 4; ++r) acc[m][r] = acc[m][r] * p.rs[m];
                    end(place[i % kRing], acc);
#pragma unroll
                    for (int m = 0; m < NM; ++m) acc[m] = f32x4{0.f, 0.f, 0.f, 0.f};
                    if (place[i % kRing].all) return;
                }
            }
        }
    }
};

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

// h of four activation rows from row and one column, below row + n (int4: in its order of columns), its second
// term nrows rows further on. PUBLISH: written through to where every XCD reads it.
template <int WF, bool PUBLISH>
__device__ __forceinline__ void store_h(void* h, long long row, int n, int nrows, int F, int col, const f32x4& g,
                                        const f32x4& u) {
    const int at = WF == YVMOE_W_INT4 ? int4_place(col) : col;
    auto put = [&](auto* p, auto v) {
        if constexpr (PUBLISH) __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        else *p = v;
    };
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (i >= n) break;
        const float f = silu(g[i]) * u[i];
        if constexpr (WF == YVMOE_W_F32) {
            put((float*)h + (row + i) * F + at, f);
        } else {
            unsigned short* p = (unsigned short*)h + (row + i) * F + at;
            const unsigned short hi = f32_to_bf16_rne(f);
            const bool finite = (hi & 0x7f80u) != 0x7f80u;
            put(p, hi);
            put(p + (long long)nrows * F, finite ? f32_to_bf16_rne(f - bf16_to_f32(hi)) : (unsigned short)0);
        }
    }
}

// A work-group's gate/up items: 16 columns of F of a tile each. at(item) sets e, n0, row0, n and the
// lane's token (-1: none). The items are first, first + own, ... (kOwnItems, below nitems), then, where
// ahead is given, those that stand in ahead[it & 7] for the it-th.
// A stream that has passed item i - 1's barrier may load item i + RING - 1 and, to know whether that is
// its last, looks at the item after it: i + 4 at most. That one is there before item i - 1's barrier.
struct GateUpItems {
    int item, nitems, own;
    const int* ahead;
    int it;
    __device__ __forceinline__ bool advance() {
        ++it;
        item = it < kOwnItems ? item + own
               : ahead != nullptr ? __builtin_amdgcn_readfirstlane(ahead[it & 7])
                                  : nitems;
        return item < nitems;
    }
};

// A streaming wavefront's way along them: the wavefronts deal out the chunks of K.
template <int WF, bool LDS, class At>
struct GateUpWalk {
    struct Place {
        bool ends, all;
    };
    const FewArgs& a;
    const void* x;
    At at;
    GateUpItems items;
    int nch, wave, lane;
    Operands<WF, 2> o;
    int c, s;
    bool stop, final;

    __device__ __forceinline__ GateUpWalk(const FewArgs& args, const void* acts, At f, const GateUpItems& list, int wv,
                                          int ln)
        : a(args), x(acts), at(f), items(list), nch(chunks<WF, 2, LDS>(args.H)), wave(wv), lane(ln), stop(false) {
        enter();
    }
    __device__ __forceinline__ void enter() {
        int e, n0, row0, n, token;
        at(items.item, e, n0, row0, n, token);
        o.set(0, a.w_gate, a.s_gate, e, a.E + a.S, a.F, a.H, n0, lane);
        o.set(1, a.w_up, a.s_up, e, a.E + a.S, a.F, a.H, n0, lane);
        o.template rows<LDS>(x, a.N, token, a.H, lane);
        s = 0;
        c = wave;
    }
    // every wavefront takes as many steps, chunks past the end among them, so that all end alike
    __device__ __forceinline__ Place place() {
        const bool last = (s + 1) * kWaves >= nch && !stop;
        if (last) final = !items.advance();
        return {last, last && final};
    }
    __device__ __forceinline__ void next() {
        if ((s + 1) * kWaves < nch || stop) {
            ++s;
            c += stop ? 0 : kWaves;
        } else if (!final) {
            enter();
        } else {
            o.set(0, a.w_gate, a.s_gate, 0, a.E + a.S, a.F, a.H, 0, lane);
            o.set(1, a.w_up, a.s_up, 0, a.E + a.S, a.F, a.H, 0, lane);
            c = 0;
            stop = true;
        }
    }
};

// Runs a list of items to their h rows; returns their number on the last wavefront. PUBLISH: h is read in
// this launch, and x is xo (the second kernel; the first makes xo). One barrier an
// item (red alternates between two sets): the last wavefront sums an item while the others stream the
// next. Items past the list's own are taken from the counter (ticket), kOwnItems ahead of their turn.
template <int WF, bool PUBLISH, bool LDS, class At>
__device__ __forceinline__ int gate_up(const FewArgs& a, At at, GateUpItems items, f32x4 (&red)[2][kWaves][2][64],
                                       int* ahead, unsigned* ticket, const char* lds, int wave, int lane) {
    if (wave < kWaves) {
        typedef GateUpWalk<WF, LDS, At> Walk;
        Walk w(a, PUBLISH ? a.xo : a.x, at, items, wave, lane);
        Ring<WF, 2, Walk, LDS, false, !PUBLISH> ring;
        ring.start_weights(w, a.H / 64);
        ring.start_acts(w, a.H / 64);
        int it = 0;
        ring.run(w, lds, a.H / 64, [&](const typename Walk::Place&, const f32x4 (&acc)[2]) {
            red[it & 1][wave][0][lane] = acc[0];
            red[it & 1][wave][1][lane] = acc[1];
            __syncthreads();
            ++it;
        });
        return 0;
    }
    const int limit = kOwnItems * items.own;
    bool more;
    do {
        int e, n0, row0, n, token;
        at(items.item, e, n0, row0, n, token);
        const int it = items.it;
        if (items.ahead != nullptr && lane == 0)
            ahead[(it + kOwnItems) & 7] =
                limit + (int)__hip_atomic_fetch_add(ticket, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __syncthreads();
        f32x4 sum[2];
        sum_waves<2>(red[it & 1], lane, sum);
        const int g = lane >> 4;
        store_h<WF, PUBLISH>(a.h, row0 + 4 * g, n - 4 * g, a.N * (a.k + a.S), a.F, n0 + (lane & 15), sum[0], sum[1]);
        more = items.advance();
    } while (more);
    return items.it;
}

// ---------------------------------------------------------------- first kernel
// The router's products: 16 columns, K's chunks [c, end) dealt out to the wavefronts.
template <int RF>
struct RouterWalk {
    struct Place {
        bool ends, all;
    };
    Operands<RF, 1> o;
    int c, end;
    __device__ __forceinline__ Place place() const { return {c < end && c + kWaves >= end, c < end && c + kWaves >= end}; }
    __device__ __forceinline__ void next() { c += kWaves; }
};

// Work-groups: the router's (16 columns, K split) items, then the shared experts' gate/up items.
template <int WF>
__global__ __launch_bounds__(kAllThreads, 3) void few_front_kernel(FewArgs a) {
    constexpr int RF = WF == YVMOE_W_F32 ? YVMOE_W_F32 : YVMOE_W_BF16;
    __shared__ f32x4 red[2][kWaves][2][64];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 15;
    int b = blockIdx.x;
    if (b == 0) {
        for (int i = threadIdx.x; i < SIG_COUNT; i += kAllThreads) a.signals[32 * i] = i < SIG_GO ? 0 : a.wait_mode;
        if (a.hparts > 1)
            for (int i = threadIdx.x; i < a.H / 16; i += kAllThreads) a.hcount[i] = 0;
    }
    if constexpr (WF == YVMOE_W_INT4)
        for (long long i = (long long)b * kAllThreads + threadIdx.x; i < (long long)a.N * a.H / 8;
             i += (long long)gridDim.x * kAllThreads)
            ((uint4*)a.xo)[i] = int4_order(((const uint4*)a.x)[i]);
    const int nrouter = a.self ? a.ncols / 16 * a.nsplit : 0;
    if (b < nrouter) {
        const int n0 = b / a.nsplit * 16, z = b % a.nsplit, nch = chunks<RF, 1, false>(a.H), nks = a.H / 64;
        RouterWalk<RF> w;
        w.o.set(0, a.w_router, nullptr, 0, 1, a.ld, a.H, n0, lane);
        w.o.template rows<false>(a.x, a.N, r < a.N ? r : -1, a.H, lane);
        w.c = z * nch / a.nsplit + wave;
        w.end = (z + 1) * nch / a.nsplit;
        if (wave < kWaves) red[0][wave][0][lane] = f32x4{0.f, 0.f, 0.f, 0.f};
        if (wave < kWaves && w.c < w.end) {
            Ring<RF, 1, RouterWalk<RF>, false> ring;
            ring.start_weights(w, nks);
            ring.start_acts(w, nks);
            ring.run(w, nullptr, nks, [&](const typename RouterWalk<RF>::Place&, const f32x4 (&acc)[1]) {
                red[0][wave][0][lane] = acc[0];
            });
        }
        __syncthreads();
        if (wave != kWaves) return;
        f32x4 sum[1];
        sum_waves<1>(red[0], lane, sum);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int tok = 4 * (lane >> 4) + i;
            if (tok < a.N) a.logits[((long long)z * a.N + tok) * a.ld + n0 + r] = sum[0][i];
        }
        return;
    }
    b -= nrouter;
    const int nfb = a.F / 16, nitems = a.S * nfb;
    if (b >= nitems) return;
    auto at = [&](int item, int& e, int& n0, int& row0, int& n, int& token) {
        const int s = item / nfb;
        e = a.E + s;
        n0 = item % nfb * 16;
        row0 = a.N * (a.k + s);
        n = a.N;
        token = r < a.N ? r : -1;
    };
    gate_up<WF, false, false>(a, at, GateUpItems{b, b + 1, 1, nullptr, 0}, red, nullptr, nullptr, nullptr, wave, lane);
}

// ---------------------------------------------------------------- second kernel
struct FewTables {
    short expert[kFewSlots];  // of each slot, -1: none
    float p[kFewSlots];       // its probability
    float w[kFewSlots];       // its weight
    int place[kFewSlots];     // slots of lower experts, earlier ones of its own, better ones of its own
    short pos[kFewSlots];     // its row, -1: none
    short slot[kFewSlots];    // slot of each routed row
    short first[kFewSlots];   // a routed row's place among its expert's
    short tile_e[kFewTiles], tile_row0[kFewTiles], tile_n[kFewTiles];
    float score[kFewTokens];
    int counts[YVMOE_MAX_EXPERTS];
    int wave_starts[4];
    int nrows, ntiles, cap, help;
    int ahead[8];
};

// Logits and predictor terms of the tokens, summed over the splits, and the predictor's constants.
struct FewLogits {
    float z[kFewTokens][YVMOE_MAX_EXPERTS];
    float pred[kFewTokens][3 * kPredDim];
    float b1[kPredDim], w2[kPredDim], b2[1], bias[YVMOE_MAX_EXPERTS];
};

// Largest of the wavefront's numbers, on every lane: rows of 16 by rotation, then row to row.
__device__ __forceinline__ unsigned wave_max(unsigned v) {
#define YV_STEP(CTRL, ROWS) v = max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, false))
    YV_STEP(0x128, 0xf);  // row_ror 8, 4, 2, 1
    YV_STEP(0x124, 0xf);
    YV_STEP(0x122, 0xf);
    YV_STEP(0x121, 0xf);
    YV_STEP(0x142, 0xa);  // row_bcast 15, 31
    YV_STEP(0x143, 0xc);
#undef YV_STEP
    return (unsigned)__builtin_amdgcn_readlane((int)v, 63);
}

// topk_token by a whole wavefront (lane l holds experts l, l + 64, ...): the same arithmetic, its 16
// partial sums included, so the same bits. A candidate's key is its probability's bits plus one; taken
// and NaN entries hold 0.
template <int NV>
__device__ __forceinline__ void topk_wave(const float* lg, const float* bias, int lane, int E, int k, int& my_id,
                                          float& my_ts, float& my_w0) {
#pragma clang fp contract(off)
    float z[NV];
    float m = -__builtin_huge_valf();
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int e = lane + 64 * i;
        z[i] = e < E ? (bias != nullptr ? lg[e] + bias[e] : lg[e]) : -__builtin_huge_valf();
        if (z[i] > m) m = z[i];
    }
    const unsigned mb = __float_as_uint(m);  // floats' order as unsigned numbers'
    const unsigned mo = wave_max(mb & 0x80000000u ? ~mb : mb | 0x80000000u);
    m = __uint_as_float(mo & 0x80000000u ? mo & 0x7fffffffu : ~mo);
#pragma unroll
    for (int i = 0; i < NV; ++i) z[i] = lane + 64 * i < E ? yv_expf(z[i] - m) : 0.0f;
    // partial l: experts l, l + 16, ... in order
    float part = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const float v = __int_as_float(__builtin_amdgcn_ds_bpermute(4 * (16 * q + (lane & 15)), __float_as_int(z[i])));
            if (64 * i + 16 * q + (lane & 15) < E) part = part + v;
        }
#define YV_SUMSTEP(O) part = part + rot16<O>(part)
    YV_BFLY16(YV_SUMSTEP);
#undef YV_SUMSTEP
    unsigned key[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const float p = z[i] / part;
        key[i] = (lane + 64 * i < E && p == p) ? __float_as_uint(p) + 1u : 0u;
    }
    my_ts = 0.0f;
    my_id = 0;
    for (int j = 0; j < k; ++j) {
        unsigned b = key[0];
#pragma unroll
        for (int i = 1; i < NV; ++i) b = max(b, key[i]);
        b = wave_max(b);
        int id = 0x7fffffff;  // the lowest expert with that key
#pragma unroll
        for (int i = NV - 1; i >= 0; --i) {
            const unsigned long long who = __ballot(key[i] == b);
            if (who != 0) id = 64 * i + __ffsll(who) - 1;
        }
        if (b == 0) id = j;  // all probabilities are NaN
#pragma unroll
        for (int i = 0; i < NV; ++i) key[i] = lane + 64 * i == id ? 0u : key[i];
        if (lane == j) {
            my_ts = b != 0 ? __uint_as_float(b - 1u) : __builtin_nanf("");
            my_id = id;
        }
    }
    const float ts0 = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(my_ts), 0));
    const float ej = yv_expf(my_ts - ts0);
    float tot = 0.0f;
    for (int j = 0; j < k; ++j) tot = tot + __int_as_float(__builtin_amdgcn_readlane(__float_as_int(ej), j));
    my_w0 = ej / tot;
}

// The routing of up to 16 tokens, from the logits or as given, and the tiles: up to ROWS rows of one
// expert each. Every work-group computes it; the first one also writes it out.
template <int ROWS>
__device__ __forceinline__ void few_routing(const FewArgs& a, FewTables& t, FewLogits& lg, bool writer) {
#pragma clang fp contract(off)
    const int tid = threadIdx.x, N = a.N, E = a.E, k = a.k, ns = N * k;
    if (tid == 0) {
        t.nrows = 0;
        t.cap = -1;
    }
    if (tid < YVMOE_MAX_EXPERTS) t.counts[tid] = 0;
    if (tid < kFewSlots) t.place[tid] = 0;
    if (a.self) {
        const bool scores = a.cap_mode == 2;
        const int Ep = (E + 15) / 16 * 16, terms = (a.ld - Ep) / kPredDim;
        const int ncols = scores ? a.ld : E;
        const long long sstride = (long long)N * a.ld;
        const int total = N * ncols;
        for (int base = 0; base < total; base += 4 * kAllThreads) {
            float part[4][4];  // unconditional loads, so that all are in flight together
            int tok[4], col[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int i = min(base + j * kAllThreads + tid, total - 1);
                tok[j] = i / ncols;
                col[j] = i - tok[j] * ncols;
                const float* p = a.logits + (long long)tok[j] * a.ld + col[j];
#pragma unroll
                for (int z = 0; z < 4; ++z) part[j][z] = p[min(z, a.nsplit - 1) * sstride];
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (base + j * kAllThreads + tid >= total) break;
                float v = part[j][0];
#pragma unroll
                for (int z = 1; z < 4; ++z) v = z < a.nsplit ? v + part[j][z] : v;
                if (col[j] < E) lg.z[tok[j]][col[j]] = v;
                else if (col[j] >= Ep) lg.pred[tok[j]][col[j] - Ep] = v;
            }
        }
        if (tid < E) lg.bias[tid] = a.bias != nullptr ? a.bias[tid] : 0.0f;
        if (scores && tid < kPredDim) {
            lg.b1[tid] = a.b1[tid];
            lg.w2[tid] = a.w2[tid];
            if (tid == 0) lg.b2[0] = a.b2[0];
        }
        __syncthreads();
        const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
        // a token's choice by a wavefront, the scores of four tokens by another
        const int njobs = N + (scores ? (N + 3) / 4 : 0);
        for (int job = wave; job < njobs; job += kWaves + 1) {
            if (job < N) {
                int id;
                float p, w;
                const float* bias = a.bias != nullptr ? lg.bias : nullptr;
                if (E <= 64) topk_wave<1>(lg.z[job], bias, lane, E, k, id, p, w);
                else if (E <= 128) topk_wave<2>(lg.z[job], bias, lane, E, k, id, p, w);
                else topk_wave<4>(lg.z[job], bias, lane, E, k, id, p, w);
                if (lane < k) {
                    t.expert[job * k + lane] = (short)id;
                    t.p[job * k + lane] = p;
                    t.w[job * k + lane] = w;
                    if (writer) a.out_routing.indices[job * k + lane] = id;
                }
            } else {
                const int tok = 4 * (job - N) + (lane >> 4), in = min(tok, N - 1);
                const float sc = predictor_token([&](int c) { return lg.pred[in][c]; }, terms, lg.b1, lg.w2, lg.b2,
                                                 lane & 15);
                if ((lane & 15) == 0 && tok < N) t.score[tok] = sc;
            }
        }
    } else if (tid < ns) {
        const int64_t id = a.rindices[tid];
        t.expert[tid] = id >= 0 && id < E ? (short)id : (short)-1;
        t.w[tid] = a.rweights_bf16 ? bf16_to_f32(((const unsigned short*)a.rweights)[tid])
                                   : ((const float*)a.rweights)[tid];
    }
    __syncthreads();
    if (tid == kThreads - 1 && a.self && a.cap_mode != 0) {
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
    // a slot's row: after all slots of lower experts and the earlier ones of its own; its rank among its
    // expert's by probability. Several threads a slot, each over a part of the slots.
    {
        int threads = kThreads, pad = 1;  // slots rounded up to a power of two: pad threads a part
        while (pad < ns) pad *= 2;
        const int nparts = threads / pad, i = tid & (pad - 1), q = tid / pad;
        const int len = (ns + nparts - 1) / nparts, s1 = min(ns, (q + 1) * len);
        const int e = i < ns ? t.expert[i] : -1;
        const float p = i < ns && a.self ? t.p[i] : 0.0f;
        int lower = 0, before = 0, better = 0;
        if (e >= 0) {
            for (int s = q * len; s < s1; s += 4) {
                int es[4];
                float ps[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    es[j] = t.expert[min(s + j, kFewSlots - 1)];
                    ps[j] = t.p[min(s + j, kFewSlots - 1)];
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const bool in = s + j < s1, same = in && es[j] == e, earlier = s + j < i;
                    lower += in && es[j] >= 0 && es[j] < e ? 1 : 0;
                    before += same && earlier ? 1 : 0;
                    better += same && (ps[j] > p || (ps[j] == p && earlier)) ? 1 : 0;
                }
            }
            atomicAdd(&t.place[i], lower | before << 10 | better << 20);
            if (q == 0) atomicAdd(&t.counts[e], 1);
        }
    }
    __syncthreads();
    int mine = -1, before = 0, better = 0;
    if (tid < ns) {
        mine = t.expert[tid];
        const int v = t.place[tid];
        before = v >> 10 & 1023;
        better = v >> 20;
        const int pos = (v & 1023) + before;
        if (mine >= 0) {
            t.slot[pos] = (short)tid;
            t.first[pos] = (short)before;
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
        start = tid < nrows && t.first[tid] % ROWS == 0;
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
        t.tile_n[i] = (short)min(ROWS, t.counts[e] - t.first[tid]);
    }
    const int ntiles = t.wave_starts[0] + t.wave_starts[1] + t.wave_starts[2] + t.wave_starts[3];
    const int each = (N + ROWS - 1) / ROWS;
    if (tid < a.S * each) {
        const int e = tid / each, from = (tid - e * each) * ROWS;
        t.tile_e[ntiles + tid] = (short)(E + e);
        t.tile_row0[ntiles + tid] = (short)(ns + e * N + from);
        t.tile_n[ntiles + tid] = (short)min(ROWS, N - from);
    }
    if (tid == 0) t.ntiles = ntiles;
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

// One term of a token's sum: weight, and row of the partial outputs, or none.
struct Term {
    float w;
    int row;
};

// The terms of all sums, in order: parts of slots 0 .. N k, then of the shared experts of each token. By the last
// wavefront, which reads them and has time for it before it waits.
__device__ __forceinline__ void list_terms(const FewArgs& a, const FewTables& t, Term* list, int nrows, int lane) {
    const int ns = a.N * a.k;
    for (int i = lane; i < nrows * a.parts; i += 64) {
        const int s = i / a.parts, q = i - s * a.parts;
        int row;
        float w;
        if (s < ns) {
            row = t.pos[s];
            w = t.w[s];
        } else {
            const int tok = (s - ns) / a.S, e = s - ns - tok * a.S;
            row = ns + e * a.N + tok;
            w = a.mix[e];
        }
        list[i] = row >= 0 ? Term{w, q * nrows + row} : Term{0.0f, -1};
    }
}

// A share's own items are done, and so are extra items that were handed out: called by one wavefront
// when their h has been written. Whoever completes the last of the words says so to everyone.
__device__ __forceinline__ void signal_done(const FewArgs& a, int share, int used, int extra, int handed, int lane) {
    auto word = [&](int i) { return a.signals + 32 * i; };
    unsigned complete = 0;
    if (lane == 0) {
        const unsigned bit = 1u << (share % 32), full = used - share / 32 * 32 >= 32 ? ~0u : (1u << (used % 32)) - 1u;
        const unsigned old =
            __hip_atomic_fetch_or(word(SIG_MARKS + share / 32), bit, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        if (old != full && (old | bit) == full) ++complete;
        if (extra > 0 && __hip_atomic_fetch_add(word(SIG_FINISHED), (unsigned)extra, __ATOMIC_RELAXED,
                                                __HIP_MEMORY_SCOPE_AGENT) + extra == (unsigned)handed)
            ++complete;
        const unsigned all = (used + 31) / 32 + (handed > 0 ? 1 : 0);
        if (complete > 0)
            complete = __hip_atomic_fetch_add(word(SIG_ROOT), complete, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) +
                               complete == all;
    }
    if (__builtin_amdgcn_readfirstlane(complete) != 0 && lane < kGoLines)
        __hip_atomic_store(word(SIG_GO + lane), (unsigned)GO_DONE, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// Waits until all is done, or kPatience looks: then a share whose mark is missing, if there is one. With none
// missing some other work-group holds items that were handed out, and the wait goes on for kMostRounds: only
// another call that has cleared the words meanwhile brings it there. Called by one wavefront.
__device__ __forceinline__ int wait_done(const FewArgs& a, int used, int lane) {
    unsigned* go = a.signals + 32 * (SIG_GO + blockIdx.x % kGoLines);
    for (int round = 0;; ++round) {
        unsigned now = 0;
        for (int i = 0; i < kPatience && now == 0; ++i) {
            now = __builtin_amdgcn_readfirstlane(__hip_atomic_load(go, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
            if (now == GO_DONE) return WAIT_DONE;
            __builtin_amdgcn_s_sleep(8);
        }
        if (now == GO_NO_WAIT) return WAIT_GIVEN_UP;
        unsigned m = ~0u;
        if (lane * 32 < used) {
            m = __hip_atomic_load(a.signals + 32 * (SIG_MARKS + lane), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            if (used - lane * 32 < 32) m |= ~0u << (used - lane * 32);
        }
        const unsigned long long open = __ballot(m != ~0u);
        if (open != 0) {
            // work-groups start to help at different places
            const unsigned long long turned = open & ~((1ull << (blockIdx.x & 7)) - 1ull);
            const int l = __ffsll(turned != 0 ? turned : open) - 1;
            return __builtin_amdgcn_readlane(32 * lane + __ffs(~m) - 1, l);
        }
        if (round >= (now == 0 ? kMostRounds : kPatience * kMostRounds)) return WAIT_GIVEN_UP;
    }
}

// Down products: an item is 16 columns of H and one of hparts shares of K, cut into parts; the wavefronts deal
// out the units (tile, part). The work-group's items are first, first + step, ... How K is cut goes by sizes
// alone, so that a token's bits do not go by what the others choose.
struct DownItems {
    int item, step, nitems;
    int hparts;
    __device__ __forceinline__ int n0() const { return item / hparts * 16; }
    __device__ __forceinline__ int share() const { return item % hparts; }
};

template <int WF, bool LDS>
struct DownWalk {
    struct Place {
        bool ends, item_ends, all, unit;  // unit: there is one, and these are its rows
        int row, n;
    };
    const FewArgs& a;
    const FewTables& t;
    DownItems items;
    int wave, parts, nch, nrows, units, lane;
    Operands<WF, 1> o;
    int unit, c, c1, row, n;
    bool stop;

    __device__ __forceinline__ DownWalk(const FewArgs& args, const FewTables& tab, const DownItems& list, int rows, int tiles,
                                        int wv, int ln)
        : a(args), t(tab), items(list), wave(wv), parts(args.parts), nch(chunks<WF, 1, LDS>(args.F)), nrows(rows),
          units(tiles * args.parts), lane(ln), stop(false) {
        enter_item();
    }
    __device__ __forceinline__ void enter_item() {
        unit = wave;
        if (unit < units) {
            enter_unit();
        } else {
            nothing();
        }
    }
    __device__ __forceinline__ void enter_unit() {
        const int tile = unit / parts, part = unit - tile * parts, e = __builtin_amdgcn_readfirstlane(t.tile_e[tile]);
        const int row0 = __builtin_amdgcn_readfirstlane(t.tile_row0[tile]);
        n = __builtin_amdgcn_readfirstlane(t.tile_n[tile]);
        row = part * nrows + row0;
        o.set(0, a.w_down, a.s_down, e, a.E + a.S, a.H, a.F, items.n0(), lane);
        const int r = lane % kTileRows<WF>, term = lane % 16 / kTileRows<WF>;
        o.template rows<LDS>(a.h, kTerms<WF> * nrows, r < n ? term * nrows + row0 + r : -1, a.F, lane);
        const int cut = items.share() * parts + part, cuts = items.hparts * parts;
        c = cut * nch / cuts;
        c1 = (cut + 1) * nch / cuts;
    }
    // no unit: a chunk past the end, from lines that everyone reads
    __device__ __forceinline__ void nothing() {
        o.set(0, a.w_down, a.s_down, 0, a.E + a.S, a.H, a.F, 0, lane);
        o.template rows<LDS>(a.h, kTerms<WF> * nrows, -1, a.F, lane);
        c = nch;
        c1 = nch + 1;
        row = 0;
        n = 0;
    }
    __device__ __forceinline__ Place place() const {
        const bool ends = c + 1 >= c1 && !stop, item_ends = ends && unit + kWaves >= units;
        return {ends, item_ends, item_ends && items.item + items.step >= items.nitems, unit < units, row, n};
    }
    __device__ __forceinline__ void next() {
        if (stop) return;
        if (c + 1 < c1) {
            ++c;
        } else if (unit + kWaves < units) {
            unit += kWaves;
            enter_unit();
        } else if (items.item + items.step < items.nitems) {
            items.item += items.step;
            enter_item();
        } else {
            nothing();
            stop = true;
        }
    }
};

// The last wavefront's part of a down item: the weighted sum, the shared mixture and the skip residual
// of 16 columns for every token, from the partial outputs y; shared between work-groups, the sum of
// their sums by the last of them.
template <int WF>
__device__ __forceinline__ void combine(const FewArgs& a, const Term* list, const DownItems& d, const float* y,
                                        int lane) {
    constexpr bool F32 = WF == YVMOE_W_F32;
    const int c = lane & 15, ns = a.N * a.k, n0 = d.n0(), parts = a.parts;
    const long long stride = (long long)a.N * a.H;
    const bool alone = d.hparts == 1;
    auto sum = [&](int first, int len) {  // eight terms under way
        float v = 0.0f;
#pragma unroll 1
        for (int i = 0; i < len; i += 8) {
            Term e[8];
            float p[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) e[j] = list[first + min(i + j, len - 1)];
#pragma unroll
            for (int j = 0; j < 8; ++j) p[j] = y[max(e[j].row, 0) * 16 + c];
#pragma unroll
            for (int j = 0; j < 8; ++j) v = i + j < len && e[j].row >= 0 ? __builtin_fmaf(e[j].w, p[j], v) : v;
        }
        return v;
    };
    auto write = [&](int tok, float v, float sh) {
        const long long at = (long long)tok * a.H + n0 + c;
        v = v + sh;
        if (a.skip != nullptr)
            v = v + 0.1f * (F32 ? ((const float*)a.skip)[at] : bf16_to_f32(((const unsigned short*)a.skip)[at]));
        if constexpr (F32) {
            ((float*)a.out)[at] = v;
            if (a.shared_out != nullptr) ((float*)a.shared_out)[at] = sh;
        } else {
            ((unsigned short*)a.out)[at] = f32_to_bf16_rne(v);
            if (a.shared_out != nullptr) ((unsigned short*)a.shared_out)[at] = f32_to_bf16_rne(sh);
        }
    };
#pragma unroll 1
    for (int tok = lane >> 4; tok < a.N; tok += 4) {
        const float v = sum(tok * a.k * parts, a.k * parts), sh = sum((ns + tok * a.S) * parts, a.S * parts);
        if (alone) {
            write(tok, v, sh);
        } else {
            float* p = a.hsum + 2 * d.share() * stride + (long long)tok * a.H + n0 + c;
            __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            __hip_atomic_store(p + stride, sh, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
    }
    if (alone) return;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    int before = 0;
    if (lane == 0)
        before = __hip_atomic_fetch_add(a.hcount + n0 / 16, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (__builtin_amdgcn_readfirstlane(before) != d.hparts - 1) return;
    for (int tok = lane >> 4; tok < a.N; tok += 4) {
        float pv[kFewParts], ps[kFewParts];
#pragma unroll
        for (int i = 0; i < kFewParts; ++i) {
            float* q = a.hsum + 2 * min(i, d.hparts - 1) * stride + (long long)tok * a.H + n0 + c;
            pv[i] = __hip_atomic_load(q, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            ps[i] = __hip_atomic_load(q + stride, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        float v = pv[0], sh = ps[0];
#pragma unroll
        for (int i = 1; i < kFewParts; ++i) {
            v = i < d.hparts ? v + pv[i] : v;
            sh = i < d.hparts ? sh + ps[i] : sh;
        }
        write(tok, v, sh);
    }
}

// LDS that h takes for the down product.
__host__ __device__ inline int h_bytes(int terms, int nrows, int bytes) {
    return (terms * nrows * (bytes + kRowPad) + 127) / 128 * 128;
}

template <int WF, bool LDSX, bool LDSH>
__global__ __launch_bounds__(kAllThreads, 3) void few_experts_kernel(FewArgs a) {
    constexpr int BYTES = WF == YVMOE_W_F32 ? 4 : 2;
    __shared__ FewTables t;
    __shared__ Term terms[kYRows];
    __shared__ __align__(128) char pool[kPoolBytes];
    static_assert(sizeof(FewLogits) <= kEndBytes && sizeof(f32x4[2][kWaves][2][64]) <= kEndBytes, "the end's room");
    FewLogits& lg = *(FewLogits*)(pool + kPoolBytes - kEndBytes);
    auto& red = *(f32x4(*)[2][kWaves][2][64])(pool + kPoolBytes - kEndBytes);
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = lane & 15, grid = gridDim.x;
    if constexpr (LDSX) stage_rows<false>(a.xo, a.N, a.H * BYTES, pool, wave, lane);
    few_routing<kTileRows<WF>>(a, t, lg, blockIdx.x == 0);
    if (a.N == 0) return;
    if constexpr (LDSX) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
    }
    const int ns = a.N * a.k;

    // gate/up: this work-group's items, then, if it waits long, the missing ones of others
    const int nfb = a.F / 16, nitems = t.ntiles * nfb;
    auto at = [&](int item, int& e, int& n0, int& row0, int& n, int& token) {
        const int tile = item / nfb;
        n0 = (item - tile * nfb) * 16;
        e = __builtin_amdgcn_readfirstlane(t.tile_e[tile]);
        row0 = __builtin_amdgcn_readfirstlane(t.tile_row0[tile]);
        n = __builtin_amdgcn_readfirstlane(t.tile_n[tile]);
        token = r < n ? t.slot[row0 + r] / a.k : -1;
    };
    // Work-groups with items: all, or so many that a few rounds come out even.
    const int rounds = (nitems + grid - 1) / grid;
    const int used = nitems > kOwnItems * grid ? grid : rounds > 0 ? (nitems + rounds - 1) / rounds : 0;
    const int handed = max(0, nitems - kOwnItems * used), hitems = a.H / 16 * a.hparts;
    if ((int)blockIdx.x >= used && (int)blockIdx.x >= hitems) return;
    const int ntiles = t.ntiles + a.S * ((a.N + kTileRows<WF> - 1) / kTileRows<WF>), nrows = ns + a.S * a.N;
    const DownItems down{(int)blockIdx.x, grid, hitems, a.hparts};
    const int yrows = nrows * a.parts;
    float* y = (float*)(pool + (LDSH ? h_bytes(kTerms<WF>, nrows, a.F * BYTES) : 0));
    auto stage_h = [&]() {
        if constexpr (LDSH) {
            stage_rows<true>(a.h, kTerms<WF> * nrows, a.F * BYTES, pool, wave, lane);
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();
        }
    };
    for (int share = blockIdx.x, own = 1;; own = 0) {
        if (share < used) {
            int* ahead = own && handed > 0 ? t.ahead : nullptr;
            const int done = gate_up<WF, true, LDSX>(a, at, GateUpItems{share, nitems, used, ahead, 0}, red, ahead,
                                                    a.signals + 32 * SIG_TICKET, pool, wave, lane);
            if (wave == kWaves) {
                // h is written through: once the stores are there, it may be said
                asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
                signal_done(a, share, used, max(0, done - kOwnItems), handed, lane);
            }
        }
        if ((int)blockIdx.x >= hitems) return;
        if (wave < kWaves) {
            typedef DownWalk<WF, LDSH> Walk;
            Walk w(a, t, down, nrows, ntiles, wave, lane);
            Ring<WF, 1, Walk, LDSH, true> ring;
            ring.start_weights(w, a.F / 64);  // no h is needed for these
            __syncthreads();
            share = __builtin_amdgcn_readfirstlane(t.help);
            if (share >= 0) continue;
            stage_h();
            ring.start_acts(w, a.F / 64);
            int it = 0;
            ring.run(w, pool, a.F / 64, [&](const typename Walk::Place& p, const f32x4 (&acc)[1]) {
                if (p.unit) {
                    f32x4 v = acc[0];
                    if constexpr (kTerms<WF> == 2)  // rows 8 .. 15 are the second terms'
#pragma unroll
                        for (int i = 0; i < 4; ++i) v[i] = v[i] + __shfl_xor(v[i], 32);
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (4 * (lane >> 4) + i < p.n)
                            y[((it & 1) * yrows + p.row + 4 * (lane >> 4) + i) * 16 + r] = v[i];
                }
                if (p.item_ends) {
                    __syncthreads();
                    ++it;
                }
            });
            return;
        }
        list_terms(a, t, terms, nrows, lane);
        const int m = nitems > 0 ? wait_done(a, used, lane) : WAIT_DONE;
        if (m == WAIT_GIVEN_UP)  // h is not all there: the work-group's columns are no numbers
            for (int i = lane; i < kYRows; i += 64) terms[i] = Term{__builtin_nanf(""), 0};
        if (lane == 0) t.help = m;
        __syncthreads();
        share = m;
        if (share >= 0) continue;
        stage_h();
        DownItems d = down;
        for (int it = 0; d.item < hitems; ++it, d.item += grid) {
            __syncthreads();
            combine<WF>(a, terms, d, y + (it & 1) * yrows * 16, lane);
        }
        return;
    }
}

// Parts of a share of K for each tile, so that the wavefronts that deal out the units end together: the fewest
// within 3 % of the least work of the busiest.
int few_parts(int tiles, int rows, int nch, int shares, int room) {
    int best = 1;
    double cost = 1e30;
    for (int q = 1; q == 1 || (q <= 32 && q * shares <= nch && q * rows <= room); ++q) {
        const double c = (double)ceil_div(tiles * q, kWaves) / q;
        if (c < 0.97 * cost) {
            best = q;
            cost = c;
        }
    }
    return best;
}

}  // namespace

// For tests: 1 makes a work-group help after one look (by default one that has waited a millisecond does), 2 has
// the waits given up at once, 0 is the default.
extern "C" void yvmoe_few_set_wait(int mode) {
    wait_mode = mode == 1 ? GO_ONE_LOOK : mode == 2 ? GO_NO_WAIT : 0;
}

int few_launch(const void* x, int act, int N, int k, const yvmoe_router* r, const void* rweights, int rweights_bf16,
               const int64_t* rindices, const yvmoe_expert_weights* w, const float* mix, const void* skip, void* out,
               void* shared_out, const yvmoe_routing* routing, int* invalid, char* ws, hipStream_t st) {
    const int E = w->num_routed, S = w->num_shared, H = w->hidden, F = w->ffn;
    const FewWs L = few_ws(N, k, E, S, H, F, w->format, act);
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
    a.xo = w->format == YVMOE_W_INT4 ? (const void*)(ws + L.xo) : x;
    a.signals = (unsigned*)(ws + L.signals);
    a.hparts = few_hparts(N, k, E, S, H, F, w->format);
    a.hcount = (int*)(ws + L.hcount);
    a.hsum = (float*)(ws + L.hsum);
    a.wait_mode = wait_mode;
    int front = (a.self ? a.ncols / 16 * a.nsplit : 0) + S * (F / 16);
    if (w->format == YVMOE_W_INT4) front = std::max(front, ceil_div(N * (H / 8), kAllThreads));
    // one work-group per CU (LDS has no room for a second), fewer where neither half has work for them
    const int items = std::max(std::min(N * k, E) * (F / 16), H / 16 * a.hparts);
    const int grid = N == 0 ? 1 : std::min(kGrid, items);
    const int esz = act == YVMOE_ACT_BF16 ? 2 : 4;
    const int nrows = N * (k + S);
    const bool ldsx = (long long)N * (H * esz + kRowPad) <= kPoolBytes - kEndBytes;
    const int terms = act == YVMOE_ACT_BF16 ? 2 : 1;
    const bool ldsh = ldsx && (long long)terms * nrows * (F * esz + kRowPad) + 128 <= kPoolBytes - 128 * nrows;
    const int room = std::min(kYRows, ldsh ? (kPoolBytes - h_bytes(terms, nrows, F * esz)) / 128 : kYRows);
    const int tiles = (int)few_tiles(N, k, E, 0) + S * ceil_div(N, 16 / terms);
#define YV_FEW(WFV)                                                                                       \
    do {                                                                                                  \
        a.parts = few_parts(tiles, nrows, ceil_div(F / 64, Wt<WFV>::DEPTH.unit(1, ldsh)), a.hparts, room); \
        if (N > 0) {                                                                                      \
            few_front_kernel<WFV><<<std::max(front, 1), kAllThreads, 0, st>>>(a);                         \
            YV_LAUNCH_CHECK("few_front");                                                                 \
        }                                                                                                 \
        if (ldsh) few_experts_kernel<WFV, true, true><<<grid, kAllThreads, 0, st>>>(a);                   \
        else if (ldsx) few_experts_kernel<WFV, true, false><<<grid, kAllThreads, 0, st>>>(a);             \
        else few_experts_kernel<WFV, false, false><<<grid, kAllThreads, 0, st>>>(a);                      \
        YV_LAUNCH_CHECK("few_experts");                                                                   \
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
