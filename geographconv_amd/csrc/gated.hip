// The gated dense block  H = act(X.Wg + bg) * (X.Wu + bu)  and its backward, over fp32, bf16 and 8-bit operands.
//
//   forward    [G | U] = X.[Wg | Wu] on the matrix pipe, the activation, the product and (for training) the kept G, U in the epilogue
//   backward   dG = dH * U * act'(G), dU = dH * act(G)                  one pass, with both bias gradients (gate_grad_kernel)
//              dX = dG.Wg^T + dU.Wu^T                                   one accumulator over both reductions
//              [dWg | dWu] = X^T.[dG | dU]                              one launch, X read once
//
// All three products run on ONE tiled kernel over bf16 TERMS: an fp32 value is the exact sum of three bf16 values, and a product of two
// fp32 matrices is the sum of its six largest cross products (the dropped ones are O(2^-24)), accumulated in fp32; a bf16 value is one term
// and so is an 8-bit checkpoint's (4 significant bits), so X^T.dG from a checkpoint costs three cross products instead of six and loses
// nothing on the way.  dG and dU of a bf16 block, formed in fp32, are two terms.  fp32 (and 8-bit) operands are written as terms side by side,
// [row][term][roundup64(cols)], by terms_kernel or by the pass that forms them; bf16 matrices whose rows are 16-byte aligned are read in place.
#include "gate.h"
#include "gemm_call.h"
#include "mx8.h"

#include <algorithm>

namespace geogcn {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

constexpr uint32_t kOob = 0x80000000u;

// ---- matrices -> their bf16 term planes: up to three of one storage type in one launch (grid.y) ----------------------------------------------
struct TermsJobs {
    int n;
    struct Job { MatIn src; int64_t total, ldo, plane; int F, qpr; uint16_t* out; } job[3];
};
template <int P, int TYPE>
__global__ __launch_bounds__(256) void terms_kernel(const TermsJobs jobs) {
    const TermsJobs::Job& j = jobs.job[blockIdx.y];
    for (int64_t q = (int64_t)blockIdx.x * 256 + threadIdx.x; q < j.total; q += (int64_t)gridDim.x * 256) {
        const int64_t r = q / j.qpr;
        const int c = (int)(q - r * j.qpr) * 4;
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
        if (c < j.F) x = mask4(mat_load4<TYPE>(j.src, r, c), c, j.F);
        uint2 t[P];
        bf16_terms4<P>(x, t);
#pragma unroll
        for (int p = 0; p < P; ++p) *reinterpret_cast<uint2*>(j.out + p * j.plane + r * j.ldo + c) = t[p];
    }
}

// ---- the tiled product ----------------------------------------------------------------------------------------------------------------------
// C[m][n] = sum_k A . B over bf16 term planes.  An operand is stored along k (rows = its output dimension, "k-contiguous") or across it (rows =
// k, "k-strided"): X is k-contiguous in the forward and k-strided in the weight gradient, W the other way round, so nothing is ever
// transposed in memory.  Stages of BK k-values go straight from global memory to LDS (16 bytes a lane, two to six buffers); a k-contiguous image is
// read as 16-byte fragments, a k-strided one through the transposing LDS read (4 k-values of a lane's own column).  Both images are
// permuted in 16-byte pieces so that the lanes of a read phase meet different banks.
// NSEG = 2: the block's columns are BN / 2 of B[0] and the same BN / 2 of B[1] -- a lane then owns g and u of one element.
// What bounds it: large products power and the barriers of the stages (8,192 x 2,048 -> 8,192 in bf16, 1.05 PFLOP/s: 1.8-2.1 GHz, the matrix pipe
// busy 52 % of the clocks, LDS 26 % and without conflicts, waves waiting 36 %), products of few tiles a load's latency per stage (9,475 x 300 ->
// 600 in fp32: matrix pipe 31 %, LDS 12 %).  Counters: profiles/gated_block_kernels.md.
struct TileArgs {
    int64_t M, N;                                     // rows of C, columns of each segment of C
    int n_mt, n_nt, nsplit, steps_per_split;
    int n_kseg;
    int64_t K[2];
    const uint16_t* A[2]; int64_t lda[2], planeA[2];
    const uint16_t* B[2]; int64_t ldb[2], planeB[2];
    // epilogue
    int mode, out_type, act;
    void* C[2]; int64_t ldc[2];
    int64_t nc[2], nck[2], ncols;                     // columns to write (N and the pads kept zero): of C, of what is kept in full, the most of all
    const float* bias[2];
    int keep;                                         // EPI_GATED: what is kept of G, U (0, GEOGCN_KEEP_FULL, GEOGCN_KEEP_MX8)
    void* keepP[2]; int64_t ldk[2]; uint8_t* keepS[2];
    float* W; int64_t ldw, segw;                      // EPI_SLAB: [split][M][ldw], segment q from column q * segw
};
enum { EPI_STORE = 0, EPI_SLAB = 1, EPI_GATED = 2 };

__device__ __forceinline__ void store_quad(void* C, int64_t ld, int type, int64_t row, int64_t col, const float (&x)[4]) {
    if (type == GEOGCN_T_F32)
        *reinterpret_cast<float4*>(static_cast<float*>(C) + row * ld + col) = make_float4(x[0], x[1], x[2], x[3]);
    else
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(C) + row * ld + col) = make_uint2(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]));
}

// One image: R output rows (or columns) by the BK k-values of a stage (one or two matrix instructions deep), one term.
template <bool STRIDED, int R, int BK>
struct Image {
    static constexpr int kBytes = R * BK * 2;
    static constexpr int kPieces = R * BK / 8;                       // 16-byte pieces
    static constexpr int kCpr = STRIDED ? R / 8 : BK / 8;            // pieces per stored row
    static_assert(kPieces % 64 == 0, "whole wave loads");
    // k-strided: the 32 bytes (two pieces) that four lanes read of a k-row lie at pair T ^ turn(k) of the row; a read phase meets k-rows lg*8 + 0..3
    // of two or four lane groups, and a stored row may be a whole round of the banks (R = 128) or less
    static constexpr bool kPow2 = (R & (R - 1)) == 0;
    static __device__ __forceinline__ int turn(int k) {
        if constexpr (!kPow2) return R % 32 == 0 ? (k >> 3) & 1 : 0;
        else if constexpr (R >= 128) return (k & 3) + 4 * ((k >> 3) & 1);
        else return ((k & 3) >> 1) + 2 * ((k >> 3) & 1);
    }
    static __device__ __forceinline__ int place(int c, int row) {   // where piece c of stored row `row` lies in that row (its own inverse)
        if constexpr (!STRIDED) return BK == 64 ? (c ^ (row & 7)) : (c ^ ((row >> 1) & 3));
        else return c ^ (2 * turn(row));
    }
    // byte offset, from the image's first row and k, of the piece that belongs at place `piece` of the image
    static __device__ __forceinline__ uint32_t source(int piece, int64_t ld) {
        const int row = piece / kCpr, c = place(piece - row * kCpr, row);
        return (uint32_t)row * (uint32_t)(ld * 2) + (uint32_t)c * 16u;
    }
    // k-contiguous: the first of the 8 k-values of a lane's piece -- the same in every wave load (64 pieces are whole rows, and whole rounds of `place`)
    static __device__ __forceinline__ int k_of_lane(int lane) { return place(lane % kCpr, lane / kCpr) * 8; }
    // Fragments: 16 output rows (tile T of the image) by 32 k-values (k-step s); lane (li, lg) gets its row's k-values s*32 + lg*8 .. + 7.
    // lane_base: the lane's byte address for T = 0, s = 0; images start on multiples of 1 KB, so the permutations are exclusive-ors on it.
    static __device__ __forceinline__ uint32_t lane_base(int li, int lg) {
        if constexpr (!STRIDED) return (uint32_t)(li * (BK * 2) + place(lg, li) * 16);
        else {
            const int k = lg * 8 + (li >> 2);
            return (uint32_t)(k * (R * 2) + turn(k) * 32 + ((li & 3) >> 1) * 16 + (li & 1) * 8);
        }
    }
    static __device__ __forceinline__ bf16x8 read(uint32_t base, int T, int s, int lg) {
        if constexpr (!STRIDED) {
            typedef __attribute__((address_space(3))) const bf16x8* lds8;
            return *(lds8)(uintptr_t)((base ^ (uint32_t)(s * 64)) + (uint32_t)(T * 16 * BK * 2));
        } else {
            typedef __attribute__((address_space(3))) s16x4* lds4;
            // (R = 80, 160: the row's length has bits of its own where T does; there turn is one bit, and T ^ turn is T +- turn)
            const int t1 = R % 32 == 0 ? lg & 1 : 0;
            const uint32_t a = kPow2 ? (base ^ (uint32_t)(T * 32)) : base + (uint32_t)(T * 32) - ((T & 1) ? (uint32_t)(t1 * 64) : 0u);
            const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(uintptr_t)(a + (uint32_t)(s * 32 * R * 2)));
            const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(uintptr_t)(a + (uint32_t)((s * 32 + 4) * R * 2)));       // (turn(k + 4) == turn(k))
            return bf16x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
        }
    }
};

// 64 lanes x 16 bytes from global memory to LDS (lane i's to lds + 16 i).  As assembly, so that the compiler, which cannot tell the buffer being
// filled from the one being read, does not wait for these loads at every LDS read: the waits stand at the stage's barrier (stage_barrier).  M0 is
// set and used inside the statement; nothing else in these kernels uses it.
typedef int i32x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ void load_to_lds(i32x4 rsrc, uint32_t voff, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(lds), "v"(voff), "s"(rsrc) : "memory");
}
// all but the newest LEFT of this wave's loads to LDS have landed, its LDS reads are done, and so they are in every wave of the block
template <int LEFT>
__device__ __forceinline__ void stage_barrier() {
    static_assert(LEFT < 64, "vmcnt");
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"i"(LEFT) : "memory");
}
// where an operand is read: the address of its first row and k of the stage, and the bytes from there to the matrix' end (reads behind: zeros)
struct Cursor {
    uint64_t p;
    int64_t left;
    __device__ __forceinline__ void set(const uint16_t* base, int64_t offset, int64_t total) {
        p = reinterpret_cast<uint64_t>(base) + (uint64_t)offset * 2;
        left = (total - offset) * 2;
    }
    __device__ __forceinline__ void advance(int64_t bytes) { p += (uint64_t)bytes; left -= bytes; }
    __device__ __forceinline__ i32x4 rsrc() const {
        const int n = left <= 0 ? 0 : left > 0x7FFFFFFFll ? 0x7FFFFFFF : (int)left;
        return i32x4{__builtin_amdgcn_readfirstlane((int)(uint32_t)p), __builtin_amdgcn_readfirstlane((int)(uint32_t)(p >> 32)),
                     __builtin_amdgcn_readfirstlane(n), 0x00020000};
    }
};

template <int PA, int PB, bool ASTR, bool BSTR, int NSEG, int BM, int BN, int BK, int WM, int WN, int ST, bool GATED>
__global__ __launch_bounds__(WM* WN * 64) void tile_kernel(const TileArgs a) {
    constexpr int NW = WM * WN;
    constexpr int BNS = BN / NSEG;                            // columns of a segment
    typedef Image<ASTR, BM, BK> IA;
    typedef Image<BSTR, BNS, BK> IB;
    constexpr int MT = BM / WM / 16;                          // 16-row tiles of a wave
    // columns: in the gated product a wave owns CW columns of both segments, otherwise the waves of a row share the segments out among them
    constexpr bool PAIR = GATED || NSEG == 1;
    constexpr int WNS = PAIR ? WN : WN / 2;                   // waves side by side over a segment
    constexpr int CW = BNS / WNS, NTS = CW / 16, NT = GATED ? NTS * 2 : NTS;
    static_assert(BM % (WM * 16) == 0 && CW % 16 == 0 && BNS % WNS == 0 && (PAIR || WN % 2 == 0) && (!GATED || (NSEG == 2 && CW % 32 == 0)), "wave tiles");
    constexpr int kA = PA * IA::kBytes, kStage = kA + PB * NSEG * IB::kBytes;
    constexpr int LIA = IA::kPieces / 64, LIB = IB::kPieces / 64;                   // wave loads of an image
    constexpr int TA = PA * LIA, TB = PB * LIB * NSEG;                              // ... of a stage
    constexpr int LA = (TA + NW - 1) / NW, LB = (TB + NW - 1) / NW;                 // ... of a stage, per wave (at most)
    static_assert(ST == 2 || (TA % NW == 0 && TB % NW == 0), "a wait that leaves loads open counts on every wave having asked for as many");
    extern __shared__ __attribute__((aligned(128))) unsigned char lds[];
    const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int li = lane & 15, lg = lane >> 4, wm = wid / WN, wn = PAIR ? wid % WN : wid % WN % WNS, wseg = PAIR ? 0 : wid % WN / WNS;

    // tile of this block: every XCD works on a run of neighbouring tiles (blocks go round the XCDs one by one), taken in groups of 8 row tiles
    // so that the operands of the tiles in flight fit that XCD's L2
    const int tiles = a.n_mt * a.n_nt, total = tiles * a.nsplit;
    int id;
    {
        const int x = blockIdx.x % kNumXCD, q = total / kNumXCD, r = total % kNumXCD;
        id = x * q + min(x, r) + (int)blockIdx.x / kNumXCD;
    }
    const int z = id / tiles;
    id -= z * tiles;
    const int grp = id / (8 * a.n_nt), first = grp * 8, rows_in = min(8, a.n_mt - first), in = id - grp * 8 * a.n_nt;
    const int mt = first + in % rows_in, nt = in / rows_in;
    const int64_t m0 = (int64_t)mt * BM, n0 = (int64_t)nt * BNS;

    const int ns0 = (int)((a.K[0] + BK - 1) / BK), nsteps = max(1, ns0 + (a.n_kseg == 2 ? (int)((a.K[1] + BK - 1) / BK) : 0));      // (no k at all: one stage of zeros)
    const int t0 = z * a.steps_per_split, t1 = min(nsteps, t0 + a.steps_per_split);

    f32x4 acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

    // this wave's loads of a stage: LA pieces of A's images, LB of B's (both segments'), 64 x 16 bytes each
    uint32_t va[LA], vb[LB];
    const int ka = IA::k_of_lane(lane), kb = IB::k_of_lane(lane);
    Cursor ca, cb[NSEG];
    int64_t k_left;
    auto seg_of = [&](int i) __attribute__((always_inline)) {                // the segment of B that this wave's load i belongs to
        if constexpr (NSEG == 1) return 0;
        else if constexpr (PB * LIB % NW == 0) return i / (PB * LIB / NW);
        else return i * NW + wid >= PB * LIB ? 1 : 0;
    };
    auto start = [&](int ks, int step) __attribute__((always_inline)) {      // cursors at stage `step` of reduction segment ks
        const int64_t k0 = (int64_t)step * BK, K = a.K[ks];
        const int64_t lda = a.lda[ks];
        k_left = K - k0;
        if constexpr (ASTR) ca.set(a.A[ks], k0 * lda + m0, K * lda);
        else ca.set(a.A[ks], m0 * lda + k0, a.M * lda);
#pragma unroll
        for (int q = 0; q < NSEG; ++q) {
            const int w = NSEG == 2 ? q : ks;
            const int64_t ldb = a.ldb[w];
            if constexpr (BSTR) cb[q].set(a.B[w], k0 * ldb + n0, K * ldb);
            else cb[q].set(a.B[w], n0 * ldb + k0, a.N * ldb);
        }
#pragma unroll
        for (int i = 0; i < LA; ++i) {
            const int l = i * NW + wid, p = l / LIA;
            va[i] = IA::source((l - p * LIA) * 64 + lane, lda) + (uint32_t)(p * a.planeA[ks] * 2);
        }
#pragma unroll
        for (int i = 0; i < LB; ++i) {
            const int q = seg_of(i), l = i * NW + wid - q * (PB * LIB), p = l / LIB;
            const int64_t ldb = NSEG == 2 ? (q ? a.ldb[1] : a.ldb[0]) : a.ldb[ks];
            vb[i] = IB::source((l - p * LIB) * 64 + lane, ldb) + (uint32_t)(p * a.planeB[NSEG == 2 ? 0 : ks] * 2);
        }
    };
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)lds + (uint32_t)wid * 1024u;
    int next = t0, fill = 0;                                  // the stage to load next, and the buffer that it goes to
    auto issue = [&]() __attribute__((always_inline)) {
        if (a.n_kseg == 2 && next == ns0) start(1, 0);
        const i32x4 ra = ca.rsrc();
        i32x4 rb[NSEG];
#pragma unroll
        for (int q = 0; q < NSEG; ++q) rb[q] = cb[q].rsrc();
        const uint32_t to = lds0 + (uint32_t)(fill * kStage);
        const bool tail = k_left < BK;                        // (k-strided rows behind the last are behind the matrix' end; k-contiguous ones are not)
#pragma unroll
        for (int i = 0; i < LA; ++i) {
            uint32_t v = va[i];
            if (!ASTR && tail) v = ka < k_left ? v : kOob;
            if (TA % NW != 0 && i * NW + wid >= TA) continue;
            load_to_lds(ra, v, to + (uint32_t)(i * NW * 1024));
        }
#pragma unroll
        for (int i = 0; i < LB; ++i) {
            uint32_t v = vb[i];
            if (!BSTR && tail) v = kb < k_left ? v : kOob;
            if (TB % NW != 0 && i * NW + wid >= TB) continue;
            load_to_lds(NSEG == 1 || seg_of(i) == 0 ? rb[0] : rb[NSEG - 1], v, to + (uint32_t)(kA + i * NW * 1024));
        }
        const int ks = a.n_kseg == 2 && next >= ns0 ? 1 : 0;
        ca.advance(ASTR ? (int64_t)BK * 2 * a.lda[ks] : BK * 2);
#pragma unroll
        for (int q = 0; q < NSEG; ++q) cb[q].advance(BSTR ? (int64_t)BK * 2 * a.ldb[NSEG == 2 ? q : ks] : BK * 2);
        k_left -= BK;
        ++next;
        fill = fill + 1 == ST ? 0 : fill + 1;
    };

    if (a.n_kseg == 2 && t0 > ns0) start(1, t0 - ns0);
    else start(0, t0);                                        // (t0 == ns0: issue() starts the second segment)

    // Two phases a stage (BK = 32: the first and the second half of the wave's columns; BK = 64: of the k-values), with the stage's barrier BETWEEN
    // them: the second phase's fragments are read while the first one's products run, so at the barrier this stage's buffer is free -- the stage ST further on is asked for at
    // once -- and the next stage's first fragments are read while the second phase's products run.  No product waits for an LDS read that
    // was not issued a phase ahead.  At BK = 32 A is held once: in the second phase its fragments are refilled in the order in which they are
    // used up.
    // Operands swapped, so that a lane owns 4 consecutive columns of one row of C; cross products of three terms from the small ones up.
#define GEOGCN_MFMA(A_, B_, J0, i, j, pa, pb) acc[i][J0 + j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(B_[j][pb], A_[i][pa], acc[i][J0 + j], 0, 0, 0);
#define GEOGCN_TERM(A_, B_, J0, JN, pa, pb) \
    _Pragma("unroll") for (int i = 0; i < MT; ++i) _Pragma("unroll") for (int j = 0; j < JN; ++j) GEOGCN_MFMA(A_, B_, J0, i, j, pa, pb)
#define GEOGCN_TERMS(A_, B_, J0, JN, REFILL)                                                                                               \
    if constexpr (PA == 3) {                                                                                                           \
        GEOGCN_TERM(A_, B_, J0, JN, 2, 0) _Pragma("unroll") for (int i = 0; i < MT; ++i) { REFILL(i, 2) }                                  \
        GEOGCN_TERM(A_, B_, J0, JN, 1, 1) GEOGCN_TERM(A_, B_, J0, JN, 1, 0) _Pragma("unroll") for (int i = 0; i < MT; ++i) { REFILL(i, 1) }    \
        GEOGCN_TERM(A_, B_, J0, JN, 0, 2) GEOGCN_TERM(A_, B_, J0, JN, 0, 1)                                                                    \
        _Pragma("unroll") for (int i = 0; i < MT; ++i) {                                                                               \
            _Pragma("unroll") for (int j = 0; j < JN; ++j) GEOGCN_MFMA(A_, B_, J0, i, j, 0, 0)                                         \
            REFILL(i, 0)                                                                                                               \
        }                                                                                                                              \
    } else if constexpr (PA == 2) {                                                                                                    \
        GEOGCN_TERM(A_, B_, J0, JN, 1, 0) _Pragma("unroll") for (int i = 0; i < MT; ++i) { REFILL(i, 1) }                                  \
        _Pragma("unroll") for (int i = 0; i < MT; ++i) {                                                                               \
            _Pragma("unroll") for (int j = 0; j < JN; ++j) GEOGCN_MFMA(A_, B_, J0, i, j, 0, 0)                                         \
            REFILL(i, 0)                                                                                                               \
        }                                                                                                                              \
    } else {                                                                                                                           \
        _Pragma("unroll") for (int i = 0; i < MT; ++i) {                                                                               \
            _Pragma("unroll") for (int pb = PB - 1; pb >= 0; --pb) _Pragma("unroll") for (int j = 0; j < JN; ++j) GEOGCN_MFMA(A_, B_, J0, i, j, 0, pb) \
            REFILL(i, 0)                                                                                                               \
        }                                                                                                                              \
    }
#define GEOGCN_NO_REFILL(i, p)
#define GEOGCN_REFILL(i, p) fa[i][p] = IA::read(la + at + (uint32_t)((p) * IA::kBytes), wm * MT + i, 0, lg);
    constexpr bool BYK = BK == 64;
    static_assert(BK == 32 || (PA == 1 && PB == 1), "two k-steps a stage: one term");
    static_assert(PA == PB || PA == 1 || (PA == 2 && PB == 1), "cross products");
    constexpr int N0 = BYK ? NT : (NT + 1) / 2, N1 = BYK ? NT : NT - N0, J1 = BYK ? 0 : N0;       // columns of the two phases, in tiles
    bf16x8 fa[MT][PA], fa1[BYK ? MT : 1][PA], b0[N0][PB], b1[N1][PB];
    const uint32_t lds_at = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)lds;
    const uint32_t la = lds_at + IA::lane_base(li, lg), lb = lds_at + kA + IB::lane_base(li, lg) + (uint32_t)(PAIR ? 0 : wseg * PB * IB::kBytes);
    uint32_t at = 0;                                          // the buffer of the stage at hand
    auto read_b = [&](auto& f, int s, int j0, int n) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < n; ++j)
#pragma unroll
            for (int p = 0; p < PB; ++p)
                f[j][p] = IB::read(lb + at + (uint32_t)(((PAIR ? (j0 + j) / NTS : 0) * PB + p) * IB::kBytes), wn * NTS + (j0 + j) % NTS, s, lg);
    };
    auto second = [&]() __attribute__((always_inline)) {      // the second phase's fragments
        if constexpr (BYK) {
#pragma unroll
            for (int i = 0; i < MT; ++i) fa1[i][0] = IA::read(la + at, wm * MT + i, 1, lg);
        }
        read_b(b1, BYK ? 1 : 0, J1, N1);
    };
#pragma unroll
    for (int i = 0; i < ST; ++i) {
        if (i == ST - 1) {                                    // the first stage has landed (its buffer is not the one asked for next)
            if (t0 + ST - 1 <= t1) stage_barrier<(ST - 2) * (LA + LB)>();
            else stage_barrier<0>();
        }
        if (next < t1) issue();
    }
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int p = 0; p < PA; ++p) { GEOGCN_REFILL(i, p) }
    read_b(b0, 0, 0, N0);
#pragma unroll 1
    for (int t = t0; t + 1 < t1; ++t) {
        second();
        GEOGCN_TERMS(fa, b0, 0, N0, GEOGCN_NO_REFILL)
        // stage t + 1 has landed: of the stages asked for so far, up to t + ST - 1, the ones behind it may be on their way
        if (t + ST <= t1) stage_barrier<(ST - 2) * (LA + LB)>();
        else stage_barrier<0>();
        if (next < t1) issue();
        at = at + kStage == ST * kStage ? 0 : at + kStage;
        // (opaque: addresses are formed where they are used instead of living in registers across the loop)
        asm volatile("" : "+s"(at));
        read_b(b0, 0, 0, N0);
        if constexpr (BYK) {
#pragma unroll
            for (int i = 0; i < MT; ++i) { GEOGCN_REFILL(i, 0) }
            GEOGCN_TERMS(fa1, b1, J1, N1, GEOGCN_NO_REFILL)
        } else {
            GEOGCN_TERMS(fa, b1, J1, N1, GEOGCN_REFILL)
        }
    }
    second();
    GEOGCN_TERMS(fa, b0, 0, N0, GEOGCN_NO_REFILL)
    if constexpr (BYK) { GEOGCN_TERMS(fa1, b1, J1, N1, GEOGCN_NO_REFILL) }
    else { GEOGCN_TERMS(fa, b1, J1, N1, GEOGCN_NO_REFILL) }
#undef GEOGCN_REFILL
#undef GEOGCN_NO_REFILL
#undef GEOGCN_TERMS
#undef GEOGCN_TERM
#undef GEOGCN_MFMA

    // ---- epilogue ----
    if constexpr (GATED) {
        if (a.mode == EPI_GATED) {
            // (all biases before the first store: a load behind stores would wait for them)
            float bias[2][NTS][4];
#pragma unroll
            for (int q = 0; q < 2; ++q)
#pragma unroll
                for (int j = 0; j < NTS; ++j) {
                    const int64_t col = n0 + wn * CW + j * 16 + lg * 4;
                    const float4 b = col < a.N ? load_bias4(a.bias[q], (int)col, (int)a.N, aligned16(a.bias[q])) : make_float4(0.f, 0.f, 0.f, 0.f);
                    bias[q][j][0] = b.x; bias[q][j][1] = b.y; bias[q][j][2] = b.z; bias[q][j][3] = b.w;
                }
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                const int64_t row = m0 + (wm * MT + i) * 16 + li;
#pragma unroll
                for (int jj = 0; jj < NTS; jj += 2) {
                    float v[2][2][4];                         // [g, u][16-column tile][column]: 32 columns = one block of a checkpoint
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int64_t col = n0 + wn * CW + (jj + h) * 16 + lg * 4;
#pragma unroll
                        for (int q = 0; q < 2; ++q)
#pragma unroll
                            for (int r = 0; r < 4; ++r) v[q][h][r] = col + r < a.N ? acc[i][q * NTS + jj + h][r] + bias[q][jj + h][r] : 0.f;
                    }
                    if (row < a.M) {
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const int64_t col = n0 + wn * CW + (jj + h) * 16 + lg * 4;
                            if (col < a.nc[0]) {
                                float x[4];
#pragma unroll
                                for (int r = 0; r < 4; ++r) x[r] = col + r < a.N ? gate_value(a.act, v[0][h][r]) * v[1][h][r] : 0.f;
                                store_quad(a.C[0], a.ldc[0], a.out_type, row, col, x);
                            }
                            if (a.keep == GEOGCN_KEEP_FULL) {
                                if (col < a.nck[0]) store_quad(a.keepP[0], a.ldk[0], a.out_type, row, col, v[0][h]);
                                if (col < a.nck[1]) store_quad(a.keepP[1], a.ldk[1], a.out_type, row, col, v[1][h]);
                            }
                        }
                    }
                    if (a.keep == GEOGCN_KEEP_MX8) {
                        const int64_t c0 = n0 + wn * CW + jj * 16;
#pragma unroll
                        for (int q = 0; q < 2; ++q) {
                            uint32_t m = 0;
#pragma unroll
                            for (int h = 0; h < 2; ++h)
#pragma unroll
                                for (int r = 0; r < 4; ++r) m = max(m, mx8_abs_bits(v[q][h][r]));
                            m = max(m, (uint32_t)__shfl_xor((int)m, 16));
                            m = max(m, (uint32_t)__shfl_xor((int)m, 32));
                            const uint32_t b = mx8_scale_byte(m);
                            const float inv = mx8_inv_scale(b);
                            if (row < a.M && c0 < a.N) {
                                uint8_t* codes = static_cast<uint8_t*>(a.keepP[q]) + row * a.ldk[q] + c0;
#pragma unroll
                                for (int h = 0; h < 2; ++h)
                                    *reinterpret_cast<uint32_t*>(codes + h * 16 + lg * 4) =
                                        mx8_encode4(v[q][h][0], v[q][h][1], v[q][h][2], v[q][h][3], inv, b != 255u);
                                if (lg == 0) a.keepS[q][row * (a.ldk[q] / kMxBlock) + c0 / kMxBlock] = (uint8_t)b;
                            }
                        }
                    }
                }
            }
            return;
        }
    }
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        const int64_t row = m0 + (wm * MT + i) * 16 + li;
        if (row >= a.M) continue;
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            const int q = PAIR ? j / NTS : wseg;
            const int64_t col = n0 + wn * CW + (j % NTS) * 16 + lg * 4;
            float x[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) x[r] = col + r < a.N ? acc[i][j][r] : 0.f;
            if (a.mode == EPI_SLAB) {
                if (col < a.segw) *reinterpret_cast<float4*>(a.W + ((int64_t)z * a.M + row) * a.ldw + q * a.segw + col) = make_float4(x[0], x[1], x[2], x[3]);
            } else if (col < (q ? a.nc[1] : a.nc[0])) {
                store_quad(a.C[q], a.ldc[q], a.out_type, row, col, x);
            }
        }
    }
}

// ---- a few rows (a served token): the weights' bytes are all there is to move -----------------------------------------------------------------
// A block takes 32 columns of both weights over the whole reduction; its 512 threads read 16 bytes (VEC values) of each weight a step, CL lanes
// side by side over the columns, KS k-rows at a time, straight from the matrices (no term planes: products are fp32 fmas of the stored
// values).  x lies in LDS as [k][row].  The partial sums meet in two rotations within 16 lanes and then in LDS, always in the same order.
// 32 columns are one checkpoint block of a row.  Bound by the latency of one round of loads and the reduction: 1 x 1024 -> 4096 in bf16 (16.8 MB)
// 6.4-7.1 us = 2.4-2.6 TB/s (8.5 + 4.8 us by tiles and a split).
struct FewArgs {
    int64_t M, ldx, ldwg, ldwu, ncols, nck[2];        // (columns to write of H and of what is kept in full)
    int K, N, act, out_type, keep;
    const void *X, *Wg, *Wu;
    const float* bias[2];
    void* H; int64_t ldh;
    void* keepP[2]; int64_t ldk[2]; uint8_t* keepS[2];
};
template <int BYTES> struct Raw { typedef uint4 type; };
template <> struct Raw<8> { typedef uint2 type; };
__device__ __forceinline__ void values_of(const uint4& w, float (&v)[4]) {                    // four fp32 values
    v[0] = __uint_as_float(w.x); v[1] = __uint_as_float(w.y); v[2] = __uint_as_float(w.z); v[3] = __uint_as_float(w.w);
}
__device__ __forceinline__ void values_of(const uint2& w, float (&v)[4]) { v[0] = bf16_lo(w.x); v[1] = bf16_hi(w.x); v[2] = bf16_lo(w.y); v[3] = bf16_hi(w.y); }
__device__ __forceinline__ void values_of(const uint4& w, float (&v)[8]) {                    // eight bf16 values
    v[0] = bf16_lo(w.x); v[1] = bf16_hi(w.x); v[2] = bf16_lo(w.y); v[3] = bf16_hi(w.y);
    v[4] = bf16_lo(w.z); v[5] = bf16_hi(w.z); v[6] = bf16_lo(w.w); v[7] = bf16_hi(w.w);
}
__device__ __forceinline__ float add_rotated(float v, int by8) {        // v + the value `8` (`4`) lanes on within each 16
    const int x = __float_as_int(v);
    return v + __int_as_float(by8 ? __builtin_amdgcn_mov_dpp(x, 0x128, 0xf, 0xf, true) : __builtin_amdgcn_mov_dpp(x, 0x124, 0xf, 0xf, true));
}
template <typename T, int VEC, int RM>
__global__ __launch_bounds__(512) void few_rows_kernel(const FewArgs a) {
    constexpr int CL = 32 / VEC, KS = 512 / CL, KC = 1024, IT = KC / KS;
    constexpr int U = RM <= 2 ? 8 : RM == 4 ? 4 : VEC == 8 ? 2 : 4;      // steps whose loads are in flight together (registers)
    static_assert(IT % U == 0 && (CL == 4 || CL == 8), "layout");
    constexpr int LDS_F = KC * RM > 32 * 64 * RM ? KC * RM : 32 * 64 * RM;
    __shared__ __attribute__((aligned(16))) float lds[LDS_F];
    const int tid = threadIdx.x, cl = tid % CL, ks = tid / CL, col = blockIdx.x * 32 + cl * VEC;
    const int64_t row0 = (int64_t)blockIdx.y * RM;
    typedef typename Raw<VEC * sizeof(T)>::type raw;
    // (columns and k-rows outside are read from inside -- the first columns, the last row -- and count as zeros)
    const int at = col < a.N ? col : 0;
    const T *Wg = static_cast<const T*>(a.Wg) + at, *Wu = static_cast<const T*>(a.Wu) + at, *X = static_cast<const T*>(a.X);
    float acc[2][RM][VEC];
#pragma unroll
    for (int q = 0; q < 2; ++q)
#pragma unroll
        for (int r = 0; r < RM; ++r)
#pragma unroll
            for (int v = 0; v < VEC; ++v) acc[q][r][v] = 0.f;
    for (int kb = 0; kb < a.K; kb += KC) {
        raw wg[U], wu[U];
        auto fetch = [&](int it) __attribute__((always_inline)) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int64_t k = min(kb + (it + u) * KS + ks, a.K - 1);
                wg[u] = *reinterpret_cast<const raw*>(Wg + k * a.ldwg);
                wu[u] = *reinterpret_cast<const raw*>(Wu + k * a.ldwu);
            }
        };
        fetch(0);                                             // (asked for before x is staged: both latencies at once)
        const int here = min(KC, a.K - kb), staged = min(KC, (here + U * KS - 1) / (U * KS) * (U * KS));
        for (int k = tid; k < staged; k += 512) {
#pragma unroll
            for (int r = 0; r < RM; ++r) {
                const int64_t row = row0 + r;
                float x = 0.f;
                if (row < a.M && k < here) {
                    if constexpr (sizeof(T) == 4) x = X[row * a.ldx + kb + k];
                    else x = __uint_as_float((uint32_t)X[row * a.ldx + kb + k] << 16);
                }
                lds[k * RM + r] = x;
            }
        }
        __syncthreads();
        for (int it = 0; it * KS < here; it += U) {
            if (it) fetch(it);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int k = (it + u) * KS + ks;
                const float* x = lds + k * RM;
                float g[VEC], w[VEC];
                values_of(wg[u], g);
                values_of(wu[u], w);
                if (it * KS + U * KS > here) {               // (a step that reaches behind the last row: zeros, whatever that row holds)
#pragma unroll
                    for (int v = 0; v < VEC; ++v) { g[v] = k < here ? g[v] : 0.f; w[v] = k < here ? w[v] : 0.f; }
                }
#pragma unroll
                for (int r = 0; r < RM; ++r)
#pragma unroll
                    for (int v = 0; v < VEC; ++v) {
                        acc[0][r][v] = fmaf(x[r], g[v], acc[0][r][v]);
                        acc[1][r][v] = fmaf(x[r], w[v], acc[1][r][v]);
                    }
            }
        }
        __syncthreads();
    }
    // 16 lanes hold 16 / CL k-rows of the same columns; the 32 groups of 16 meet in LDS as [group][q][row][column]
#pragma unroll
    for (int q = 0; q < 2; ++q)
#pragma unroll
        for (int r = 0; r < RM; ++r)
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                float s = acc[q][r][v];
                if constexpr (CL == 4) s = add_rotated(s, 0);
                s = add_rotated(s, 1);
                if ((tid & 15) < CL) lds[((tid >> 4) * 2 + q) * (RM * 32) + r * 32 + cl * VEC + v] = s;
            }
    __syncthreads();
    for (int e = tid; e < RM * 32; e += 512) {
        const int r = e >> 5, c = blockIdx.x * 32 + (e & 31);
        const int64_t row = row0 + r;
        float s[2];
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            float p[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int g = 0; g < 32; ++g) p[g & 3] += lds[(g * 2 + q) * (RM * 32) + e];
            s[q] = c < a.N ? (p[0] + p[1]) + (p[2] + p[3]) + (a.bias[q] ? a.bias[q][c] : 0.f) : 0.f;
        }
        const float h = c < a.N ? gate_value(a.act, s[0]) * s[1] : 0.f;
        auto put = [&](void* p, int64_t ld, float x) __attribute__((always_inline)) {
            if (a.out_type == GEOGCN_T_F32) static_cast<float*>(p)[row * ld + c] = x;
            else static_cast<uint16_t*>(p)[row * ld + c] = (uint16_t)(pack_bf16(x, 0.f) & 0xffffu);
        };
        const bool in = row < a.M;
        if (in && c < a.ncols) put(a.H, a.ldh, h);
        if (a.keep == GEOGCN_KEEP_FULL) {
            if (in && c < a.nck[0]) put(a.keepP[0], a.ldk[0], s[0]);
            if (in && c < a.nck[1]) put(a.keepP[1], a.ldk[1], s[1]);
        }
        if (a.keep == GEOGCN_KEEP_MX8) {
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                uint32_t m = mx8_abs_bits(s[q]);
#pragma unroll
                for (int d = 1; d < 32; d <<= 1) m = max(m, (uint32_t)__shfl_xor((int)m, d));
                const uint32_t b = mx8_scale_byte(m);
                if (in && blockIdx.x * 32 < a.N) {
                    static_cast<uint8_t*>(a.keepP[q])[row * a.ldk[q] + c] = (uint8_t)mx8_encode4(s[q], 0.f, 0.f, 0.f, mx8_inv_scale(b), b != 255u);
                    if ((e & 31) == 0) a.keepS[q][row * (a.ldk[q] / kMxBlock) + blockIdx.x] = (uint8_t)b;
                }
            }
        }
    }
}

// ---- partial products of a split reduction, added in split order, and the epilogue that they were waiting for ---------------------------
struct FinishArgs {
    int64_t M, N, segw, ldw, nc[2], nck[2];           // (TileArgs)
    int nsplit, nseg, mode, out_type, act, keep;
    const float* W;
    void* C[2]; int64_t ldc[2];
    const float* bias[2];
    void* keepP[2]; int64_t ldk[2]; uint8_t* keepS[2];
};
__global__ __launch_bounds__(256) void finish_kernel(const FinishArgs a) {
    // quads of columns; in the gated epilogue whole checkpoint blocks of 8 lanes stay together (segw is a multiple of 32)
    const int64_t qpr = a.segw / 4, total = a.M * qpr;
    for (int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x; e < total; e += (int64_t)gridDim.x * 256) {
        const int64_t row = e / qpr, col = (e - row * qpr) * 4;
        float v[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            if (q >= a.nseg) break;
            const float* w = a.W + row * a.ldw + q * a.segw + col;
            const int64_t zs = a.M * a.ldw;
            int z = 0;
            for (; z + 8 <= a.nsplit; z += 8) {               // eight loads in flight, added in order
                float4 t[8];
#pragma unroll
                for (int u = 0; u < 8; ++u) t[u] = *reinterpret_cast<const float4*>(w + (z + u) * zs);
#pragma unroll
                for (int u = 0; u < 8; ++u) { v[q][0] += t[u].x; v[q][1] += t[u].y; v[q][2] += t[u].z; v[q][3] += t[u].w; }
            }
            for (; z < a.nsplit; ++z) {
                const float4 t = *reinterpret_cast<const float4*>(w + z * zs);
                v[q][0] += t.x; v[q][1] += t.y; v[q][2] += t.z; v[q][3] += t.w;
            }
        }
        if (a.mode != EPI_GATED) {
            for (int q = 0; q < a.nseg; ++q)
                if (col < a.nc[q]) store_quad(a.C[q], a.ldc[q], a.out_type, row, col, v[q]);
            continue;
        }
#pragma unroll
        for (int q = 0; q < 2; ++q)
#pragma unroll
            for (int r = 0; r < 4; ++r) v[q][r] = col + r < a.N ? v[q][r] + (a.bias[q] ? a.bias[q][col + r] : 0.f) : 0.f;
        if (col < a.nc[0]) {
            float x[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) x[r] = col + r < a.N ? gate_value(a.act, v[0][r]) * v[1][r] : 0.f;
            store_quad(a.C[0], a.ldc[0], a.out_type, row, col, x);
        }
        if (a.keep == GEOGCN_KEEP_FULL) {
#pragma unroll
            for (int q = 0; q < 2; ++q)
                if (col < a.nck[q]) store_quad(a.keepP[q], a.ldk[q], a.out_type, row, col, v[q]);
        }
        if (a.keep == GEOGCN_KEEP_MX8) {
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                uint32_t m = max(max(mx8_abs_bits(v[q][0]), mx8_abs_bits(v[q][1])), max(mx8_abs_bits(v[q][2]), mx8_abs_bits(v[q][3])));
                m = max(m, (uint32_t)__shfl_xor((int)m, 1));
                m = max(m, (uint32_t)__shfl_xor((int)m, 2));
                m = max(m, (uint32_t)__shfl_xor((int)m, 4));
                const uint32_t b = mx8_scale_byte(m);
                if (col / kMxBlock * kMxBlock < a.N) {
                    *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(a.keepP[q]) + row * a.ldk[q] + col) =
                        mx8_encode4(v[q][0], v[q][1], v[q][2], v[q][3], mx8_inv_scale(b), b != 255u);
                    if (col % kMxBlock == 0) a.keepS[q][row * (a.ldk[q] / kMxBlock) + col / kMxBlock] = (uint8_t)b;
                }
            }
        }
    }
}

// ---- dG, dU as term planes (P = 0: as fp32 matrices), with the partial column sums of both (bias gradients) ------------------------------
// One pass over dH, G, U, bound by HBM: 440,000 x 300 in fp32 0.57 ms for 2.64 GB (4.6 TB/s, a large copy's rate), from checkpoints 0.39 ms.
// A block takes `rows` rows of qw * 4 columns; its partial sums are rows / rw sequential adds per thread, then rw.
template <int P, int TD, int TK>
__global__ __launch_bounds__(256) void gate_grad_kernel(MatIn dH, MatIn G, MatIn U, int64_t M, int N, int act, uint16_t* __restrict__ oG,
                                                        uint16_t* __restrict__ oU, int cols, int64_t ldo, int64_t plane, int rows, int qw, float* __restrict__ part, int64_t part_ld) {
    __shared__ float red[256][8];
    // qw quads of columns side by side, rw = 256 / qw rows at a time (300 columns: 75 x 3, not 64 of one block and 11 of the next)
    const int w = threadIdx.x / qw, lane = threadIdx.x - w * qw, rw = 256 / qw;
    const int c = w < rw ? (blockIdx.x * qw + lane) * 4 : cols;
    const int64_t r0 = (int64_t)blockIdx.y * rows, r1 = min(M, r0 + rows);
    const int cc = c < N ? c : 0;                             // (a lane of pad columns reads the first ones and writes zeros)
    float sg[4] = {0.f, 0.f, 0.f, 0.f}, su[4] = {0.f, 0.f, 0.f, 0.f};
    if (c < cols) {                     // (the pad columns of the result are written as zeros)
        auto one = [&](int64_t r, const float4& d, const float4& g, const float4& u) __attribute__((always_inline)) {
            const float dv[4] = {d.x, d.y, d.z, d.w}, gv[4] = {g.x, g.y, g.z, g.w}, uv[4] = {u.x, u.y, u.z, u.w};
            float og[4], ou[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                float v, s;
                gate_value_grad(act, gv[k], v, s);
                og[k] = c + k < N ? dv[k] * uv[k] * s : 0.f;
                ou[k] = c + k < N ? dv[k] * v : 0.f;
                sg[k] += og[k];
                su[k] += ou[k];
            }
            const float4 dg = make_float4(og[0], og[1], og[2], og[3]), du = make_float4(ou[0], ou[1], ou[2], ou[3]);
            if constexpr (P == 0) {
                *reinterpret_cast<float4*>(reinterpret_cast<float*>(oG) + r * ldo + c) = dg;
                *reinterpret_cast<float4*>(reinterpret_cast<float*>(oU) + r * ldo + c) = du;
            } else {
                uint2 tg[P], tu[P];
                bf16_terms4<P>(dg, tg);
                bf16_terms4<P>(du, tu);
#pragma unroll
                for (int p = 0; p < P; ++p) {
                    *reinterpret_cast<uint2*>(oG + p * plane + r * ldo + c) = tg[p];
                    *reinterpret_cast<uint2*>(oU + p * plane + r * ldo + c) = tu[p];
                }
            }
        };
        int64_t r = r0 + w;
        for (; r + rw < r1; r += 2 * rw) {                    // two rows' loads in flight
            const float4 d0 = mat_load4<TD>(dH, r, cc), g0 = mat_load4<TK>(G, r, cc), u0 = mat_load4<TK>(U, r, cc);
            const float4 d1 = mat_load4<TD>(dH, r + rw, cc), g1 = mat_load4<TK>(G, r + rw, cc), u1 = mat_load4<TK>(U, r + rw, cc);
            one(r, d0, g0, u0);
            one(r + rw, d1, g1, u1);
        }
        if (r < r1) one(r, mat_load4<TD>(dH, r, cc), mat_load4<TK>(G, r, cc), mat_load4<TK>(U, r, cc));
    }
    if (!part) return;
#pragma unroll
    for (int k = 0; k < 4; ++k) { red[threadIdx.x][k] = sg[k]; red[threadIdx.x][4 + k] = su[k]; }
    __syncthreads();
    if (w == 0 && c < N) {
        float s[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        for (int i = 0; i < rw; ++i)
#pragma unroll
            for (int k = 0; k < 8; ++k) s[k] += red[i * qw + lane][k];
        *reinterpret_cast<float4*>(part + (int64_t)blockIdx.y * part_ld + c) = make_float4(s[0], s[1], s[2], s[3]);
        *reinterpret_cast<float4*>(part + ((int64_t)gridDim.y + blockIdx.y) * part_ld + c) = make_float4(s[4], s[5], s[6], s[7]);
    }
}

// column sums of the partials: 64 columns a block, its 16 waves take every 16th part each, four at a time (grid.y: dbg, dbu)
__global__ __launch_bounds__(1024) void bias_sum_kernel(const float* __restrict__ part, int nparts, int64_t part_ld, int N, float* __restrict__ d0, float* __restrict__ d1) {
    __shared__ float red[16][64];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, c = blockIdx.x * 64 + lane;
    float s[4] = {0.f, 0.f, 0.f, 0.f};
    if (c < N) {
        const float* p = part + (int64_t)blockIdx.y * nparts * part_ld + c;
        int i = w;
        for (; i + 48 < nparts; i += 64) {
#pragma unroll
            for (int u = 0; u < 4; ++u) s[u] += p[(int64_t)(i + 16 * u) * part_ld];
        }
        for (; i < nparts; i += 16) s[0] += p[(int64_t)i * part_ld];
    }
    red[w][lane] = (s[0] + s[1]) + (s[2] + s[3]);
    __syncthreads();
    if (w == 0 && c < N) {
        float t = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) t += red[i][lane];
        (blockIdx.y ? d1 : d0)[c] = t;
    }
}

// ---- host side ----------------------------------------------------------------------------------------------------------------------------
int64_t up(int64_t n, int64_t m) { return (n + m - 1) / m * m; }

// bump allocator over the caller's workspace; one with base == nullptr only counts (`counting`: nothing is launched)
struct Arena {
    unsigned char* base;
    bool counting = base == nullptr;
    size_t used = 0;
    void* take(int64_t bytes) {
        void* p = counting ? nullptr : base + used;
        used += (size_t)up(bytes, 256);
        return p;
    }
};

// an operand as the tiled kernel reads it
struct Planes { const uint16_t* p; int64_t ld, plane; };

// in place where a bf16 matrix's rows start on 16 bytes (and its k-extent is whole pieces, `whole_cols`), else term planes in the workspace,
// written by the launch that run_terms makes of all jobs gathered in `jobs`
Planes make_planes(Arena& ar, const MatIn& m, int64_t n, int64_t F, int P, bool whole_cols, TermsJobs& jobs) {
    if (m.type == GEOGCN_T_BF16 && m.ld % 8 == 0 && aligned16(m.p) && (!whole_cols || F % 8 == 0)) return Planes{static_cast<const uint16_t*>(m.p), m.ld, 0};
    const int64_t plane = up(F, 64), ld = P * plane;
    uint16_t* o = static_cast<uint16_t*>(ar.take(n * ld * 2));
    if (n * ld > 0) jobs.job[jobs.n++] = TermsJobs::Job{m, n * (plane / 4), ld, plane, (int)F, (int)(plane / 4), o};
    return Planes{o, ld, plane};
}
int run_terms(const Arena& ar, const TermsJobs& jobs, int P, hipStream_t st) {
    if (ar.counting || jobs.n == 0) return 0;
    const int type = jobs.job[0].src.type;
    int64_t most = 0;
    for (int i = 0; i < jobs.n; ++i) most = std::max(most, jobs.job[i].total);
    auto* k = P == 3 ? &terms_kernel<3, GEOGCN_T_F32> : type == GEOGCN_T_F32 ? &terms_kernel<1, GEOGCN_T_F32>
              : type == GEOGCN_T_BF16 ? &terms_kernel<1, GEOGCN_T_BF16> : &terms_kernel<1, GEOGCN_T_MX8>;          // (three terms: fp32 only)
    hipLaunchKernelGGL(k, dim3((unsigned)std::min<int64_t>(cdiv(most, 256), (int64_t)kNumCU * 32), jobs.n), dim3(256), 0, st, jobs);
    GEOGCN_LAUNCH_CHECK("terms_kernel");
    return 0;
}

template <int PA, int PB, bool ASTR, bool BSTR, int NSEG, int BM, int BN, int BK, int WM, int WN, int ST, bool GATED>
int launch_tile(const TileArgs& a, hipStream_t st) {
    constexpr int bytes = ST * BK * 2 * (PA * BM + PB * BN);
    static_assert(bytes <= 160 * 1024, "LDS of a CU");
    static LdsAttrOnce attr;
    auto* k = &tile_kernel<PA, PB, ASTR, BSTR, NSEG, BM, BN, BK, WM, WN, ST, GATED>;
    if (const int rc = attr.ensure(reinterpret_cast<const void*>(k), bytes)) return rc;
    hipLaunchKernelGGL(k, dim3((unsigned)(a.n_mt * a.n_nt * a.nsplit)), dim3(WM * WN * 64), bytes, st, a);
    GEOGCN_LAUNCH_CHECK("tile_kernel");
    return 0;
}

// how a product is cut: tiles of the output, and its reduction over `nsplit` blocks where the tiles alone leave CUs idle
struct Cut { int n_mt, n_nt, nsplit, steps; };

int64_t out_cols(int type, int64_t N, int64_t ld) { return std::min<int64_t>(ld, up(N, type == GEOGCN_T_F32 ? 4 : 64)); }

int finish(const TileArgs& t, int nseg, int mode, hipStream_t st) {
    FinishArgs f;
    f.M = t.M; f.N = t.N; f.segw = t.segw; f.ldw = t.ldw;
    f.nsplit = t.nsplit; f.nseg = nseg; f.mode = mode; f.out_type = t.out_type; f.act = t.act; f.keep = t.keep;
    f.W = t.W;
    for (int q = 0; q < 2; ++q) {
        f.C[q] = t.C[q]; f.ldc[q] = t.ldc[q]; f.bias[q] = t.bias[q]; f.nc[q] = t.nc[q]; f.nck[q] = t.nck[q];
        f.keepP[q] = t.keepP[q]; f.ldk[q] = t.ldk[q]; f.keepS[q] = t.keepS[q];
    }
    const unsigned grid = (unsigned)std::min<int64_t>(cdiv(t.M * (t.segw / 4), 256), (int64_t)kNumCU * 32);
    hipLaunchKernelGGL(finish_kernel, dim3(grid), dim3(256), 0, st, f);
    GEOGCN_LAUNCH_CHECK("finish_kernel");
    return 0;
}

// one product on one tile shape: run it, and add up what was split
template <int PA, int PB, bool ASTR, bool BSTR, int NSEG, int BM, int BN, int BK, int WM, int WN, int ST, bool GATED>
int run_tiles(Arena& ar, TileArgs& t, const Cut& c, hipStream_t st) {
    t.n_mt = c.n_mt; t.n_nt = c.n_nt; t.nsplit = c.nsplit; t.steps_per_split = c.steps;
    t.segw = (int64_t)c.n_nt * (BN / NSEG); t.ldw = NSEG * t.segw;
    // (threads of a launch are counted with 32 bits)
    GEOGCN_REQUIRE((int64_t)c.n_mt * c.n_nt * c.nsplit < ((int64_t)1 << 32) / (WM * WN * 64), GEOGCN_E_SIZE, "gated: a product of %lld x %lld is too large",
                   (long long)t.M, (long long)t.N);
    if (c.nsplit > 1) t.W = static_cast<float*>(ar.take((int64_t)c.nsplit * t.M * t.ldw * 4));
    if (ar.counting) return 0;
    t.mode = c.nsplit > 1 ? EPI_SLAB : GATED ? EPI_GATED : EPI_STORE;
    const int rc = launch_tile<PA, PB, ASTR, BSTR, NSEG, BM, BN, BK, WM, WN, ST, GATED>(t, st);
    if (rc || c.nsplit == 1) return rc;
    return finish(t, NSEG, GATED ? EPI_GATED : EPI_STORE, st);
}

// Which tile shape, and how many ways the reduction is split: the pair with the least estimated time, in clocks.  The busiest CU has R tiles, `per_cu`
// of them at a time: it takes the products of R tiles at 0.7 of the matrix pipe's rate times the shape's measured standing (`eff`: 1 for the
// fastest of its list on a large product), or, where few blocks are there to cover for each other, a load's latency (1,900) for every
// stage that is not asked for ahead; a tile begins and ends in 6,000.  A split writes and reads its slabs (1,500 bytes a clock) and
// takes one more launch.  (The constants are fitted to sweeps of the shapes over 100 to 440,000 rows and widths of 256 to 4,096; the estimate errs by
// up to 15 % where it takes a shape that is not the fastest: the input gradient of 512 x 4,096 -> 4,096 in two terms 82 us, 73 on 256 x 256.)
struct Shape {
    int bm, bns, bk, stages, per_cu;
    double eff;
    int (*run)(Arena&, TileArgs&, const Cut&, hipStream_t);
};
template <int N>
int run_best(const Shape (&shapes)[N], Arena& ar, TileArgs& t, int64_t cols, int nseg, int terms, hipStream_t st) {
    double best = 0;
    const Shape* pick = nullptr;
    Cut cut{};
    for (const Shape& s : shapes) {
        const int64_t n_mt = cdiv(t.M, s.bm), n_nt = cdiv(cols, s.bns), tiles = n_mt * n_nt;
        const int64_t steps = std::max<int64_t>(1, t.n_kseg * cdiv(t.K[0], s.bk));
        for (int64_t want = 1; want == 1 || (want <= steps / 4 && tiles * want <= 2 * kNumCU); want += want < 8 ? 1 : want / 4) {
            const int64_t per = cdiv(steps, want), nsplit = cdiv(steps, per), R = cdiv(tiles * nsplit, kNumCU), turns = cdiv(R, s.per_cu);
            const double products = (double)R * s.bm * s.bns * nseg * (per * s.bk) * terms / (2048 * 0.7 * s.eff);
            double clk = std::max(products, (double)turns * per * 1900 / (s.stages - 1)) + turns * 6000.0;
            if (nsplit > 1) clk += 2.0 * nsplit * t.M * n_nt * s.bns * nseg * 4 / 1500 + 16000;
            if (!pick || clk < best) {
                best = clk;
                pick = &s;
                cut = Cut{(int)n_mt, (int)n_nt, (int)nsplit, (int)per};
            }
        }
    }
    return pick->run(ar, t, cut, st);
}

// X.[Wg | Wu] and the gate.  (Shapes of two blocks a CU where LDS and registers allow: one block's epilogue and barriers run under the other's
// products.  8192 x 2048 -> 8192 in bf16: 128 x 256 524-660 us from machine to machine, the same with 64 k-values a stage and one block a CU 650-790.)
int run_forward(Arena& ar, TileArgs& t, int P, hipStream_t st) {
    static const Shape fp32[] = {{128, 128, 32, 2, 1, 1.0, run_tiles<3, 3, false, true, 2, 128, 256, 32, 2, 4, 2, true>},
                                 {256, 64, 32, 2, 1, 0.95, run_tiles<3, 3, false, true, 2, 256, 128, 32, 4, 2, 2, true>},
                                 {64, 64, 32, 2, 2, 0.85, run_tiles<3, 3, false, true, 2, 64, 128, 32, 2, 2, 2, true>}};
    static const Shape bf16[] = {{128, 128, 32, 3, 2, 1.0, run_tiles<1, 1, false, true, 2, 128, 256, 32, 2, 4, 3, true>},
                                 {256, 64, 32, 3, 2, 0.97, run_tiles<1, 1, false, true, 2, 256, 128, 32, 4, 2, 3, true>},
                                 {128, 64, 32, 3, 3, 0.88, run_tiles<1, 1, false, true, 2, 128, 128, 32, 4, 2, 3, true>},
                                 {128, 64, 64, 4, 1, 0.8, run_tiles<1, 1, false, true, 2, 128, 128, 64, 4, 2, 4, true>}};
    const int64_t cols = t.keep == GEOGCN_KEEP_MX8 ? std::max(t.ncols, up(t.N, kMxBlock)) : t.ncols;
    return P == 3 ? run_best(fp32, ar, t, cols, 2, 6, st) : run_best(bf16, ar, t, cols, 2, 1, st);
}

// dG.Wg^T + dU.Wu^T: both operands run along k, so the one-term shapes take 64 k-values a stage (whole 128-byte lines of a row)
int run_input_grad(Arena& ar, TileArgs& t, int P, hipStream_t st) {
    static const Shape fp32[] = {{256, 160, 32, 2, 1, 1.0, run_tiles<3, 3, false, false, 1, 256, 160, 32, 4, 2, 2, false>},
                                 {256, 128, 32, 2, 1, 0.92, run_tiles<3, 3, false, false, 1, 256, 128, 32, 4, 2, 2, false>},
                                 {64, 128, 32, 2, 2, 0.68, run_tiles<3, 3, false, false, 1, 64, 128, 32, 2, 2, 2, false>}};
    static const Shape bf16[] = {{256, 256, 64, 2, 1, 1.0, run_tiles<1, 1, false, false, 1, 256, 256, 64, 2, 4, 2, false>},
                                 {256, 128, 64, 3, 1, 0.85, run_tiles<1, 1, false, false, 1, 256, 128, 64, 4, 2, 3, false>},
                                 {128, 128, 64, 4, 1, 0.75, run_tiles<1, 1, false, false, 1, 128, 128, 64, 2, 4, 4, false>}};
    // dG, dU of a bf16 block as two terms (256 x 256 / 128 x 128: 8,192 x 1,024 -> 4,096 250 / 288 us, 60,000 x 600 -> 600 214 / 230, 9,475 x 300 ->
    // 600 63 / 25; 256 x 128 lies between them: 275, 251, 40)
    static const Shape two[] = {{256, 256, 32, 3, 1, 1.0, run_tiles<2, 1, false, false, 1, 256, 256, 32, 2, 4, 3, false>},
                                {128, 128, 32, 3, 2, 0.78, run_tiles<2, 1, false, false, 1, 128, 128, 32, 2, 4, 3, false>}};
    if (P == 2) return run_best(two, ar, t, t.ncols, 1, 2, st);
    return P == 3 ? run_best(fp32, ar, t, t.ncols, 1, 6, st) : run_best(bf16, ar, t, t.ncols, 1, 1, st);
}

// X^T.[B0 | B1] (nseg = 2) or X^T.B0
int run_weight_grad(Arena& ar, TileArgs& t, int PA, int PB, int nseg, hipStream_t st) {
    static const Shape fp32[] = {{128, 128, 32, 2, 1, 1.0, run_tiles<3, 3, true, true, 2, 128, 256, 32, 2, 4, 2, false>}};
    static const Shape mx8[] = {{160, 160, 32, 2, 1, 1.0, run_tiles<1, 3, true, true, 2, 160, 320, 32, 2, 4, 2, false>},
                                {128, 128, 32, 2, 1, 0.85, run_tiles<1, 3, true, true, 2, 128, 256, 32, 2, 4, 2, false>}};
    static const Shape bf16[] = {{128, 128, 64, 3, 1, 1.0, run_tiles<1, 1, true, true, 2, 128, 256, 64, 2, 4, 3, false>},
                                 {128, 64, 64, 4, 1, 0.7, run_tiles<1, 1, true, true, 2, 128, 128, 64, 2, 4, 4, false>}};
    // dG, dU of a bf16 block as two terms (128 / 64 columns of each, with the gate pass: 8,192 x 1,024 -> 4,096 330 / 362 us, 4,097 x 1,024 ->
    // 1,536 91 / 88, 440,000 x 300 -> 300 882 / 843)
    static const Shape two[] = {{128, 128, 32, 3, 1, 1.0, run_tiles<1, 2, true, true, 2, 128, 256, 32, 2, 4, 3, false>},
                                {128, 64, 32, 2, 2, 0.8, run_tiles<1, 2, true, true, 2, 128, 128, 32, 2, 4, 2, false>}};
    static const Shape mx8_one[] = {{160, 256, 32, 2, 1, 1.0, run_tiles<1, 3, true, true, 1, 160, 256, 32, 2, 4, 2, false>},
                                    {128, 128, 32, 5, 1, 0.8, run_tiles<1, 3, true, true, 1, 128, 128, 32, 2, 4, 5, false>}};
    static const Shape bf16_one[] = {{128, 128, 32, 6, 1, 1.0, run_tiles<1, 1, true, true, 1, 128, 128, 32, 2, 4, 6, false>}};
    if (nseg == 2) {
        if (PA == 3) return run_best(fp32, ar, t, t.ncols, 2, 6, st);
        if (PB == 2) return run_best(two, ar, t, t.ncols, 2, 2, st);
        return PB == 3 ? run_best(mx8, ar, t, t.ncols, 2, 3, st) : run_best(bf16, ar, t, t.ncols, 2, 1, st);
    }
    return PB == 3 ? run_best(mx8_one, ar, t, t.ncols, 1, 3, st) : run_best(bf16_one, ar, t, t.ncols, 1, 1, st);
}

TileArgs tile_args() {
    TileArgs t;
    memset(&t, 0, sizeof(t));
    t.n_kseg = 1;
    return t;
}

int elem_align(int type) { return type == GEOGCN_T_F32 ? 16 : type == GEOGCN_T_BF16 ? 8 : 4; }

int check_mat(const char* who, const char* name, int type, const void* p, int64_t ld, const uint8_t* scale, int64_t F) {
    GEOGCN_REQUIRE(p, GEOGCN_E_NULL, "%s: %s is null", who, name);
    GEOGCN_REQUIRE(reinterpret_cast<uintptr_t>(p) % elem_align(type) == 0, GEOGCN_E_ALIGN, "%s: %s is not aligned", who, name);
    // (a tile's 256 rows are addressed with 32 bits)
    GEOGCN_REQUIRE(ld <= (1 << 21), GEOGCN_E_SIZE, "%s: pitch %lld of %s is too large", who, (long long)ld, name);
    if (type == GEOGCN_T_MX8) {
        GEOGCN_REQUIRE(scale, GEOGCN_E_NULL, "%s: %s has no scales", who, name);
        GEOGCN_REQUIRE(ld % kMxBlock == 0 && ld >= F, GEOGCN_E_ALIGN, "%s: code pitch %lld of %s (%lld columns) is not whole blocks", who,
                       (long long)ld, name, (long long)F);
    } else {
        GEOGCN_REQUIRE(ld % 4 == 0 && ld >= up(F, 4), GEOGCN_E_ALIGN, "%s: pitch %lld of %s (%lld columns)", who, (long long)ld, name, (long long)F);
    }
    return 0;
}

bool act_ok(int act) {
    return act == GEOGCN_ACT_NONE || act == GEOGCN_ACT_TANH || act == GEOGCN_ACT_SIGMOID || act == GEOGCN_ACT_RELU || act == GEOGCN_ACT_SILU ||
           act == GEOGCN_ACT_GELU;
}

// terms per value of an operand: bf16 and 8-bit values are one term; fp32 three, or one (rounded) where the caller asked for bf16 products
int terms_of(int type, int precision) { return type == GEOGCN_T_F32 && precision != GEOGCN_GEMM_BF16 ? 3 : 1; }
// ... of dG and dU, which are formed in fp32 whatever the block's type: in a bf16 block two (2^-16 of a value; one would add 2^-8 of every
// product to results that are rounded to 2^-8 once: 0.0023 from the 64-bit results in the norm, 0.0017 with two) unless bf16 products are asked for
int grad_terms_of(int type, int precision) { return precision == GEOGCN_GEMM_BF16 ? 1 : type == GEOGCN_T_F32 ? 3 : 2; }

int check_dims(const char* who, int64_t M, int64_t K, int64_t N) {
    GEOGCN_REQUIRE(M >= 0 && K >= 0 && N >= 0, GEOGCN_E_SIZE, "%s: negative size", who);
    GEOGCN_REQUIRE(K <= (1 << 20) && N <= (1 << 20) && M <= (int64_t)1 << 31, GEOGCN_E_SIZE, "%s: %lld x %lld -> %lld is too large", who, (long long)M,
                   (long long)K, (long long)N);
    return 0;
}

struct FwdArgs {
    int64_t M, K, N;
    int type, precision, keep, act;
    MatIn X, Wg, Wu;
    const float *bg, *bu;
    void* H; int64_t ldh;
    void* keepP[2]; int64_t ldk[2]; uint8_t* keepS[2];
};
// The rows up to which every 8 rows take one more pass over the weights (from L2) instead of term planes and whole tiles.  So / by tiles, us on the
// GPU, 1, 8, 16, 32, 64 rows: 300 -> 300 fp32 4.6 / 15.4, 7.1 / 15.3, 7.2 / 15.3, 7.3 / 16.8, 7.4 / 17.9; 1,024 -> 4,096 fp32 7.3 / 31.4, 12.7 / 31.8,
// 12.8 / 31.9, 23.0 / 34.8, 42.9 / 35.6; the same in bf16 6.3 / 14.3, 14.5 / 14.2, 15.0 / 14.0, 27.7 / 15.4, 52.3 / 15.8.  (Few columns under a long
// reduction fill few CUs: 4,096 -> 1,024 in bf16 is 16.6 / 12.6 at one row and 39.4 / 14.1 at 16.)
constexpr int64_t kFewRows = 16;
template <typename T, int VEC>
int launch_few(const FewArgs& a, hipStream_t st) {
    const int rm = a.M == 1 ? 1 : a.M == 2 ? 2 : a.M <= 4 ? 4 : 8;
    auto* k = rm == 1 ? &few_rows_kernel<T, VEC, 1> : rm == 2 ? &few_rows_kernel<T, VEC, 2> : rm == 4 ? &few_rows_kernel<T, VEC, 4> : &few_rows_kernel<T, VEC, 8>;
    const int64_t cols = std::max(a.ncols, a.keep == GEOGCN_KEEP_MX8 ? up(a.N, kMxBlock) : std::max(a.nck[0], a.nck[1]));
    hipLaunchKernelGGL(k, dim3((unsigned)cdiv(cols, 32), (unsigned)cdiv(a.M, rm)), dim3(512), 0, st, a);
    GEOGCN_LAUNCH_CHECK("few_rows_kernel");
    return 0;
}
int forward_few(const FwdArgs& f, hipStream_t st) {
    FewArgs a;
    a.M = f.M; a.K = (int)f.K; a.N = (int)f.N; a.act = f.act; a.out_type = f.type; a.keep = f.keep;
    a.X = f.X.p; a.ldx = f.X.ld; a.Wg = f.Wg.p; a.ldwg = f.Wg.ld; a.Wu = f.Wu.p; a.ldwu = f.Wu.ld;
    a.bias[0] = f.bg; a.bias[1] = f.bu; a.H = f.H; a.ldh = f.ldh; a.ncols = out_cols(f.type, f.N, f.ldh);
    for (int q = 0; q < 2; ++q) {
        a.keepP[q] = f.keepP[q]; a.ldk[q] = f.ldk[q]; a.keepS[q] = f.keepS[q];
        a.nck[q] = f.keep == GEOGCN_KEEP_FULL ? out_cols(f.type, f.N, f.ldk[q]) : 0;
    }
    if (f.type == GEOGCN_T_F32) return launch_few<float, 4>(a, st);
    const bool wide = f.Wg.ld % 8 == 0 && f.Wu.ld % 8 == 0 && aligned16(f.Wg.p) && aligned16(f.Wu.p);
    return wide ? launch_few<uint16_t, 8>(a, st) : launch_few<uint16_t, 4>(a, st);
}
// (an fp32 block at bf16 products: its operands are to be rounded, and this kernel multiplies the stored values)
bool few_rows(const FwdArgs& f) { return f.M <= kFewRows && !(f.type == GEOGCN_T_F32 && f.precision == GEOGCN_GEMM_BF16); }

// what the gated epilogue writes
void gated_outputs(TileArgs& t, const FwdArgs& f) {
    t.out_type = f.type; t.act = f.act; t.keep = f.keep;
    t.bias[0] = f.bg; t.bias[1] = f.bu;
    t.C[0] = f.H; t.ldc[0] = f.ldh;
    t.nc[0] = t.ncols = out_cols(f.type, f.N, f.ldh);
    for (int q = 0; q < 2; ++q) {
        t.keepP[q] = f.keepP[q]; t.ldk[q] = f.ldk[q]; t.keepS[q] = f.keepS[q];
        if (f.keep == GEOGCN_KEEP_FULL) t.ncols = std::max(t.ncols, t.nck[q] = out_cols(f.type, f.N, f.ldk[q]));
    }
}
int forward_exact(Arena& ar, const FwdArgs& f, hipStream_t st) {
    // [G | U] by the library's dual product into one slab, the gate by the pass that finishes split reductions
    TileArgs t = tile_args();
    t.M = f.M; t.N = f.N; t.nsplit = 1;
    t.segw = up(f.N, kMxBlock); t.ldw = 2 * t.segw;
    t.W = static_cast<float*>(ar.take(f.M * t.ldw * 4));
    gated_outputs(t, f);
    const size_t need = f.K ? geogcn_gemm_dual_workspace_bytes(0, f.M, f.N, f.N, f.K, GEOGCN_GEMM_F32) : 0;
    void* w = ar.take((int64_t)need);
    if (ar.counting) return 0;
    if (f.K == 0) {
        if (const int rc = zero_rows_async(t.W, f.M, t.ldw, t.ldw, st)) return rc;
    } else if (const int rc = geogcn_gemm_dual_f32(0, f.M, f.N, f.N, f.K, static_cast<const float*>(f.X.p), f.X.ld, static_cast<const float*>(f.Wg.p),
                                                   f.Wg.ld, static_cast<const float*>(f.Wu.p), f.Wu.ld, t.W, t.ldw, t.W + t.segw, t.ldw, nullptr,
                                                   GEOGCN_ACT_NONE, nullptr, GEOGCN_ACT_NONE, GEOGCN_GEMM_F32, need ? w : nullptr, need, st)) return rc;
    return finish(t, 2, EPI_GATED, st);
}
// fp32 blocks of many rows: the library's whole-rows kernel reads X as it is (no term planes in memory) and takes all columns of 64 rows.
// It starts at 16,384 rows, where its 64-row blocks go round the CUs -- 32,768 where either width passes 640 and a block works longer --, and
// not for kept checkpoints, whose blocks its waves share.  By tiles / by whole rows, G and U kept: 440,000 x 300 -> 300 1,598 / 1,156 us,
// 20,000 x 300 -> 300 92 / 80, 60,000 x 600 -> 600 628 / 566, 20,000 x 900 -> 930 449 / 523, 60,000 x 900 -> 900 1,243 / 1,169.
constexpr int64_t kWholeRowsMin = 16384;
int whole_rows(const FwdArgs& f, GemmCall* c) {
    if (f.type != GEOGCN_T_F32 || f.precision != GEOGCN_GEMM_BF16X3 || f.keep == GEOGCN_KEEP_MX8 || f.K == 0) return 0;
    if (f.M < (std::max(f.K, f.N) > 640 ? 2 * kWholeRowsMin : kWholeRowsMin)) return 0;
    *c = GemmCall{};
    c->M = f.M; c->n_nseg = 2; c->n_kseg = 1; c->precision = GEOGCN_GEMM_BF16X3;
    c->A[0] = static_cast<const float*>(f.X.p); c->lda[0] = f.X.ld; c->K[0] = f.K;
    c->B[0] = static_cast<const float*>(f.Wg.p); c->ldb[0] = f.Wg.ld; c->B[1] = static_cast<const float*>(f.Wu.p); c->ldb[1] = f.Wu.ld;
    c->N[0] = c->N[1] = f.N; c->bias[0] = f.bg; c->bias[1] = f.bu;
    const bool kept = f.keep == GEOGCN_KEEP_FULL;             // (G waits for U in its own matrix, or where H comes to stand)
    c->C[0] = static_cast<float*>(kept ? f.keepP[0] : f.H); c->ldc[0] = kept ? f.ldk[0] : f.ldh;
    c->C[1] = static_cast<float*>(kept ? f.keepP[1] : nullptr); c->ldc[1] = kept ? f.ldk[1] : f.ldh;
    c->gluH = static_cast<float*>(f.H); c->ldgluH = f.ldh; c->glu_act = f.act;
    return x3_rows_kc(*c, false, false);
}
int forward(Arena& ar, const FwdArgs& f, hipStream_t st) {
    if (few_rows(f)) return ar.counting ? 0 : forward_few(f, st);
    if (f.precision == GEOGCN_GEMM_F32 && f.type == GEOGCN_T_F32) return forward_exact(ar, f, st);
    GemmCall call;
    if (const int kc = whole_rows(f, &call)) {
        void* w = ar.take((int64_t)x3_rows_ws_bytes(call, kc));
        return ar.counting ? 0 : x3_run_rows(kc, false, call, w, st);
    }
    const int P = terms_of(f.type, f.precision);
    TermsJobs jobs{};
    const Planes x = make_planes(ar, f.X, f.M, f.K, P, true, jobs), wg = make_planes(ar, f.Wg, f.K, f.N, P, false, jobs),
                 wu = make_planes(ar, f.Wu, f.K, f.N, P, false, jobs);
    if (const int rc = run_terms(ar, jobs, P, st)) return rc;
    TileArgs t = tile_args();
    t.M = f.M; t.N = f.N; t.K[0] = f.K;
    t.A[0] = x.p; t.lda[0] = x.ld; t.planeA[0] = x.plane;
    t.B[0] = wg.p; t.ldb[0] = wg.ld; t.planeB[0] = wg.plane;
    t.B[1] = wu.p; t.ldb[1] = wu.ld; t.planeB[1] = wu.plane;
    gated_outputs(t, f);
    return run_forward(ar, t, P, st);
}

struct BwdArgs {
    int64_t M, K, N;
    int type, precision, act;
    MatIn dH, X, G, U, Wg, Wu;
    void *dX; int64_t lddx;
    void* dW[2]; int64_t lddw[2];
    float* db[2];
};
// P = 0: dG, dU as fp32 matrices of pitch ldo
int gate_gradients(Arena& ar, const BwdArgs& b, int P, int64_t ldo, hipStream_t st, uint16_t** dG_out, uint16_t** dU_out) {
    const int64_t ldt = P ? P * ldo : ldo, plane = ldo, bytes = b.M * ldt * (P ? 2 : 4);
    uint16_t* dG = *dG_out = static_cast<uint16_t*>(ar.take(bytes));
    uint16_t* dU = *dU_out = static_cast<uint16_t*>(ar.take(bytes));
    // quads of columns of a block: all of them, or equal shares where there are more than 256; rows: enough blocks to keep every CU at eight, not
    // fewer than eight rows (each block writes a row of partial sums) and 1,024 where they are long anyway
    const int64_t quads = cdiv(ldo, 4), cblocks = cdiv(quads, 256);
    const int qw = (int)cdiv(quads, cblocks), rw = 256 / qw;
    const int64_t fill = std::max<int64_t>(8, cdiv(b.M * cblocks, (int64_t)kNumCU * 8));
    const int rows = (int)up(std::max(std::min<int64_t>(1024, fill), cdiv(b.M, 65535)), 2 * rw);      // (65,535: grid.y)
    const int64_t nparts = cdiv(b.M, rows), part_ld = up(b.N, 4);
    float* part = b.db[0] ? static_cast<float*>(ar.take(2 * nparts * part_ld * 4)) : nullptr;
    if (!ar.counting) {
        const dim3 grid((unsigned)cblocks, (unsigned)nparts);
        const bool f32 = b.type == GEOGCN_T_F32, q8 = b.G.type == GEOGCN_T_MX8;
        constexpr int F = GEOGCN_T_F32, H = GEOGCN_T_BF16, Q = GEOGCN_T_MX8;
        auto* k = !f32 ? (P == 2 ? (q8 ? &gate_grad_kernel<2, H, Q> : &gate_grad_kernel<2, H, H>) : (q8 ? &gate_grad_kernel<1, H, Q> : &gate_grad_kernel<1, H, H>))
                  : P == 3 ? (q8 ? &gate_grad_kernel<3, F, Q> : &gate_grad_kernel<3, F, F>)
                  : P == 1 ? (q8 ? &gate_grad_kernel<1, F, Q> : &gate_grad_kernel<1, F, F>)
                           : (q8 ? &gate_grad_kernel<0, F, Q> : &gate_grad_kernel<0, F, F>);
        hipLaunchKernelGGL(k, grid, dim3(256), 0, st, b.dH, b.G, b.U, b.M, (int)b.N, b.act, dG, dU, (int)ldo, ldt, plane, rows, qw, part, part_ld);
        GEOGCN_LAUNCH_CHECK("gate_grad_kernel");
        if (part) {
            hipLaunchKernelGGL(bias_sum_kernel, dim3((unsigned)cdiv(b.N, 64), 2), dim3(1024), 0, st, part, (int)nparts, part_ld, (int)b.N, b.db[0], b.db[1]);
            GEOGCN_LAUNCH_CHECK("bias_sum_kernel");
        }
    }
    return 0;
}
// X^T.[B0 | B1] of a checkpointed X and fp32 matrices by the library's A^T.B kernel: X's codes and the fp32 values are read as they are
int tn_q8(Arena& ar, const MatIn& X, int64_t M, int64_t K, int64_t N, int nseg, const float* const* B, int64_t ldb, void* const* dW, const int64_t* lddw,
          hipStream_t st) {
    const int bn = up(N, 256) <= up(N, 320) ? 256 : 320;
    X3TnCall t{};
    t.M = K; t.K = M; t.A8 = static_cast<const uint8_t*>(X.p); t.S8 = X.scale; t.ld8 = X.ld;
    t.n_mt = (int)cdiv(K, 160); t.nt_per_seg = (int)cdiv(N, bn); t.n_nt = nseg * t.nt_per_seg;
    // one block a CU and the tiles of a slab on one XCD: as many whole slabs as its 32 CUs take
    const int T = t.n_mt * t.n_nt;
    t.kchunk = up(cdiv(M, (int64_t)kNumXCD * std::max(1, kNumCU / kNumXCD / T)), 32);
    t.nsplit = (int)cdiv(M, t.kchunk);
    t.seg_w = up(N, kMxBlock); t.ldw = nseg * t.seg_w;
    t.W = static_cast<float*>(ar.take((int64_t)t.nsplit * K * t.ldw * 4));
    if (ar.counting) return 0;
    TileArgs f = tile_args();
    f.M = K; f.N = N; f.nsplit = t.nsplit; f.W = t.W; f.segw = t.seg_w; f.ldw = t.ldw; f.out_type = GEOGCN_T_F32;
    for (int q = 0; q < nseg; ++q) {
        f.nc[q] = up(N, 4);
        t.B[q] = B[q]; t.ldb[q] = ldb; t.N[q] = N;
        f.C[q] = dW[q]; f.ldc[q] = lddw[q];
    }
    if (const int rc = x3_tn_launch(160, bn, t, st)) return rc;
    return finish(f, nseg, EPI_STORE, st);
}
// The library's fp32 products leave the pad columns of a result as they are where they add up a split reduction: a result that they form gets its
// pads (fewer than four columns) from here.
int zero_pads(void* C, int64_t rows, int64_t cols, int64_t ld, hipStream_t st) {
    const int64_t pads = up(cols, 4) - cols;
    return pads ? zero_rows_async(static_cast<float*>(C) + cols, rows, pads, ld, st) : 0;
}
// the products by the library's fp32 kernels: dG, dU (and a checkpointed X) as fp32 matrices
int backward_exact(Arena& ar, const BwdArgs& b, int precision, hipStream_t st) {
    const int64_t ldo = up(b.N, 4);
    uint16_t *g, *u;
    if (const int rc = gate_gradients(ar, b, 0, ldo, st, &g, &u)) return rc;
    const float *dG = reinterpret_cast<const float*>(g), *dU = reinterpret_cast<const float*>(u);
    if (b.dX) {
        const size_t need = geogcn_gemm_kcat_workspace_bytes(1, b.M, b.K, b.N, b.N, precision);
        void* w = ar.take((int64_t)need);
        if (!ar.counting)
            if (const int rc = zero_pads(b.dX, b.M, b.K, b.lddx, st)) return rc;
        if (!ar.counting)
            if (const int rc = geogcn_gemm_kcat_f32(1, b.M, b.K, b.N, b.N, dG, ldo, static_cast<const float*>(b.Wg.p), b.Wg.ld, dU, ldo,
                                                    static_cast<const float*>(b.Wu.p), b.Wu.ld, static_cast<float*>(b.dX), b.lddx, 0, precision,
                                                    need ? w : nullptr, need, st)) return rc;
    }
    if (b.dW[0] && precision == GEOGCN_GEMM_BF16X3 && b.X.type == GEOGCN_T_MX8) {
        const float* B[2] = {dG, dU};
        if (const int rc = tn_q8(ar, b.X, b.M, b.K, b.N, 2, B, ldo, b.dW, b.lddw, st)) return rc;
    } else if (b.dW[0]) {
        const float* X = static_cast<const float*>(b.X.p);
        int64_t ldx = b.X.ld;
        if (b.X.type == GEOGCN_T_MX8) {
            ldx = up(b.K, 4);
            float* x = static_cast<float*>(ar.take(b.M * ldx * 4));
            if (!ar.counting)
                if (const int rc = geogcn_mx8_unpack(b.M, (int32_t)b.K, GEOGCN_T_F32, static_cast<const uint8_t*>(b.X.p), b.X.ld, b.X.scale, x, ldx, st)) return rc;
            X = x;
        }
        const size_t need = geogcn_gemm_dual_workspace_bytes(1, b.K, b.N, b.N, b.M, precision);
        void* w = ar.take((int64_t)need);
        for (int q = 0; q < 2 && !ar.counting; ++q)
            if (const int rc = zero_pads(b.dW[q], b.K, b.N, b.lddw[q], st)) return rc;
        if (!ar.counting)
            if (const int rc = geogcn_gemm_dual_f32(1, b.K, b.N, b.N, b.M, X, ldx, dG, ldo, dU, ldo, static_cast<float*>(b.dW[0]), b.lddw[0],
                                                    static_cast<float*>(b.dW[1]), b.lddw[1], nullptr, GEOGCN_ACT_NONE, nullptr, GEOGCN_ACT_NONE, precision,
                                                    need ? w : nullptr, need, st)) return rc;
    }
    return 0;
}
int backward(Arena& ar, const BwdArgs& b, hipStream_t st) {
    if (b.precision == GEOGCN_GEMM_F32 && b.type == GEOGCN_T_F32) return backward_exact(ar, b, GEOGCN_GEMM_F32, st);
    // fp32 over many rows and 192 to 320 inputs (two whole tiles of the library's A^T.B kernel, a column pass of its whole-rows kernel): dG, dU stay
    // fp32 matrices and the library's split-bf16 kernels multiply them.  So / by tiles: 440,000 x 300 -> 300 2.5 / 3.1 ms, 100,000 x 300 -> 300
    // 550 / 715 us, 20,000 x 192 -> 640 224 / 242; outside, 100,000 x 160 -> 300 480 / 511 but 20,000 x 160 -> 640 247 / 214, 60,000 x 600 ->
    // 600 1.40 / 1.14 ms.
    if (b.type == GEOGCN_T_F32 && b.precision == GEOGCN_GEMM_BF16X3 && b.M >= kWholeRowsMin && b.K >= 192 && b.K <= 320 && b.N <= 1024)
        return backward_exact(ar, b, GEOGCN_GEMM_BF16X3, st);
    const int P = terms_of(b.type, b.precision), PX = b.X.type == GEOGCN_T_F32 ? P : 1, PG = grad_terms_of(b.type, b.precision);
    const int64_t plane = up(b.N, 64), ldo = PG * plane;
    uint16_t *dG, *dU;
    if (const int rc = gate_gradients(ar, b, PG, plane, st, &dG, &dU)) return rc;
    TermsJobs jobs{};
    Planes wg{}, wu{}, x{};
    if (b.dX) {
        wg = make_planes(ar, b.Wg, b.K, b.N, P, true, jobs);
        wu = make_planes(ar, b.Wu, b.K, b.N, P, true, jobs);
    }
    if (b.dW[0] && b.X.type != b.Wg.type) {                   // (a checkpointed X: a storage type of its own)
        TermsJobs own{};
        x = make_planes(ar, b.X, b.M, b.K, PX, false, own);
        if (const int rc = run_terms(ar, own, PX, st)) return rc;
    } else if (b.dW[0]) {
        x = make_planes(ar, b.X, b.M, b.K, PX, false, jobs);
    }
    if (const int rc = run_terms(ar, jobs, P, st)) return rc;
    if (b.dX) {
        TileArgs t = tile_args();
        t.M = b.M; t.N = b.K; t.n_kseg = 2; t.K[0] = t.K[1] = b.N;
        t.A[0] = dG; t.A[1] = dU;
        t.B[0] = wg.p; t.ldb[0] = wg.ld; t.planeB[0] = wg.plane;
        t.B[1] = wu.p; t.ldb[1] = wu.ld; t.planeB[1] = wu.plane;
        for (int q = 0; q < 2; ++q) { t.lda[q] = ldo; t.planeA[q] = plane; }
        t.out_type = b.type; t.C[0] = b.dX; t.ldc[0] = b.lddx; t.nc[0] = t.ncols = out_cols(b.type, b.K, b.lddx);
        if (const int rc = run_input_grad(ar, t, PG, st)) return rc;
    }
    if (b.dW[0]) {
        TileArgs t = tile_args();
        t.M = b.K; t.N = b.N; t.K[0] = b.M;
        t.A[0] = x.p; t.lda[0] = x.ld; t.planeA[0] = x.plane;
        t.B[0] = dG; t.B[1] = dU;
        for (int q = 0; q < 2; ++q) { t.ldb[q] = ldo; t.planeB[q] = plane; t.C[q] = b.dW[q]; t.ldc[q] = b.lddw[q]; }
        t.out_type = b.type;
        for (int q = 0; q < 2; ++q) t.ncols = std::max(t.ncols, t.nc[q] = out_cols(b.type, b.N, b.lddw[q]));
        if (const int rc = run_weight_grad(ar, t, PX, PG, 2, st)) return rc;
    }
    return 0;
}

struct WgradArgs { int64_t M, K, N; int type, precision; MatIn X, dZ; void* dW; int64_t lddw; };
int weight_grad_exact(Arena& ar, const WgradArgs& w, hipStream_t st) {
    const int64_t ldx = up(w.K, 4);
    float* x = static_cast<float*>(ar.take(w.M * ldx * 4));
    const size_t need = geogcn_gemm_workspace_bytes(1, 0, w.K, w.N, w.M, GEOGCN_GEMM_F32);
    void* g = ar.take((int64_t)need);
    if (ar.counting) return 0;
    if (const int rc = geogcn_mx8_unpack(w.M, (int32_t)w.K, GEOGCN_T_F32, static_cast<const uint8_t*>(w.X.p), w.X.ld, w.X.scale, x, ldx, st)) return rc;
    if (const int rc = zero_pads(w.dW, w.K, w.N, w.lddw, st)) return rc;
    return geogcn_gemm_f32(1, 0, w.K, w.N, w.M, x, ldx, static_cast<const float*>(w.dZ.p), w.dZ.ld, static_cast<float*>(w.dW), w.lddw, nullptr,
                           GEOGCN_ACT_NONE, 0, GEOGCN_GEMM_F32, need ? g : nullptr, need, st);
}
int weight_grad(Arena& ar, const WgradArgs& w, hipStream_t st) {
    if (w.precision == GEOGCN_GEMM_F32 && w.type == GEOGCN_T_F32) return weight_grad_exact(ar, w, st);
    // one narrow side: the operands are read once or twice, and terms in memory would cost more than the products (codes / terms: 440,000 x 300 x
    // 256 249 / 577 us, 60,000 x 600 x 600 180 / 245, 20,000 x 300 x 2,048 104 / 182; but 20,000 x 1,024 x 1,024 196 / 183)
    if (w.type == GEOGCN_T_F32 && w.precision == GEOGCN_GEMM_BF16X3 && std::min(w.K, w.N) <= 640 && std::max(w.K, w.N) <= 2048) {
        const float* B[1] = {static_cast<const float*>(w.dZ.p)};
        return tn_q8(ar, w.X, w.M, w.K, w.N, 1, B, w.dZ.ld, &w.dW, &w.lddw, st);
    }
    const int P = terms_of(w.type, w.precision);
    TermsJobs jx{}, jz{};
    const Planes x = make_planes(ar, w.X, w.M, w.K, 1, false, jx), dz = make_planes(ar, w.dZ, w.M, w.N, P, false, jz);
    if (const int rc = run_terms(ar, jx, 1, st)) return rc;
    if (const int rc = run_terms(ar, jz, P, st)) return rc;
    TileArgs t = tile_args();
    t.M = w.K; t.N = w.N; t.K[0] = w.M;
    t.A[0] = x.p; t.lda[0] = x.ld; t.planeA[0] = x.plane;
    t.B[0] = dz.p; t.ldb[0] = dz.ld; t.planeB[0] = dz.plane;
    t.C[0] = w.dW; t.ldc[0] = w.lddw; t.out_type = w.type; t.nc[0] = t.ncols = out_cols(w.type, w.N, w.lddw);
    return run_weight_grad(ar, t, 1, P, 1, st);
}

// the pads of an fp32 matrix's quad lie inside its pitch (checked), so whole quads can be written; a zero-sized reduction gives zeros
int zero_matrix(void* p, int type, int64_t n, int64_t cols, int64_t ld, hipStream_t st) {
    if (type == GEOGCN_T_F32) return zero_rows_async(static_cast<float*>(p), n, cols, ld, st);
    return zero_rows_async(static_cast<float*>(p), n, cols / 2, ld / 2, st);
}

// 0: go on; else the call's return code.  *have is set to what the call needs where that is missing.
int check_ws(const char* who, size_t need, const void* ws, size_t* have) {
    if (need == 0) return 0;
    const size_t got = ws ? *have : 0;
    if (got < need) *have = need;
    GEOGCN_REQUIRE(got >= need, GEOGCN_E_WORKSPACE, "%s: workspace of %zu bytes, %zu needed", who, got, need);
    GEOGCN_REQUIRE(reinterpret_cast<uintptr_t>(ws) % 256 == 0, GEOGCN_E_ALIGN, "%s: workspace not on 256 bytes", who);
    return 0;
}

}  // namespace
}  // namespace geogcn

using namespace geogcn;

extern "C" int geogcn_gated_fwd(int64_t M, int64_t K, int64_t N, int32_t type, const void* X, int64_t ldx, const void* Wg, int64_t ldwg, const void* Wu,
                                int64_t ldwu, const float* bg, const float* bu, int32_t act, void* H, int64_t ldh, int32_t keep, void* G, int64_t ldg,
                                uint8_t* Gs, void* U, int64_t ldu, uint8_t* Us, int32_t precision, void* ws, size_t* ws_bytes, void* stream) {
    const char* who = "gated_fwd";
    if (const int rc = check_dims(who, M, K, N)) return rc;
    GEOGCN_REQUIRE(ws_bytes, GEOGCN_E_NULL, "%s: ws_bytes is null", who);
    GEOGCN_REQUIRE(type == GEOGCN_T_F32 || type == GEOGCN_T_BF16, GEOGCN_E_ARG, "%s: type %d is neither fp32 nor bf16", who, type);
    GEOGCN_REQUIRE(precision >= GEOGCN_GEMM_F32 && precision <= GEOGCN_GEMM_BF16, GEOGCN_E_ARG, "%s: precision %d", who, precision);
    GEOGCN_REQUIRE(act_ok(act), GEOGCN_E_ARG, "%s: activation %d", who, act);
    GEOGCN_REQUIRE(keep == GEOGCN_KEEP_NONE || keep == GEOGCN_KEEP_FULL || keep == GEOGCN_KEEP_MX8, GEOGCN_E_ARG, "%s: keep %d", who, keep);
    FwdArgs f;
    f.M = M; f.K = K; f.N = N; f.type = type; f.precision = precision; f.keep = keep; f.act = act;
    f.X = MatIn{type, X, ldx, nullptr}; f.Wg = MatIn{type, Wg, ldwg, nullptr}; f.Wu = MatIn{type, Wu, ldwu, nullptr};
    f.bg = bg; f.bu = bu; f.H = H; f.ldh = ldh;
    f.keepP[0] = G; f.keepP[1] = U; f.ldk[0] = ldg; f.ldk[1] = ldu; f.keepS[0] = Gs; f.keepS[1] = Us;
    const bool empty = M == 0 || N == 0;
    if (!empty) {
        if (K > 0) {
            if (const int rc = check_mat(who, "X", type, X, ldx, nullptr, K)) return rc;
            if (const int rc = check_mat(who, "Wg", type, Wg, ldwg, nullptr, N)) return rc;
            if (const int rc = check_mat(who, "Wu", type, Wu, ldwu, nullptr, N)) return rc;
        }
        if (const int rc = check_mat(who, "H", type, H, ldh, nullptr, N)) return rc;
        if (keep != GEOGCN_KEEP_NONE) {
            const int kt = keep == GEOGCN_KEEP_MX8 ? GEOGCN_T_MX8 : type;
            if (const int rc = check_mat(who, "G", kt, G, ldg, Gs, N)) return rc;
            if (const int rc = check_mat(who, "U", kt, U, ldu, Us, N)) return rc;
            if (keep == GEOGCN_KEEP_FULL)
                GEOGCN_REQUIRE(out_cols(type, N, ldg) >= out_cols(type, N, ldh) && out_cols(type, N, ldu) >= out_cols(type, N, ldh), GEOGCN_E_ALIGN,
                               "%s: G and U need H's pitch", who);
        }
    }
    Arena count{nullptr};
    if (!empty)
        if (const int rc = forward(count, f, nullptr)) return rc;
    if (empty) return 0;
    if (const int rc = check_ws(who, count.used, ws, ws_bytes)) return rc;
    Arena ar{static_cast<unsigned char*>(ws), false};
    return forward(ar, f, static_cast<hipStream_t>(stream));
}

extern "C" int geogcn_gated_bwd(int64_t M, int64_t K, int64_t N, int32_t type, const void* dH, int64_t lddh, int32_t x_type, const void* X, int64_t ldx,
                                const uint8_t* Xs, const void* Wg, int64_t ldwg, const void* Wu, int64_t ldwu, int32_t kept_type, const void* G,
                                int64_t ldg, const uint8_t* Gs, const void* U, int64_t ldu, const uint8_t* Us, int32_t act, void* dX, int64_t lddx,
                                void* dWg, int64_t lddwg, void* dWu, int64_t lddwu, float* dbg, float* dbu, int32_t precision, void* ws,
                                size_t* ws_bytes, void* stream) {
    const char* who = "gated_bwd";
    if (const int rc = check_dims(who, M, K, N)) return rc;
    GEOGCN_REQUIRE(ws_bytes, GEOGCN_E_NULL, "%s: ws_bytes is null", who);
    GEOGCN_REQUIRE(type == GEOGCN_T_F32 || type == GEOGCN_T_BF16, GEOGCN_E_ARG, "%s: type %d is neither fp32 nor bf16", who, type);
    GEOGCN_REQUIRE((x_type == type || x_type == GEOGCN_T_MX8) && (kept_type == type || kept_type == GEOGCN_T_MX8), GEOGCN_E_ARG,
                   "%s: X and the kept G, U are of the block's type or 8-bit checkpoints (got %d, %d)", who, x_type, kept_type);
    GEOGCN_REQUIRE(precision >= GEOGCN_GEMM_F32 && precision <= GEOGCN_GEMM_BF16, GEOGCN_E_ARG, "%s: precision %d", who, precision);
    GEOGCN_REQUIRE(act_ok(act), GEOGCN_E_ARG, "%s: activation %d", who, act);
    GEOGCN_REQUIRE((dWg == nullptr) == (dWu == nullptr) && (dbg == nullptr) == (dbu == nullptr), GEOGCN_E_NULL,
                   "%s: the weight (bias) gradients come in pairs", who);
    BwdArgs b;
    b.M = M; b.K = K; b.N = N; b.type = type; b.precision = precision; b.act = act;
    b.dH = MatIn{type, dH, lddh, nullptr}; b.X = MatIn{x_type, X, ldx, Xs}; b.G = MatIn{kept_type, G, ldg, Gs}; b.U = MatIn{kept_type, U, ldu, Us};
    b.Wg = MatIn{type, Wg, ldwg, nullptr}; b.Wu = MatIn{type, Wu, ldwu, nullptr};
    b.dX = dX; b.lddx = lddx; b.dW[0] = dWg; b.dW[1] = dWu; b.lddw[0] = lddwg; b.lddw[1] = lddwu; b.db[0] = dbg; b.db[1] = dbu;
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (M > 0 && N > 0) {
        if (const int rc = check_mat(who, "dH", type, dH, lddh, nullptr, N)) return rc;
        if (const int rc = check_mat(who, "G", kept_type, G, ldg, Gs, N)) return rc;
        if (const int rc = check_mat(who, "U", kept_type, U, ldu, Us, N)) return rc;
        if (K > 0 && dX) {
            if (const int rc = check_mat(who, "Wg", type, Wg, ldwg, nullptr, N)) return rc;
            if (const int rc = check_mat(who, "Wu", type, Wu, ldwu, nullptr, N)) return rc;
        }
        if (K > 0 && dWg)
            if (const int rc = check_mat(who, "X", x_type, X, ldx, Xs, K)) return rc;
    }
    if (dX && M > 0 && K > 0)
        if (const int rc = check_mat(who, "dX", type, dX, lddx, nullptr, K)) return rc;
    if (dWg && K > 0 && N > 0) {
        if (const int rc = check_mat(who, "dWg", type, dWg, lddwg, nullptr, N)) return rc;
        if (const int rc = check_mat(who, "dWu", type, dWu, lddwu, nullptr, N)) return rc;
    }
    if (dbg) GEOGCN_REQUIRE(aligned16(dbg) && aligned16(dbu), GEOGCN_E_ALIGN, "%s: bias gradients not aligned", who);
    if (K == 0) { b.dX = nullptr; b.dW[0] = b.dW[1] = nullptr; }
    const bool empty = M == 0 || N == 0;
    Arena count{nullptr};
    if (!empty)
        if (const int rc = backward(count, b, nullptr)) return rc;
    if (empty) {                                             // no rows, or no units: sums over nothing
        if (b.dX && M > 0)
            if (const int rc = zero_matrix(dX, type, M, out_cols(type, K, lddx), lddx, st)) return rc;
        for (int q = 0; q < 2; ++q) {
            if (b.dW[q] && N > 0)
                if (const int rc = zero_matrix(b.dW[q], type, K, out_cols(type, N, b.lddw[q]), b.lddw[q], st)) return rc;
            if (b.db[q] && N > 0)
                if (const int rc = zero_rows_async(b.db[q], 1, N, N, st)) return rc;
        }
        return 0;
    }
    if (const int rc = check_ws(who, count.used, ws, ws_bytes)) return rc;
    Arena ar{static_cast<unsigned char*>(ws), false};
    return backward(ar, b, st);
}

extern "C" int geogcn_mx8_weight_grad(int64_t M, int64_t K, int64_t N, int32_t type, const uint8_t* X, int64_t ldx, const uint8_t* Xs, const void* dZ,
                                      int64_t lddz, void* dW, int64_t lddw, int32_t precision, void* ws, size_t* ws_bytes, void* stream) {
    const char* who = "mx8_weight_grad";
    if (const int rc = check_dims(who, M, K, N)) return rc;
    GEOGCN_REQUIRE(ws_bytes, GEOGCN_E_NULL, "%s: ws_bytes is null", who);
    GEOGCN_REQUIRE(type == GEOGCN_T_F32 || type == GEOGCN_T_BF16, GEOGCN_E_ARG, "%s: type %d is neither fp32 nor bf16", who, type);
    GEOGCN_REQUIRE(precision >= GEOGCN_GEMM_F32 && precision <= GEOGCN_GEMM_BF16, GEOGCN_E_ARG, "%s: precision %d", who, precision);
    const bool none = K == 0 || N == 0;
    if (!none) {
        if (const int rc = check_mat(who, "dW", type, dW, lddw, nullptr, N)) return rc;
        if (M > 0) {
            if (const int rc = check_mat(who, "X", GEOGCN_T_MX8, X, ldx, Xs, K)) return rc;
            if (const int rc = check_mat(who, "dZ", type, dZ, lddz, nullptr, N)) return rc;
        }
    }
    WgradArgs w{M, K, N, type, precision, MatIn{GEOGCN_T_MX8, X, ldx, Xs}, MatIn{type, dZ, lddz, nullptr}, dW, lddw};
    Arena count{nullptr};
    if (!none && M > 0)
        if (const int rc = weight_grad(count, w, nullptr)) return rc;
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (none) return 0;
    if (M == 0) return zero_matrix(dW, type, K, out_cols(type, N, lddw), lddw, st);
    if (const int rc = check_ws(who, count.used, ws, ws_bytes)) return rc;
    Arena ar{static_cast<unsigned char*>(ws), false};
    return weight_grad(ar, w, st);
}
