// 16-bit MFMA contraction core for gfx950 (v_mfma_f32_32x32x16_{f16,bf16}, sums in fp32), shared by the vocabulary
// cross entropy and the orthogonalised weight update.
//
//   D[i,j] = sum_k P(i,k) Q(j,k)        j on the lane, i in the registers of the 32x32 accumulators
//
// Each operand is stored either k-contiguous ([x][k], "N") or x-contiguous ([k][x], "T": the contraction runs over its
// leading axis).  Tiles reach LDS by global_load_lds (1 KiB pieces, lane l at byte 16 l, XOR-swizzled through the source
// address), in a ring of three or four buffers: the other tiles are in flight while one is multiplied, one barrier per tile.  T
// tiles are transposed by the LDS read itself (ds_read_b64_tr_b16).
//
// SPLIT operands carry 32-bit values as two fp16 numbers, v * s = hi + lo with s a power of two: 22 significant bits.
// They are stored with twice the columns, [row][col / 16][hi, lo][16], which serves both orientations; a k-tile is then
// 16 wide and feeds three products, lo*hi + hi*lo + hi*hi (lo*lo is below 2^-22 of the result; tiles of 64 x 64, which wait
// for memory, take it along).  Three MFMA passes against sixteen for the fp32 matrix instruction at the same flops.
//
// Bounds: rows of an N operand past its end are copies of its last row, columns of a T operand past its end are copies
// of its last 8 (both feed only outputs that are not stored); k-tiles are whole, so operands are padded to 32 columns
// (16 k when SPLIT) by their producers; T operands may name a limit on their k rows, past which the last row is read
// against zeros of the other operand.
#pragma once
#include "common.h"

namespace mma16 {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));

enum { F16 = 0, BF16 = 1 };

// ---- element conversions (round to nearest even; 16-bit values as raw bits) ------------------------------------------
template <int ELT>
__device__ __forceinline__ short to_bits(float v) {
    if (ELT == BF16) {
        __bf16 b = (__bf16)v;
        return __builtin_bit_cast(short, b);
    }
    _Float16 h = (_Float16)v;
    return __builtin_bit_cast(short, h);
}
template <int ELT>
__device__ __forceinline__ float from_bits(short b) {
    if (ELT == BF16) return (float)__builtin_bit_cast(__bf16, b);
    return (float)__builtin_bit_cast(_Float16, b);
}
// v = hi + lo in fp16; an infinite or not-a-number v stays that in hi.  v is made a rounded fp32 number first: where it is
// a product, the compiler may round that straight to fp16 for hi and by way of fp32 for lo's difference, which are not
// always the same number (an error of a whole fp16 step in one of some thousand values).
__device__ __forceinline__ void split16(float v, short& hi, short& lo) {
    asm("" : "+v"(v));
    const _Float16 h = (_Float16)v;
    const _Float16 l = (_Float16)(v - (float)h);
    hi = __builtin_bit_cast(short, h);
    lo = __builtin_bit_cast(short, l);
}
// first of the two stored columns of logical column c of a SPLIT matrix (the other is 16 further on)
__host__ __device__ __forceinline__ int64_t split_col(int64_t c) { return (c >> 4) * 32 + (c & 15); }

template <int ELT>
__device__ __forceinline__ f32x16 mfma(s16x8 a, s16x8 b, f32x16 c) {
    if (ELT == BF16) return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// accumulator register e of lane half h is row (e & 3) + 8 (e >> 2) + 4 h of the 32x32 tile
__device__ __forceinline__ int acc_row(int e, int h) { return (e & 3) + 8 * (e >> 2) + 4 * h; }

// 16 bytes per lane from `src` to 1 KiB of LDS at `dst` (wave-uniform), asynchronously.  Written as assembly because the
// compiler, where it knows of such loads, waits for all of them before every transposing LDS read; it has no output
// registers, and contract() waits for it by count.  m0 is reserved, so that no clobber list takes it: it has no other
// user, since a kernel's tiles all come this way, or all through the builtin (the generated code has no kernel with both).
__device__ __forceinline__ void dma16(const short* src, short* dst) {
    const unsigned at = __builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)(__attribute__((address_space(3))) short*)dst);
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(at), "v"(src) : "memory");
}

struct View {               // one operand
    const short* p;
    int64_t ld;             // stored elements between rows
    int n;                  // extent of the i or j axis (logical)
    int klim;               // T: number of k rows that exist
};

template <int NX, bool T, bool SPLIT>
struct Operand {
    static constexpr int PIECES = NX / 16;                    // 1 KiB each
    static constexpr int NXS = NX * (SPLIT ? 2 : 1);          // T: stored columns per k row of the tile
    static constexpr int KT = SPLIT ? 16 : 32;                // logical k per tile
    static constexpr int CPR = NXS / 8, KPP = 512 / NXS;      // T: 16-byte chunks per k row, k rows per piece
    static_assert(NX % 64 == 0 && NXS <= 512, "tile width not built");

    // N: rows of four 16-byte slots.  The 16-lane groups of a ds_read_b128 read rows whose (row / 4) % 8 are
    // {0,3,5,6} or {1,2,4,7} for each row % 4; this maps them to four different slots.
    __device__ static int swz_n(int row) {
        const int q = (row >> 2) & 7;
        return (q & 3) ^ ((q >> 2) * 3);
    }
    // T: 32-byte granules (16 x of one k).  A half-wave reads two granules of each of four k rows: granules g, g+1
    // (SPLIT: g, g+2, hi and lo alternate); the XOR spreads them over the eight granules of a 256-byte bank row.
    __device__ static int swz_t(int k) {
        if (SPLIT) return (k & 1) | ((k & 2) << 1);
        return NXS >= 128 ? 2 * (k & 3) : (k & 2);
    }
    __device__ static const short* source(const View& v, int x0, int kt, int piece, int lane) {
        if (!T) {
            const int row = piece * 16 + (lane >> 2);
            const int slot = (lane & 3) ^ swz_n(row);
            return v.p + (int64_t)min(x0 + row, v.n - 1) * v.ld + (int64_t)kt * 32 + slot * 8;
        }
        const int kr = piece * KPP + lane / CPR;
        const int chunk = (lane % CPR) ^ (swz_t(kr) << 1);
        const int k = min(kt * KT + kr, v.klim - 1);
        return v.p + (int64_t)k * v.ld + min(x0 * (SPLIT ? 2 : 1) + chunk * 8, v.n * (SPLIT ? 2 : 1) - 8);
    }
    // elements a source pointer moves per k-tile
    __device__ static int64_t step(const View& v) { return T ? (int64_t)KT * v.ld : 32; }
    // eight k values of row w0 + (lane & 31): k = 8 (lane >> 5) + 0..7 of k-chunk kc (SPLIT: kc is the plane)
    __device__ static s16x8 frag(const short* img, int w0, int kc, int lane) {
        const int h = lane >> 5;
        if (!T) {
            const int row = w0 + (lane & 31);
            return *reinterpret_cast<const s16x8*>(img + row * 32 + (((kc * 2 + h) ^ swz_n(row)) * 8));
        }
        const int li = lane & 15;
        const int k = (SPLIT ? 0 : kc * 16) + 8 * h + (li >> 2);
        const int blk = (w0 >> 4) + ((lane >> 4) & 1);
        const int gran = (SPLIT ? 2 * blk + kc : blk) ^ swz_t(k);
        const short* a = img + k * NXS + gran * 16 + (li & 3) * 4;
        typedef __attribute__((address_space(3))) s16x4* lp;
        const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)a);
        const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(a + 4 * NXS));
        return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    }
};

// A workgroup of WI x WJ wavefronts, each holding TI x TJ accumulators of 32x32, with a ring of STAGES k-tiles.
// SPREAD: the loads of a later k-tile are issued between the matrix instructions, at raised priority, which suits
// workgroups that share a CU (256 x 128: 223 against 243 us for 7424 x 10000 x 512 in fp32); else ahead of them, with the
// LDS reads spread instead (256 x 256: 1076 against 1090 us for 8192 x 32768 x 2048 in bf16, gradients 941 against 1041).
// KG: groups of WI x WJ wavefronts that share a tile's k-tiles in turn and add their sums through LDS at the end, for launches
// that leave CUs idle: a k-tile's way through LDS takes some 750 cycles however deep the ring (eight buffers instead of
// three changed nothing).  A launch for 512 x 512 x 512, 64 workgroups: 11.3 -> 9.1 us.
template <int WI_, int WJ_, int TI_, int TJ_, int STAGES_, bool SPREAD_, int KG_ = 1>
struct Tile {
    static constexpr int WI = WI_, WJ = WJ_, TI = TI_, TJ = TJ_, STAGES = STAGES_;
    static constexpr bool SPREAD = SPREAD_;
    static constexpr int KG = KG_;
    static constexpr int EU = KG > 1 ? 4 : 2;                 // wavefronts per SIMD that the registers are for
    static constexpr int BI = 32 * WI * TI, BJ = 32 * WJ * TJ;
    static constexpr int WAVES = WI * WJ, GROUP = 64 * WAVES, THREADS = GROUP * KG;
    static constexpr int STAGE = (BI + BJ) * 32;              // 16-bit elements of one ring buffer
    static constexpr int LDS_BYTES = KG * STAGES * STAGE * 2;
    static_assert((KG - 1) * GROUP * TI * TJ * 64 <= LDS_BYTES, "the groups' sums do not fit");
};
typedef Tile<2, 4, 4, 2, 4, false> Wide;    // 256 x 256: 128 KiB of LDS, one workgroup per CU
typedef Tile<2, 2, 4, 2, 3, true> Big;     // 256 x 128: 72 KiB, two workgroups per CU
typedef Tile<2, 2, 2, 2, 3, true> Mid;     // 128 x 128: 48 KiB, three
typedef Tile<2, 2, 1, 1, 3, false> Small;      //  64 x  64: 24 KiB
typedef Tile<2, 2, 1, 1, 3, false, 4> Deep;    //  64 x  64 by four groups: 96 KiB

// Waits until at most min(ahead, MOST) k-tiles of PER loads each are in flight and this wavefront's LDS reads are done,
// then for the workgroup.
template <int MOST, int PER>
__device__ __forceinline__ void wait_tiles(int ahead) {
    static_assert(MOST * PER < 64, "vmcnt counts to 63");
    if (MOST == 0 || ahead >= MOST) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(MOST * PER) : "memory");
    else wait_tiles<(MOST > 0 ? MOST - 1 : 0), PER>(ahead);
}

// Sums k-tiles [kt0, kt1) of the tile at (i0, j0); the sums are the first group's.  Ends behind a barrier: the caller may
// reuse `lds`.
template <class C, int ELT, bool TP, bool TQ, bool SPLIT>
__device__ __forceinline__ void contract(const View& P, const View& Q, int i0, int j0, int kt0, int kt1, short* lds,
                                         f32x16 (&acc)[C::TI][C::TJ]) {
    using OpP = Operand<C::BI, TP, SPLIT>;
    using OpQ = Operand<C::BJ, TQ, SPLIT>;
    constexpr int W = C::WAVES, S = C::STAGES, NPW = (OpP::PIECES + OpQ::PIECES) / W;
    static_assert(OpP::PIECES % W == 0 && OpQ::PIECES % W == 0, "pieces do not divide over the wavefronts");
    constexpr int KG = C::KG;
    const int lane = threadIdx.x & 63;
    const int group = KG > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x / C::GROUP) : 0;
    const int wave = __builtin_amdgcn_readfirstlane((threadIdx.x % C::GROUP) >> 6);
    const int wi = wave / C::WJ, wj = wave % C::WJ;
#pragma unroll
    for (int ti = 0; ti < C::TI; ++ti)
#pragma unroll
        for (int tj = 0; tj < C::TJ; ++tj)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[ti][tj][e] = 0.f;

    const short* src[NPW];
    auto seek = [&](int kt) {
#pragma unroll
        for (int i = 0; i < NPW; ++i) {
            const int piece = i * W + wave;
            src[i] = i * W < OpP::PIECES ? OpP::source(P, i0, kt, piece, lane)
                                         : OpQ::source(Q, j0, kt, piece - OpP::PIECES, lane);
        }
    };
    const int64_t stepP = OpP::step(P) * KG, stepQ = OpQ::step(Q) * KG;
    // the first k-tile that reaches past a T operand's rows: its addresses are clamped one by one
    const int ragged = min(TP ? P.klim / OpP::KT : kt1, TQ ? Q.klim / OpQ::KT : kt1);
    // one of this wavefront's pieces of k-tile kt
    auto issue_piece = [&](short* buf, int i) {
        const int piece = i * W + wave;
        if (TP || TQ)
            dma16(src[i], buf + piece * 512);
        else
            __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)src[i],
                                             (__attribute__((address_space(3))) void*)(buf + piece * 512), 16, 0, 0);
        src[i] += i * W < OpP::PIECES ? stepP : stepQ;
    };
    auto issue = [&](short* buf, int kt) {
        if ((TP || TQ) && kt >= ragged) seek(kt);
#pragma unroll
        for (int i = 0; i < NPW; ++i) issue_piece(buf, i);
    };
    // Two halves (k-chunks; SPLIT: planes) of fragments, the products over them, and between the products the loads of a
    // later tile when `more`.
    auto compute = [&](const short* ip, short* buf, bool more) {
        const short* iq = ip + C::BI * 32;
        s16x8 a[2][C::TI], b[2][C::TJ];
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
#pragma unroll
            for (int tj = 0; tj < C::TJ; ++tj) b[hf][tj] = OpQ::frag(iq, (wj * C::TJ + tj) * 32, hf, lane);
#pragma unroll
            for (int ti = 0; ti < C::TI; ++ti) a[hf][ti] = OpP::frag(ip, (wi * C::TI + ti) * 32, hf, lane);
        }
        if (C::SPREAD) __builtin_amdgcn_sched_barrier(0);
        // one 32x32 block per wavefront: the fourth product, lo*lo, costs nothing there, and small matrices have no long sums
        // in which the other roundings drown its loss
        constexpr int TERMS = SPLIT ? (C::TI * C::TJ == 1 ? 4 : 3) : 2, N = TERMS * C::TI * C::TJ, EVERY = N / NPW > 0 ? N / NPW : 1;
        static_assert(!C::SPREAD || N >= NPW, "not every piece would be issued");
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int t = n / (C::TI * C::TJ), ti = n / C::TJ % C::TI, tj = n % C::TJ;
            // SPLIT: hi*hi, hi*lo, lo*hi, lo*lo
            acc[ti][tj] = mfma<ELT>(a[SPLIT ? t >> 1 : t][ti], b[SPLIT ? t & 1 : t][tj], acc[ti][tj]);
            if (C::SPREAD && n % EVERY == 0 && n / EVERY < NPW) {
                __builtin_amdgcn_sched_barrier(0);
                if (more) issue_piece(buf, n / EVERY);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    };
    // group g takes the tiles kt0 + g, kt0 + g + KG, ...: `mine` of them, in as many rounds as group 0 needs
    const int first = kt0 + group, rounds = (kt1 - kt0 + KG - 1) / KG;
    const int mine = KG == 1 ? rounds : max(0, (kt1 - first + KG - 1) / KG);
    short* const ring = lds + group * S * C::STAGE;
    short* rd = ring;                          // the buffer of this round's tile
    short* wr = ring + (S - 1) * C::STAGE;     // the buffer of the tile S - 1 rounds later
#pragma unroll
    for (int t = 0; t < S - 1; ++t)
        if (t < mine) {
            if (t == 0) seek(first);
            issue(ring + t * C::STAGE, first + t * KG);
        }
    for (int it = 0; it < rounds; ++it) {
        // this wavefront's pieces of its tile have landed (those of later tiles may stay in flight, loads retire in order)
        // and it is done reading the buffer that the next loads go to; the barrier says so for all wavefronts
        wait_tiles<S - 2, NPW>(mine - 1 - it);
        __builtin_amdgcn_sched_barrier(0);
        const bool more = it + S - 1 < mine;
        const int later = first + (it + S - 1) * KG;
        if (C::SPREAD) {
            if ((TP || TQ) && more && later >= ragged) seek(later);
            __builtin_amdgcn_s_setprio(1);
            compute(rd, wr, more);
            __builtin_amdgcn_s_setprio(0);
        } else {
            if (more) issue(wr, later);
            __builtin_amdgcn_sched_barrier(0);
            if (KG == 1 || it < mine) compute(rd, wr, more);
            // the first half's LDS reads, then one read between matrix instructions
            constexpr int READS = C::TI * (TP ? 2 : 1) + C::TJ * (TQ ? 2 : 1);
            __builtin_amdgcn_sched_group_barrier(0x100, READS, 0);
#pragma unroll
            for (int i = 0; i < READS; ++i) {
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
            }
            __builtin_amdgcn_sched_group_barrier(0x008, 4 * C::TI * C::TJ, 0);      // the rest
        }
        __builtin_amdgcn_sched_barrier(0);
        wr = rd;
        rd = rd == ring + (S - 1) * C::STAGE ? ring : rd + C::STAGE;
    }
    __syncthreads();
    if (KG > 1) {
        constexpr int PER = C::TI * C::TJ * 16 * C::GROUP;       // floats of one group
        float* const red = reinterpret_cast<float*>(lds) + threadIdx.x % C::GROUP;
        if (group > 0) {
#pragma unroll
            for (int e = 0; e < C::TI * C::TJ * 16; ++e)
                red[(group - 1) * PER + e * C::GROUP] = acc[e / 16 / C::TJ][e / 16 % C::TJ][e % 16];
        }
        __syncthreads();
        if (group == 0) {
#pragma unroll
            for (int g = 0; g < KG - 1; ++g)
#pragma unroll
                for (int e = 0; e < C::TI * C::TJ * 16; ++e)
                    acc[e / 16 / C::TJ][e / 16 % C::TJ][e % 16] += red[g * PER + e * C::GROUP];
        }
        __syncthreads();
    }
}

// The same tile sum from fp32 operands on the fp32 matrix instruction (v_mfma_f32_32x32x2_f32, the same accumulators), for
// operands whose entries are too far apart for pairs.  Elements past an operand's k limit count as zero, rows past its end
// are copies of its last.  k-tiles of 32 in LDS, rows 33 apart, so that reads and both orders of writes meet no bank twice;
// loads are neither ahead nor wide, and nothing is assumed of their alignment.
struct View32 {             // one fp32 operand
    const float* p;
    int64_t ld;             // elements between rows of the stored matrix
    const int* order;       // N: where row x is stored; nullable
    int n;                  // extent of the i or j axis
};
template <int NX, int THREADS, bool T>
__device__ __forceinline__ void stage32(const View32& v, int x0, int k0, int klim, float* img) {
    constexpr int BATCH = 16, STEP = T ? THREADS / NX : THREADS / 32;      // loads in flight; rows between a thread's elements
    static_assert(NX * 32 % (THREADS * BATCH) == 0 && (!T || THREADS % NX == 0), "elements do not divide over the threads");
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));        // addresses are made here each time: kept over the k-tiles they cost other code its registers
    const int fix = T ? tid % NX : tid % 32, var = T ? tid / NX : tid / 32;
    const int at = T ? min(x0 + fix, v.n - 1) : min(k0 + fix, klim - 1);   // always inside; zeros are put in afterwards
#pragma unroll 1
    for (int i = 0; i < NX * 32 / THREADS; i += BATCH) {
        float q[BATCH];
#pragma unroll
        for (int e = 0; e < BATCH; ++e) {
            const int r = var + (i + e) * STEP;
            const int row = T ? min(k0 + r, klim - 1) : min(x0 + r, v.n - 1);
            q[e] = v.p[(int64_t)(!T && v.order ? v.order[row] : row) * v.ld + at];
        }
#pragma unroll
        for (int e = 0; e < BATCH; ++e) {
            const int r = var + (i + e) * STEP, k = T ? r : fix;
            img[(T ? fix : r) * 33 + k] = k0 + k < klim ? q[e] : 0.f;
        }
    }
}
// k in [k0, k1); elements from klim on are zero.  Ends behind a barrier.
template <class C, bool TP, bool TQ>
__device__ __forceinline__ void contract32(const View32& P, const View32& Q, int i0, int j0, int k0, int k1, int klim, short* lds,
                                           f32x16 (&acc)[C::TI][C::TJ]) {
    static_assert(C::KG == 1 && (C::BI + C::BJ) * 33 * 4 <= C::LDS_BYTES, "the tile does not fit");
    float* const ip = reinterpret_cast<float*>(lds);
    float* const iq = ip + C::BI * 33;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wi = wave / C::WJ, wj = wave % C::WJ, h = lane >> 5;
#pragma unroll
    for (int ti = 0; ti < C::TI; ++ti)
#pragma unroll
        for (int tj = 0; tj < C::TJ; ++tj)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[ti][tj][e] = 0.f;
    klim = min(klim, k1);
    for (int k = k0; k < klim; k += 32) {
        stage32<C::BI, C::THREADS, TP>(P, i0, k, klim, ip);
        stage32<C::BJ, C::THREADS, TQ>(Q, j0, k, klim, iq);
        __syncthreads();
        const float* a = ip + (wi * C::TI * 32 + (lane & 31)) * 33 + h;
        const float* b = iq + (wj * C::TJ * 32 + (lane & 31)) * 33 + h;
#pragma unroll 2
        for (int kk = 0; kk < 32; kk += 2) {
            float av[C::TI], bv[C::TJ];
#pragma unroll
            for (int ti = 0; ti < C::TI; ++ti) av[ti] = a[ti * 32 * 33 + kk];
#pragma unroll
            for (int tj = 0; tj < C::TJ; ++tj) bv[tj] = b[tj * 32 * 33 + kk];
#pragma unroll
            for (int ti = 0; ti < C::TI; ++ti)
#pragma unroll
                for (int tj = 0; tj < C::TJ; ++tj)
                    acc[ti][tj] = __builtin_amdgcn_mfma_f32_32x32x2f32(av[ti], bv[tj], acc[ti][tj], 0, 0, 0);
        }
        __syncthreads();
    }
    __syncthreads();
}

// Workgroup -> tile.  Workgroup ids go round-robin to the 8 XCDs, each with an L2 of its own: XCD x takes the x-th
// eighth of the tile sequence, and the sequence walks blocks of eight i-tiles by all j, so that the workgroups that run
// on one XCD at a time share operand rows.  A performance assumption only.
struct Map {
    int ni, nj, nz, per;       // per: tiles per XCD
};
inline unsigned make_map(Map& m, int ni, int nj, int nz) {
    m.ni = ni; m.nj = nj; m.nz = nz;
    const int64_t total = (int64_t)ni * nj * nz;
    m.per = (int)((total + 7) / 8);
    return (unsigned)m.per * 8u;
}
__device__ __forceinline__ bool tile_of(const Map& m, unsigned block, int& ti, int& tj, int& z) {
    if ((int)(block >> 3) >= m.per) return false;            // (no tiles at all: per is 0)
    const int t = (int)(block & 7) * m.per + (int)(block >> 3);
    const int plane = m.ni * m.nj;
    z = t / plane;
    if (z >= m.nz) return false;
    int u = t - z * plane;
    const int band = u / (8 * m.nj);
    u -= band * 8 * m.nj;
    const int rows = min(8, m.ni - band * 8);
    ti = band * 8 + u % rows;
    tj = u / rows;
    return true;
}

}  // namespace mma16
