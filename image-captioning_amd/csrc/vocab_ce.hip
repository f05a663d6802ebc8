// Softmax cross entropy of a vocabulary projection without keeping the logits, and its gradients.
//
//   z = x W^T + b;  nll_r = log(sum_v exp z_rv) - z_rt;  G_rv = (exp(z_rv - lse_r) - [v = t_r]) g_r
//   dx = G W,  dW = G^T x,  db = sum_r G_r
//
// Forward: rows with a counted target are compacted, the product runs tile by tile on the matrix cores and each tile
// leaves (max, sum of exp) per row.  Backward: G is rebuilt for one piece of the vocabulary at a time from x, W and the
// rows' log-sum-exp, and contracted with W and x while it is in the caches.  Four products of 2 M V K flops in all for
// loss and gradients, bound by the matrix cores at large sizes and by reading W at few rows.
// fp32 operands are split into two fp16 numbers (mma16.h), but for batches of at most 64 rows, which have kernels of their
// own that read W as it is, and for rows too far apart (FAR below); 16-bit operands are multiplied as they are.  Sums, softmax
// statistics and the partial sums of the gradients are fp32.  G takes the operands' 16-bit type (fp16 scaled by 2^14,
// so that probabilities down to 2^-28 stay normal).  That rounding averages out in sums over rows or words, except
// at the targets, whose entries are near -g_r: what it takes off them is carried beside G and added to dx, and to dW up to
// 64 rows, and db sums the unrounded values.  Against rounding of the results alone: dx and db 1.0, dW 1.0 - 1.3 times.
// Every sum has a fixed order: results repeat bit for bit.
#include "mma16.h"
#include <math.h>
#include <type_traits>

using namespace mma16;

namespace {

constexpr float L2E = 1.44269504088896340736f, LN2 = 0.69314718055994530942f;
constexpr int G_EXP = 14;                        // G is stored times 2^14 where it is fp16 numbers, and as it is in fp32 and bf16
constexpr size_t PIECE_BYTES = (size_t)512 << 20;
constexpr int FEW = 64;                          // rows of fp32 up to which W is read as it is
constexpr int FEW_WAVES = 1024;                  // from so many words / 32 on, no sum is shared by wavefronts
constexpr int AMAX_BLOCKS = 256;
// Pairs of fp16 numbers carry a matrix with one power of two, which brings its largest entry to [2^14, 2^15): a value is
// off by 2^-23 of itself or, since fp16 ends in steps of 2^-24, by 2^-39 of that largest entry.  A row whose own largest
// entry is at least 2^-16 of it thus keeps 2^-23 of its largest entry, as it would with a power of two of its own.  Where
// a row that is not zero lies below that (a word far larger than the others but masked, say), or W holds infinities, whose
// low part would be NaN (a logit of -inf is a number), x, W and G stay in fp32 and the products take the fp32 matrix
// instruction (10240 x 10000 x 512, loss and gradients: 1.4 -> 7.7 ms).  Found on the device, in the pass that takes the
// maxima; the kernels hold both forms.
constexpr float FAR = 65536.f;

// dx has as many row tiles as there are counted rows, which only the device knows: the number of parts for each possible
// number of row tiles goes along (one part beyond 64 of them, 16384 rows, where there are tiles enough).
struct Splits {
    unsigned char s[64];
};
__host__ __device__ __forceinline__ int splits_of(const Splits& t, int tiles) {
    return tiles < 1 || tiles > 64 ? 1 : t.s[tiles - 1];
}

// ---- memory plan (host and device agree through it) ------------------------------------------------------------------
struct Plan {
    int M, V, K, Mp, Vp, Kp, split, elt;         // Mp: rows and Vp: words rounded up to 256, Kp: width to 32
    int xs;                                      // stored columns of the packed operands: Kp, or 2 Kp when split
    bool pack_w;
    int piece, pieces;                           // vocabulary words per piece (a multiple of 256)
    Splits sx;                                   // contraction splits of dx, by row tiles
    int64_t dx_tiles;                            // most workgroups of a dx launch, and
    int64_t dx_rows;                             // most rows of partial sums
    int sw;                                      // contraction splits of dW
    bool wide_z, wide_dx, wide_dw;               // tiles of 256 x 256 for the logits, dx and dW
    bool few_z;                                  // tiles of 128 x 128 for the logits
    bool by_row;                                 // fp32 and no backward call: every row of x and W has a scale of its own
    bool few;                                    // fp32 and at most 64 rows: kernels of their own
    int few_rows;                                // rows of z and G there: 16, 32 or 64
    int few_split, few_words;                    // parts of the dx contraction, and words of a part
    int z_words, z_rows;                         // the logits' tile
    size_t o_order, o_slot, o_tgt, o_lse, o_dlt, o_b2, o_x, o_w, o_z, o_sx, o_sw, saved;
    size_t o_part, o_amax, fwd;
    size_t o_rw, o_rest, o_g, o_dx, o_dw, o_db, bwd;
};

size_t take(size_t& at, size_t bytes) {
    const size_t o = at;
    at += (bytes + 255) & ~(size_t)255;
    return o;
}

// Contractions with few output tiles and a long sum are cut into s parts.  Workgroups run in rounds of `slots`; a part takes
// 1 / s of the time.  Starting a tile costs about 6 k-tiles of time, writing partial sums and adding them later 16 more.
int splits_for(int64_t tiles, int kt, int slots) {
    int best = 1;
    double least = 1e300;
    for (int s = 1; s <= 128 && kt / s >= 8; s += s < 16 ? 1 : 16) {
        const double t = (double)((tiles * s + slots - 1) / slots) * ((kt + s - 1) / s + (s > 1 ? 22 : 6));
        if (t < least * 0.97) least = t, best = s;
    }
    return best;
}

// Tiles of 256 x 256 when the contraction is long enough to make up for an epilogue that nothing overlaps (from 48 k-tiles
// on: 1076 against 1213 us at 64, 243 against 223 at 32) and there is one for every CU; else 256 x 128, two to a CU.
bool wide_pays(int64_t wide_tiles, int kt) { return kt >= 48 && wide_tiles >= 256; }

bool make_plan(const capdec_vocab_ce* a, Plan& p) {
    if (!a || a->M < 1 || a->V < 1 || a->K < 1 || a->dtype < 0 || a->dtype > 2) return false;
    if (a->M > (1 << 24) || a->V > (1 << 24) || a->K > (1 << 20)) return false;
    p = Plan{};
    p.M = a->M; p.V = a->V; p.K = a->K;
    p.Mp = (a->M + 255) / 256 * 256;
    p.Vp = (a->V + 255) / 256 * 256;
    // a launch has less than 2^32 work-items; the logits take one for 128 of them, in workgroups of up to 512, eight of which
    // may be added to make their number a multiple of 8
    if ((int64_t)p.Mp * p.Vp > ((int64_t)1 << 39) - ((int64_t)1 << 19)) return false;
    p.Kp = (a->K + 31) / 32 * 32;
    p.split = a->dtype == CAPDEC_F32;
    p.elt = a->dtype == CAPDEC_BF16 ? BF16 : F16;
    p.xs = p.Kp * (p.split ? 2 : 1);
    // 16-bit weights are read where they are when their rows are made of whole k-tiles of aligned vectors
    p.pack_w = p.split || a->K % 32 != 0 || a->ldw % 8 != 0 || !capdec_aligned16(a->W);
    size_t at = 256;
    p.o_order = take(at, (size_t)p.M * 4);
    p.o_slot = take(at, (size_t)p.M * 4);
    p.o_tgt = take(at, (size_t)p.Mp * 4);
    p.o_lse = take(at, (size_t)p.Mp * 4);
    p.o_dlt = take(at, (size_t)p.Mp * 4);
    if (p.split && p.M <= FEW) {
        p.few = true;
        p.few_rows = p.M <= 16 ? 16 : p.M <= 32 ? 32 : 64;
        p.o_x = take(at, (size_t)p.few_rows * p.Kp * 4);
        p.o_z = take(at, (size_t)p.few_rows * p.Vp * 4);
        p.saved = at;
        at = 256;
        p.o_part = take(at, (size_t)p.few_rows * (p.Vp / 32) * 8);
        p.fwd = at;
        // about 1024 workgroups for dx, each of them 64 columns by at least 128 words
        const int cols = (p.Kp + 63) / 64;
        int n = 1024 / cols < 1 ? 1 : 1024 / cols > 255 ? 255 : 1024 / cols;
        p.few_words = ((p.Vp + n - 1) / n + 127) / 128 * 128;
        p.few_split = (p.Vp + p.few_words - 1) / p.few_words;
        at = 256;
        p.o_rw = take(at, (size_t)p.Mp * 4);
        p.o_g = take(at, (size_t)p.few_rows * p.Vp * 4);
        p.o_dx = take(at, (size_t)p.few_split * p.few_rows * p.Kp * 4);
        p.bwd = at;
        return true;
    }
    p.o_b2 = take(at, (size_t)p.Vp * 4);
    p.o_x = take(at, (size_t)p.Mp * p.xs * 2);
    p.o_w = p.pack_w ? take(at, (size_t)p.V * p.xs * 2) : 0;
    p.by_row = p.split && a->loss_only;
    if (p.by_row) {
        p.o_sx = take(at, (size_t)p.Mp * 4);
        p.o_sw = take(at, (size_t)p.Vp * 4);
    }
    p.saved = at;

    at = 256;
    p.wide_z = wide_pays((int64_t)(p.Mp / 256) * (p.Vp / 256), p.xs / 32);
    p.few_z = !p.wide_z && (int64_t)(p.Mp / 128) * (p.Vp / 256) < 512;
    p.z_words = p.few_z ? Mid::BI : p.wide_z ? Wide::BI : Big::BI;
    p.z_rows = p.few_z ? Mid::BJ : p.wide_z ? Wide::BJ : Big::BJ;
    p.o_part = take(at, (size_t)(p.Vp / p.z_words) * p.Mp * 8);
    p.o_amax = take(at, 2 * AMAX_BLOCKS * 8);
    p.fwd = at;

    const int es = p.split ? 4 : 2;
    int64_t most = (int64_t)(PIECE_BYTES / ((size_t)p.Mp * es)) / 256 * 256;
    if (most < 256) most = 256;
    p.pieces = (int)((p.Vp + most - 1) / most);
    p.piece = ((p.Vp + p.pieces - 1) / p.pieces + 255) / 256 * 256;
    p.pieces = (p.Vp + p.piece - 1) / p.piece;
    const int kt = p.split ? 16 : 32;
    const int64_t row_tiles = p.Mp / 256, word_tiles = p.piece / 256;
    auto grad = [&](int64_t tiles, int n, int& split) {      // tiles of 256 along the first axis
        const int s2 = splits_for(tiles * ((p.Kp + 127) / 128), n, 512), s1 = splits_for(tiles * ((p.Kp + 255) / 256), n, 256);
        const bool wide = p.Kp % 256 == 0 && wide_pays(tiles * (p.Kp / 256) * s1, n / s1);
        split = wide ? s1 : s2;
        return wide;
    };
    int full;
    p.wide_dx = grad(row_tiles, p.piece / kt, full);
    p.wide_dw = grad(word_tiles, p.Mp / kt, p.sw);
    const int cols = p.wide_dx ? p.Kp / 256 : (p.Kp + 127) / 128;
    p.dx_tiles = row_tiles * cols;
    p.dx_rows = p.Mp;
    for (int t = 1; t <= 64; ++t) {
        p.sx.s[t - 1] = (unsigned char)splits_for((int64_t)t * cols, p.piece / kt, p.wide_dx ? 256 : 512);
        if (t > row_tiles) continue;
        const int64_t n = (int64_t)t * p.sx.s[t - 1];
        if (n * cols > p.dx_tiles) p.dx_tiles = n * cols;
        if (n * 256 > p.dx_rows) p.dx_rows = n * 256;
    }
    at = 256;
    p.o_rw = take(at, (size_t)p.Mp * 4);
    p.o_rest = take(at, (size_t)p.Mp * 4);
    p.o_g = take(at, (size_t)p.Mp * p.piece * es);
    p.o_dx = take(at, (size_t)p.dx_rows * p.Kp * 4);
    p.o_dw = p.sw > 1 ? take(at, (size_t)p.sw * p.piece * p.Kp * 4) : 0;
    p.o_db = a->bias ? take(at, (size_t)(p.Mp / 128) * p.piece * 4) : 0;
    p.bwd = at;
    return true;
}

struct Head {               // first 256 bytes of the saved buffer
    int count;              // rows with a counted target
    int ex, ew;             // split operands: x and W are packed times 2^ex and 2^ew
    int far;                // fp32 operands that are multiplied as they are; the packed x is fp32 then, W is not packed
};
struct BwdHead {            // first 256 bytes of the backward workspace (upstream gradients of the rows)
    float factor;           // what dx, dW and db are to be multiplied by
};
struct Upstream {           // where that factor comes from: a BwdHead, or one scalar (NULL: 1) for the sum or mean of the rows
    const BwdHead* bh;
    const float* grad;
    int mean;
    int gexp;               // G_EXP, or 0 where G is not fp16 numbers
};
__device__ __forceinline__ float factor_of(const Upstream& u, const Head* head) {
    if (u.bh) return u.bh->factor;
    if (head->count == 0) return 0.f;
    return ldexpf((u.grad ? u.grad[0] : 1.f) / (u.mean ? (float)head->count : 1.f), head->far ? 0 : -u.gexp);
}

// power of two that brings amax to [2^14, 2^15), denormal numbers below it (-113 .. 141, more than one fp32 number holds)
__device__ __forceinline__ int scale_exp(float amax) {
    const unsigned bits = __float_as_uint(amax);
    return bits == 0 ? 0 : 14 - ((int)(bits >> 23) - 127);
}
__device__ __forceinline__ float pow2(int e) { return ldexpf(1.f, e); }

// ---- rows with a counted target -------------------------------------------------------------------------------------
__device__ __forceinline__ float load_as_f32(const void* p, int64_t i, int dtype) {
    if (dtype == CAPDEC_F32) return ((const float*)p)[i];
    const short b = ((const short*)p)[i];
    return dtype == CAPDEC_BF16 ? from_bits<BF16>(b) : from_bits<F16>(b);
}

struct ScanArgs {
    const int64_t* targets;
    int M, V, K;
    int64_t ignore;
    Head* head;
    int *order, *slot, *tgt;
    const float* x; int64_t ldx;          // split operands: also the largest finite magnitudes of x (counted rows) and W
    const float* W; int64_t ldw;
    int nparts, vec;
    float2* part;                         // [2][AMAX_BLOCKS]: largest magnitude; that of the row where it is least, or 0
};

// The first workgroup compacts the rows: stable, 4096 targets per round.
__device__ void compact(const ScanArgs& a) {
    __shared__ int wsum[16];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int done = 0;
    for (int base = 0; base < a.M; base += 4096) {
        int64_t t[4];
        int n = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int r = base + threadIdx.x * 4 + k;
            t[k] = r < a.M ? a.targets[r] : a.ignore;
            n += t[k] != a.ignore;
        }
        int pre = n;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int v = __shfl_up(pre, o, 64);
            if (lane >= o) pre += v;
        }
        if (lane == 63) wsum[wave] = pre;
        __syncthreads();
        int before = 0, all = 0;
#pragma unroll
        for (int w = 0; w < 16; ++w) {
            if (w < wave) before += wsum[w];
            all += wsum[w];
        }
        int s = done + before + pre - n;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int r = base + threadIdx.x * 4 + k;
            if (r >= a.M) break;
            if (t[k] != a.ignore) {
                a.order[s] = r;
                a.tgt[s] = (t[k] >= 0 && t[k] < a.V) ? (int)t[k] : -1;    // -1: outside the vocabulary, the row's loss is NaN
                a.slot[r] = s++;
            } else {
                a.slot[r] = -1;
            }
        }
        done += all;
        __syncthreads();
    }
    if (threadIdx.x == 0) {
        a.head->count = done;
        a.head->ex = a.head->ew = a.head->far = 0;
    }
}

// The others take the maxima, one partial each: a wavefront reads four rows at a time.  Beside the largest magnitude the
// least of the rows' own (of rows that are not zero), 0 once W has shown an infinity.  (An infinity of x needs no exact
// products: its row's loss is not finite either way.)
__device__ void partial_max(const ScanArgs& a, int block) {
    const bool isw = block >= a.nparts;
    const int rows = isw ? a.V : a.M, nw = a.nparts * 16;
    float top = 0.f, least = INFINITY;
    bool inf = false;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int r = (block - (isw ? a.nparts : 0)) * 16 + wave; r < rows; r += 4 * nw) {
        const float* row[4];
        bool use[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int q = min(r + k * nw, rows - 1);             // the last row again past the end
            use[k] = isw || a.targets[q] != a.ignore;
            row[k] = isw ? a.W + (int64_t)q * a.ldw : a.x + (int64_t)q * a.ldx;
        }
        float m[4] = {0.f, 0.f, 0.f, 0.f};
        auto see = [&](int k, float v) {
            v = fabsf(v);
            if (v < INFINITY) m[k] = fmaxf(m[k], v);
            inf |= v == INFINITY;
        };
        if (a.vec) {
            for (int c = lane * 4; c < a.K; c += 256) {
                f32x4 v[4] = {};
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (use[k]) v[k] = *reinterpret_cast<const f32x4*>(row[k] + c);
#pragma unroll
                for (int k = 0; k < 4; ++k)
#pragma unroll
                    for (int e = 0; e < 4; ++e) see(k, v[k][e]);
            }
        } else {
            for (int c = lane; c < a.K; c += 64) {
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (use[k]) see(k, row[k][c]);
            }
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            m[k] = wave_max(m[k]);
            top = fmaxf(top, m[k]);
            if (m[k] > 0.f) least = fminf(least, m[k]);
        }
    }
    if (isw && __any(inf)) least = 0.f;
    __shared__ float2 wm[16];
    if (lane == 0) wm[wave] = make_float2(top, least);
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < 16; ++w) {
            top = fmaxf(top, wm[w].x);
            least = fminf(least, wm[w].y);
        }
        a.part[(isw ? AMAX_BLOCKS - a.nparts : 0) + block] = make_float2(top, least);
    }
}

__global__ __launch_bounds__(1024) void scan_kernel(ScanArgs a) {
    if (blockIdx.x == 0) compact(a);
    else partial_max(a, blockIdx.x - 1);
}

// Packed operands: rows of whole k-tiles, zero beyond the width; x by slot (zero rows up to the next multiple of 32
// behind the last), W by word, and the bias times log2(e) with -inf behind the vocabulary.  A thread makes 8 columns.
struct PackArgs {
    const void* x; int64_t ldx;
    const void* W; int64_t ldw;
    const void* bias;
    int M, V, K, Kp, xs, dtype, split, Vp, pack_w, vec;
    Head* head;
    const int* order;
    short* px; short* pw; float* b2;
    int64_t nx, nw;           // 8-column chunks of x and W
    const float2* part;       // split operands: the partial maxima
    int nparts;
};
__global__ __launch_bounds__(256) void pack_kernel(PackArgs a) {
    const int64_t total = a.nx + a.nw + a.Vp;
    const int cpr = a.Kp / 8;
    const int count = a.head->count;
    int scale[2] = {0, 0};
    bool far = false;
    if (a.split) {                                  // every block joins the partial maxima for itself; the first notes them
        __shared__ float wm[4][4];
        float m[4] = {0.f, 0.f, INFINITY, INFINITY};
        for (int k = threadIdx.x; k < a.nparts; k += 256) {
#pragma unroll
            for (int o = 0; o < 2; ++o) {
                const float2 v = a.part[o * AMAX_BLOCKS + k];
                m[o] = fmaxf(m[o], v.x);
                m[2 + o] = fminf(m[2 + o], v.y);
            }
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            m[k] = k < 2 ? wave_max(m[k]) : -wave_max(-m[k]);
            if ((threadIdx.x & 63) == 0) wm[k][threadIdx.x >> 6] = m[k];
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 4; ++k)
            m[k] = k < 2 ? fmaxf(fmaxf(wm[k][0], wm[k][1]), fmaxf(wm[k][2], wm[k][3]))
                         : fminf(fminf(wm[k][0], wm[k][1]), fminf(wm[k][2], wm[k][3]));
        far = m[2] * FAR < m[0] || m[3] * FAR < m[1];
        if (!far) scale[0] = scale_exp(m[0]), scale[1] = scale_exp(m[1]);
        if (blockIdx.x == 0 && threadIdx.x == 0) {
            a.head->ex = scale[0];
            a.head->ew = scale[1];
            a.head->far = far;
        }
    }
    for (int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x; t < total; t += (int64_t)gridDim.x * 256) {
        if (t >= a.nx + a.nw) {
            const int v = (int)(t - a.nx - a.nw);
            a.b2[v] = v >= a.V ? -INFINITY : a.bias ? load_as_f32(a.bias, v, a.dtype) * L2E : 0.f;
            continue;
        }
        const bool isw = t >= a.nx;
        if (isw && far) continue;
        const int64_t u = isw ? t - a.nx : t;
        const int row = (int)(u / cpr), c = (int)(u - (int64_t)row * cpr) * 8;
        if (!isw && row >= ((count + 31) & ~31)) continue;
        const bool zero = !isw && row >= count;
        const int64_t base = isw ? (int64_t)row * a.ldw : zero ? 0 : (int64_t)a.order[row] * a.ldx;
        const void* src = isw ? a.W : a.x;
        short* dst = (isw ? a.pw : a.px) + (int64_t)row * a.xs;
        if (!a.split) {
            s16x8 o;
            if (!zero && a.vec && c + 8 <= a.K) {
                o = *reinterpret_cast<const s16x8*>((const short*)src + base + c);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) o[e] = (!zero && c + e < a.K) ? ((const short*)src)[base + c + e] : (short)0;
            }
            *reinterpret_cast<s16x8*>(dst + c) = o;
        } else {
            float v[8];
            if (!zero && a.vec && c + 8 <= a.K) {
                const f32x4* q = reinterpret_cast<const f32x4*>((const float*)src + base + c);
                const f32x4 p0 = q[0], p1 = q[1];
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = p0[e], v[4 + e] = p1[e];
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = (!zero && c + e < a.K) ? ((const float*)src)[base + c + e] : 0.f;
            }
            if (far) {
                f32x4* d = reinterpret_cast<f32x4*>(reinterpret_cast<float*>(dst) + c);
                d[0] = f32x4{v[0], v[1], v[2], v[3]};
                d[1] = f32x4{v[4], v[5], v[6], v[7]};
                continue;
            }
            const int s = scale[isw];
            s16x8 hi, lo;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                short h, l;
                split16(ldexpf(v[e], s), h, l);
                hi[e] = h;
                lo[e] = l;
            }
            short* d = dst + split_col(c);
            *reinterpret_cast<s16x8*>(d) = hi;
            *reinterpret_cast<s16x8*>(d + 16) = lo;
        }
    }
}

// Where no backward call follows, the scales of fp32 rows need not be one for all of a matrix: a wavefront takes a row's
// maximum and packs it at once, and W is read from memory once instead of twice (100 x 50000 x 1024 loss 216 -> 193 us).
struct RowScales {
    float *x, *w;             // what each slot's and each word's products are to be multiplied by
};
template <bool VEC>
__global__ __launch_bounds__(256) void pack_rows_kernel(PackArgs a, RowScales f) {
    const int lane = threadIdx.x & 63, count = a.head->count;
    const int64_t wave = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6), waves = (int64_t)gridDim.x * 4;
    for (int64_t t = wave; t < (int64_t)a.M + a.V; t += waves) {
        const bool isw = t >= a.M;
        const int row = (int)(isw ? t - a.M : t);
        if (!isw && row >= count) continue;
        const float* src = isw ? (const float*)a.W + (int64_t)row * a.ldw : (const float*)a.x + (int64_t)a.order[row] * a.ldx;
        short* dst = (isw ? a.pw : a.px) + (int64_t)row * a.xs;
        float m = 0.f;
        bool inf = false;
        auto see = [&](float v) {
            v = fabsf(v);
            if (v < INFINITY) m = fmaxf(m, v);
            inf |= v == INFINITY;
        };
        if (VEC) {
#pragma unroll 2
            for (int c = lane * 4; c < a.K; c += 256) {
                const f32x4 v = *reinterpret_cast<const f32x4*>(src + c);
#pragma unroll
                for (int e = 0; e < 4; ++e) see(v[e]);
            }
        } else {
#pragma unroll 4
            for (int c = lane; c < a.K; c += 64) see(src[c]);
        }
        m = wave_max(m);
        const int s = scale_exp(m);
        if (lane == 0) (isw ? f.w : f.x)[row] = pow2(-s);
        if (isw && inf) a.head->far = 1;                               // (whoever says so says the same)
        for (int c = lane * 4; c < a.Kp; c += 256) {                   // four columns: halves of a group's hi and lo
            f32x4 v = {0.f, 0.f, 0.f, 0.f};
            if (VEC) {
                if (c < a.K) v = *reinterpret_cast<const f32x4*>(src + c);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (c + e < a.K) v[e] = src[c + e];
            }
            s16x4 hi, lo;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                short h, l;
                split16(ldexpf(v[e], s), h, l);
                hi[e] = h;
                lo[e] = l;
            }
            short* d = dst + split_col(c);
            *reinterpret_cast<s16x4*>(d) = hi;
            *reinterpret_cast<s16x4*>(d + 16) = lo;
        }
    }
    for (int64_t v = (int64_t)blockIdx.x * 256 + threadIdx.x; v < a.Vp; v += (int64_t)gridDim.x * 256) {
        a.b2[v] = v >= a.V ? -INFINITY : a.bias ? load_as_f32(a.bias, v, a.dtype) * L2E : 0.f;
        if (v >= a.V) f.w[v] = 1.f;
    }
}

// ---- (max, sum of exp) of every row over each tile of 256 words; values in units of log 2 ---------------------------
struct LogitArgs {
    View W, X;
    View32 W32, X32;                             // split operands: the fp32 ones
    int K;
    const float* b2;
    const Head* head;
    int kt, Mp;
    Map map;
    float2* part;                                // forward: [tile][slot]
    float* zt;                                   // forward: [slot] the target's logit, from the tile that has its word
    RowScales f;                                 // forward, by row
    // dlogits
    const float *lse, *dlt, *rw;
    const int* tgt;
    short* g; int64_t ldg;                       // [slot][word of the piece]
    float* dbp;                                  // [row tile][word of the piece], nullable
    float* rest;                                 // [slot] what rounding took off the target's entry (16-bit operands)
    int v0, piece;
    int gexp;
};

template <bool SPLIT>
__device__ __forceinline__ float logit_scale(const Head* head) {
    return SPLIT ? ldexpf(L2E, -(head->ex + head->ew)) : L2E;
}

// the logits of a tile times logit_scale() (or the rows' scales)
template <class C, int ELT, bool SPLIT>
__device__ __forceinline__ void logits(const LogitArgs& a, bool far, int i0, int j0, short* lds, f32x16 (&acc)[C::TI][C::TJ]) {
    if (SPLIT && far) {
        const View32 x{a.X32.p, a.X32.ld, a.X32.order, a.head->count};
        contract32<C, false, false>(a.W32, x, i0, j0, 0, a.K, a.K, lds, acc);
    } else contract<C, ELT, false, false, SPLIT>(a.W, a.X, i0, j0, 0, a.kt, lds, acc);
}

template <class C, int ELT, bool SPLIT, bool BY_ROW>
__global__ __launch_bounds__(C::THREADS, C::EU) void lse_kernel(LogitArgs a) {
    extern __shared__ __attribute__((aligned(16))) short lds[];
    int ti_, tj_, z;
    if (!tile_of(a.map, blockIdx.x, ti_, tj_, z)) return;
    const int count = a.head->count;
    const int i0 = ti_ * C::BI, j0 = tj_ * C::BJ;
    if (j0 >= count) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wi = wave / C::WJ, wj = wave % C::WJ, h = lane >> 5;
    int at[C::TJ];                                // the targets among the wavefront's words
#pragma unroll
    for (int tj = 0; tj < C::TJ; ++tj) {
        const int slot = j0 + (wj * C::TJ + tj) * 32 + (lane & 31);
        at[tj] = slot < count ? a.tgt[slot] - i0 - wi * C::TI * 32 : -1;
    }
    f32x16 acc[C::TI][C::TJ];
    const bool far = SPLIT && a.head->far;
    logits<C, ELT, SPLIT>(a, far, i0, j0, lds, acc);
    const float c0 = logit_scale<SPLIT>(a.head);
    float2* red = reinterpret_cast<float2*>(lds);
#pragma unroll
    for (int tj = 0; tj < C::TJ; ++tj) {
        float m = -INFINITY;
        float c1 = c0;
        if (BY_ROW) c1 = far ? 1.f : a.f.x[j0 + (wj * C::TJ + tj) * 32 + (lane & 31)];
#pragma unroll
        for (int ti = 0; ti < C::TI; ++ti)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int word = i0 + (wi * C::TI + ti) * 32 + 8 * q + 4 * h;
                const f32x4 b = *reinterpret_cast<const f32x4*>(a.b2 + word);
                f32x4 c = {c1, c1, c1, c1};
                if (BY_ROW) {          // (the two powers first: one alone may be denormal, which would round its product with L2E)
                    const f32x4 f = *reinterpret_cast<const f32x4*>(a.f.w + word);
#pragma unroll
                    for (int e = 0; e < 4; ++e) c[e] = c[e] * (far ? 1.f : f[e]) * L2E;
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float v = fmaf(acc[ti][tj][4 * q + e], c[e], b[e]);
                    acc[ti][tj][4 * q + e] = v;
                    m = fmaxf(m, v);
                }
            }
        const int to = at[tj];
        if (__any(to >= 0 && to < C::TI * 32)) {
            float zt = 0.f;
#pragma unroll
            for (int ti = 0; ti < C::TI; ++ti)
#pragma unroll
                for (int e = 0; e < 16; ++e) zt = to - 4 * h == ti * 32 + acc_row(e, 0) ? acc[ti][tj][e] : zt;
            if (to >= 0 && to < C::TI * 32 && ((to >> 2) & 1) == h) a.zt[j0 + (wj * C::TJ + tj) * 32 + (lane & 31)] = zt;
        }
        const float m0 = m == -INFINITY ? 0.f : m;          // a tile whose words are all masked by the bias
        float s = 0.f;
#pragma unroll
        for (int ti = 0; ti < C::TI; ++ti)
#pragma unroll
            for (int e = 0; e < 16; ++e) s += __builtin_amdgcn_exp2f(acc[ti][tj][e] - m0);
        // the other half of the words, then the other pair of wavefronts
        const float mo = __shfl_xor(m, 32, 64), so = __shfl_xor(s, 32, 64);
        const float mm = fmaxf(m, mo), mz = mm == -INFINITY ? 0.f : mm;
        s = s * __builtin_amdgcn_exp2f(m - mz) + so * __builtin_amdgcn_exp2f(mo - mz);
        if (h == 0) red[wi * C::BJ + (wj * C::TJ + tj) * 32 + lane] = make_float2(mm, s);
    }
    __syncthreads();
    for (int j = threadIdx.x; j < C::BJ; j += C::THREADS) {
        const float2 u = red[j], v = red[C::BJ + j];
        const float mm = fmaxf(u.x, v.x), mz = mm == -INFINITY ? 0.f : mm;
        a.part[(int64_t)ti_ * a.Mp + j0 + j] =
            make_float2(mm, u.y * __builtin_amdgcn_exp2f(u.x - mz) + v.y * __builtin_amdgcn_exp2f(v.x - mz));
    }
}

// Per slot: the tiles' statistics joined, and the loss.  The target's logit is the very number that went into the sum, so
// that a row which is sure of its target loses 0 and not the rounding of two sums (the logit as a dot product of its own:
// +-4e-6 at a logit of 64).  dlt: the target's logit in, the log of its probability out.  Rows that are not counted get
// loss 0.  A workgroup has 64 slots, whose statistics lie side by side, or (ROW) one, whose tiles do.
template <bool ROW>
__global__ __launch_bounds__(1024) void nll_kernel(const float2* __restrict__ part, int ntiles, int Mp, int M,
                                                   const Head* __restrict__ head, const int* __restrict__ order,
                                                   const int* __restrict__ slot, const int* __restrict__ tgt,
                                                   float* __restrict__ lse, float* __restrict__ dlt, float* __restrict__ nll) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int s = ROW ? blockIdx.x : blockIdx.x * 64 + lane, count = head->count;
    if (s < M && threadIdx.x < 64 && slot[s] < 0 && (!ROW || lane == 0)) nll[s] = 0.f;         // as a row
    float m = -INFINITY, sum = 0.f;
    auto join = [&](float mo, float so) {
        const float mm = fmaxf(m, mo), mz = mm == -INFINITY ? 0.f : mm;
        sum = sum * __builtin_amdgcn_exp2f(m - mz) + so * __builtin_amdgcn_exp2f(mo - mz);
        m = mm;
    };
    if (s < count) {
#pragma unroll 4
        for (int t = ROW ? threadIdx.x : wave; t < ntiles; t += ROW ? 1024 : 16) {
            const float2 v = ROW ? part[(int64_t)s * ntiles + t] : part[(int64_t)t * Mp + s];
            join(v.x, v.y);
        }
    }
    if (ROW) {
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) {
            const float mo = __shfl_xor(m, o, 64), so = __shfl_xor(sum, o, 64);
            join(mo, so);
        }
    }
    __shared__ float2 st[16][64];
    st[wave][lane] = make_float2(m, sum);
    __syncthreads();
    if (wave > 0 || s >= count || (ROW && lane > 0)) return;
    for (int w = 1; w < 16; ++w) join(st[w][lane].x, st[w][lane].y);
    const bool known = tgt[s] >= 0;
    const float l = __log2f(sum), d = known ? ((dlt[s] - m) - l) * LN2 : NAN;       // log of the target's probability
    lse[s] = known ? m + l : NAN;
    dlt[s] = d;
    nll[order[s]] = -d;
}

// loss[0] = mean over the counted rows, loss[1] = sum, loss[2] = number of counted rows; one workgroup, fixed order
__global__ __launch_bounds__(1024) void loss_kernel(const float* __restrict__ nll, int M, const Head* __restrict__ head,
                                                    float* __restrict__ loss) {
    double s = 0.0;
    for (int r = threadIdx.x; r < M; r += 1024) s += (double)nll[r];
    __shared__ double part[16];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        s = 0.0;
        for (int w = 0; w < 16; ++w) s += part[w];
        loss[0] = (float)(s / (double)head->count);    // no counted row: 0 / 0, as torch has it
        loss[1] = (float)s;
        loss[2] = (float)head->count;
    }
}

// ---- backward -----------------------------------------------------------------------------------------------------
// The rows' own upstream gradients, brought to [2^(gexp - 1), 2^gexp] at most by a power of two, and the factor that undoes
// it.  (One scalar for all rows needs no kernel: G is stored times 2^gexp, and factor_of() has the rest.)
__global__ __launch_bounds__(1024) void weights_kernel(const float* __restrict__ row_grad, const Head* __restrict__ head,
                                                       const int* __restrict__ order, int Mp, int gexp,
                                                       float* __restrict__ rw, BwdHead* __restrict__ bh) {
    const int count = head->count;
    __shared__ float wm[16];
    float m = 0.f;
    for (int s = threadIdx.x; s < count; s += 1024) {
        const float v = fabsf(row_grad[order[s]]);
        if (v < INFINITY) m = fmaxf(m, v);
    }
    m = wave_max(m);
    if ((threadIdx.x & 63) == 0) wm[threadIdx.x >> 6] = m;
    __syncthreads();
    m = 0.f;
    for (int w = 0; w < 16; ++w) m = fmaxf(m, wm[w]);
    // m * scale in [2^(gexp - 1), 2^gexp)
    if (head->far) gexp = 0;
    const int e = (int)(__float_as_uint(m) >> 23) - 127;
    const float scale = m > 0.f ? pow2(min(gexp - 1 - e, 126)) : 1.f;
    for (int s = threadIdx.x; s < Mp; s += 1024) rw[s] = s < count ? row_grad[order[s]] * scale : 0.f;
    if (threadIdx.x == 0) bh->factor = count > 0 ? 1.f / scale : 0.f;
}

// G of one piece of the vocabulary.  The tile is turned through LDS (a wavefront's 64 rows x 128 words at a time), so
// that rows are stored 256 contiguous bytes at a time; on the way the targets' entries are put in, (p_t - 1) g as
// expm1(log p_t) g, and each word's column is summed for the bias gradient.
template <class C, int ELT, bool SPLIT>
__global__ __launch_bounds__(C::THREADS, C::EU) void dlogits_kernel(LogitArgs a) {
    extern __shared__ __attribute__((aligned(16))) short lds[];
    int ti_, tj_, z;
    if (!tile_of(a.map, blockIdx.x, ti_, tj_, z)) return;
    const int count = a.head->count;
    const int i0 = a.v0 + ti_ * C::BI, j0 = tj_ * C::BJ;
    if (j0 >= count) return;
    f32x16 acc[C::TI][C::TJ];
    const bool far = SPLIT && a.head->far;
    logits<C, ELT, SPLIT>(a, far, i0, j0, lds, acc);
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));       // the addresses below are made here, not ahead of the contraction (72 spills)
    const int lane = tid & 63, wave = tid >> 6, wi = wave / C::WJ, wj = wave % C::WJ, h = lane >> 5;
    const float c1 = logit_scale<SPLIT>(a.head);
    constexpr int WORDS = 32 * C::TI;                     // of a wavefront
    constexpr int PL = SPLIT ? 2 : 1;
    constexpr int LOW = SPLIT ? 16 : WORDS;               // from a value to its low part
    constexpr int LD = WORDS * 2 + 8;                     // 16-bit elements per row of the turned tile: G, and its low parts
    auto finish = [&](auto as_fp32) {        // G in fp32, or in pairs or 16 bits: two copies of the code, no branches within
        constexpr bool AS32 = decltype(as_fp32)::value;
        // one 32-row block of the wavefront at a time
        short* tile = lds + wave * 32 * LD;
        float* colsum = reinterpret_cast<float*>(lds + C::WAVES * 32 * LD);      // [WJ][BI]
        float sums[2] = {0.f, 0.f};
#pragma unroll
        for (int tj = 0; tj < C::TJ; ++tj) {
            const int s = j0 + (wj * C::TJ + tj) * 32 + (lane & 31);
            const bool live = s < count;
            const float l2 = live ? a.lse[s] : 0.f;
            const float w = live ? (a.rw ? a.rw[s] : pow2(AS32 ? 0 : a.gexp)) : 0.f;
            const float* b2 = a.b2 + i0 + wi * WORDS;
#pragma unroll
            for (int ti = 0; ti < C::TI; ++ti) {
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int wd = ti * 32 + 8 * q + 4 * h;       // word inside the wavefront's range
                    const f32x4 b = *reinterpret_cast<const f32x4*>(b2 + wd);
                    s16x4 hi, lo;
                    f32x4 full;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        float v = __builtin_amdgcn_exp2f(fmaf(acc[ti][tj][4 * q + e], c1, b[e]) - l2) * w;
                        if (!live) v = 0.f;
                        full[e] = v;
                        if (SPLIT) {
                            short p, r;
                            split16(v, p, r);
                            hi[e] = p;
                            lo[e] = r;
                        } else {
                            asm("" : "+v"(v));
                            hi[e] = to_bits<ELT>(v);
                            lo[e] = to_bits<ELT>(v - from_bits<ELT>(hi[e]));
                        }
                    }
                    if (AS32) {
                        *reinterpret_cast<f32x4*>(tile + (lane & 31) * LD + 2 * wd) = full;
                        continue;
                    }
                    short* d = tile + (lane & 31) * LD + (SPLIT ? (int)split_col(wd) : wd);
                    *reinterpret_cast<s16x4*>(d) = hi;
                    if (SPLIT || a.dbp) *reinterpret_cast<s16x4*>(d + LOW) = lo;
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            // (the tile belongs to this wavefront alone: LDS operations of a wavefront complete in order)
            // What rounding takes off a target's entry, usually its row's largest by far, is kept: dx gets it back, and dW of
            // a batch too small for such errors to average out.
            if (h == 0 && live) {
                const int t = a.tgt[s] - (i0 + wi * WORDS);
                if (t >= 0 && t < WORDS) {
                    float v = expm1f(a.dlt[s]) * w;
                    asm("" : "+v"(v));
                    short* d = tile + lane * LD + (SPLIT ? (int)split_col(t) : t);
                    if (AS32) {
                        *reinterpret_cast<float*>(tile + lane * LD + 2 * t) = v;
                    } else if (SPLIT) {
                        short p, r;
                        split16(v, p, r);
                        d[0] = p;
                        d[16] = r;
                    } else {
                        const short q = to_bits<ELT>(v);
                        const float rest = v - from_bits<ELT>(q);
                        d[0] = q;
                        d[LOW] = to_bits<ELT>(rest);
                        a.rest[s] = rest;
                    }
                }
            }
            __builtin_amdgcn_wave_barrier();
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            constexpr int CH = WORDS * PL / 8;                     // 16-byte chunks per row
            constexpr int RPP = 64 / CH;                           // rows per pass
            static_assert(64 % CH == 0, "row does not divide over the wavefront");
            const int row0 = j0 + (wj * C::TJ + tj) * 32;
            short* gp = a.g + (int64_t)(ti_ * C::BI + wi * WORDS) * PL;
#pragma unroll 4
            for (int r = lane / CH; r < 32; r += RPP) {
                const s16x8 v = *reinterpret_cast<const s16x8*>(tile + r * LD + (lane % CH) * 8);
                *reinterpret_cast<s16x8*>(gp + (int64_t)(row0 + r) * a.ldg + (lane % CH) * 8) = v;
            }
            if (a.dbp) {
#pragma unroll
                for (int k = 0; k < WORDS / 64; ++k) {
                    const int wd = lane + 64 * k;
                    const short* d = tile + (SPLIT ? (int)split_col(wd) : wd);
                    float sum = 0.f;
#pragma unroll 8
                    for (int r = 0; r < 32; ++r) {
                        sum += AS32 ? *reinterpret_cast<const float*>(tile + r * LD + 2 * wd)
                                            : from_bits<ELT>(d[r * LD]) + from_bits<ELT>(d[r * LD + LOW]);
                    }
                    sums[k] += sum;
                }
            }
            __builtin_amdgcn_wave_barrier();
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        }
        if (a.dbp) {
#pragma unroll
            for (int k = 0; k < WORDS / 64; ++k) colsum[wj * C::BI + wi * WORDS + lane + 64 * k] = sums[k];
            __syncthreads();
            for (int i = threadIdx.x; i < C::BI; i += C::THREADS) {
                float sum = 0.f;
#pragma unroll
                for (int w = 0; w < C::WJ; ++w) sum += colsum[w * C::BI + i];
                a.dbp[(int64_t)tj_ * a.piece + ti_ * C::BI + i] = sum;
            }
        }
    };
    if (SPLIT && far) finish(std::integral_constant<bool, SPLIT>{});
    else finish(std::false_type{});
}

// dx and dW of one piece.  OUT 0: fp32 partial sums [split][i][j], added onto what earlier pieces left when `add`;
// OUT 1: times the factor, in the weights' type.
constexpr int REST_ROWS = 64;
struct GradArgs {
    View P, Q;
    View32 P32, Q32;               // split operands: the fp32 ones
    int k32;                       // dx: words of the piece that exist
    const Head* head;
    Upstream up;
    int I, J;                      // rows and columns stored
    int rows_live;                 // dx: only the first count rows exist
    int k_live;                    // dW: the contraction runs over the counted rows; else over kt k-tiles
    int kt, nsplit;
    Splits splits;                 // dx: instead of nsplit
    Map map;
    const int* tgt; const float* rest; int v0;     // dW of at most REST_ROWS rows
    float* part; int64_t ldp, plane; int add;      // dx: plane is of the live row tiles
    void* out; int64_t ldo; int dtype;
    int vec;                       // 16-bit results: rows of whole aligned 16-byte pieces
};
__device__ __forceinline__ void store_as(void* p, int64_t i, float v, int dtype) {
    if (dtype == CAPDEC_F32) ((float*)p)[i] = v;
    else ((short*)p)[i] = dtype == CAPDEC_BF16 ? to_bits<BF16>(v) : to_bits<F16>(v);
}

template <class C, int ELT, bool TP, bool SPLIT, int OUT>
__global__ __launch_bounds__(C::THREADS, C::EU) void grad_kernel(GradArgs a) {
    extern __shared__ __attribute__((aligned(16))) short lds[];
    int ti_, tj_, z;
    const int count = a.head->count;
    if (a.rows_live) {
        a.map.ni = (count + C::BI - 1) / C::BI;
        a.map.nz = a.nsplit = splits_of(a.splits, a.map.ni);
        a.map.per = (a.map.ni * a.map.nj * a.map.nz + 7) / 8;
        a.plane = (int64_t)a.map.ni * C::BI * a.ldp;
    }
    if (!tile_of(a.map, blockIdx.x, ti_, tj_, z)) return;
    const int i0 = ti_ * C::BI, j0 = tj_ * C::BJ;
    const int nI = a.rows_live ? min(a.I, count) : a.I;
    constexpr int KT = SPLIT ? 16 : 32;
    const int kt = a.k_live ? (count + KT - 1) / KT : a.kt;
    const int per = (kt + a.nsplit - 1) / a.nsplit;
    f32x16 acc[C::TI][C::TJ];
    const int kt1 = min(kt, (z + 1) * per);
    if (SPLIT && a.head->far) contract32<C, TP, true>(a.P32, a.Q32, i0, j0, z * per * KT, kt1 * KT, a.k_live ? count : a.k32, lds, acc);
    else contract<C, ELT, TP, true, SPLIT>(a.P, a.Q, i0, j0, z * per, kt1, lds, acc);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wi = wave / C::WJ, wj = wave % C::WJ, h = lane >> 5;
    if (TP && !SPLIT && z == 0 && count <= REST_ROWS) {
        // row m adds rest[m] x[m] to its target's row of dW
        for (int m = 0; m < count; ++m) {
            const int at = a.tgt[m] - a.v0 - i0;
            if (a.tgt[m] < a.v0 || at < 0 || at >= C::BI) continue;
            const float q = a.rest[m];
#pragma unroll
            for (int tj = 0; tj < C::TJ; ++tj) {
                const int j = min(j0 + (wj * C::TJ + tj) * 32 + (lane & 31), a.Q.n - 1);
                const float x = q * from_bits<ELT>(a.Q.p[(int64_t)m * a.Q.ld + j]);
#pragma unroll
                for (int ti = 0; ti < C::TI; ++ti)
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        if ((wi * C::TI + ti) * 32 + acc_row(e, h) == at) acc[ti][tj][e] += x;
            }
        }
    }
    const float f = OUT == 1 ? factor_of(a.up, a.head) : 1.f;
    const int ex = OUT == 1 && SPLIT ? -a.head->ex : 0;
    if (OUT == 1 && !SPLIT && a.vec) {
        // 16-bit results go through LDS, 32 rows of the wavefront at a time: stores of 16 bytes a lane instead of 2
        constexpr int COLS = 32 * C::TJ, LD = COLS + 8, CH = COLS / 8;
        short* tile = lds + wave * 32 * LD;
#pragma unroll
        for (int ti = 0; ti < C::TI; ++ti) {
#pragma unroll
            for (int tj = 0; tj < C::TJ; ++tj)
#pragma unroll
                for (int e = 0; e < 16; ++e) tile[acc_row(e, h) * LD + tj * 32 + (lane & 31)] = to_bits<ELT>(acc[ti][tj][e] * f);
            __builtin_amdgcn_wave_barrier();
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            const int j = j0 + wj * COLS + (lane % CH) * 8;
#pragma unroll
            for (int r = 0; r < 32; r += 64 / CH) {
                const int i = i0 + (wi * C::TI + ti) * 32 + r + lane / CH;
                const s16x8 v = *reinterpret_cast<const s16x8*>(tile + (r + lane / CH) * LD + (lane % CH) * 8);
                if (i < nI && j < a.J) *reinterpret_cast<s16x8*>((short*)a.out + (int64_t)i * a.ldo + j) = v;
            }
            __builtin_amdgcn_wave_barrier();
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        }
        return;
    }
#pragma unroll
    for (int tj = 0; tj < C::TJ; ++tj) {
        const int j = j0 + (wj * C::TJ + tj) * 32 + (lane & 31);
        if (j >= a.J) continue;
#pragma unroll
        for (int ti = 0; ti < C::TI; ++ti) {
            const int ib = i0 + (wi * C::TI + ti) * 32;
            float* d = a.part + (int64_t)z * a.plane + j;
            if (OUT == 0 && a.add) {
                float old[16];
#pragma unroll
                for (int e = 0; e < 16; ++e) old[e] = d[(int64_t)min(ib + acc_row(e, h), nI - 1) * a.ldp];
#pragma unroll
                for (int e = 0; e < 16; ++e) acc[ti][tj][e] += old[e];
            }
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int i = ib + acc_row(e, h);
                if (i >= nI) continue;
                if (OUT == 0) d[(int64_t)i * a.ldp] = acc[ti][tj][e];
                else store_as(a.out, (int64_t)i * a.ldo + j, SPLIT ? ldexpf(acc[ti][tj][e] * f, ex) : acc[ti][tj][e] * f, a.dtype);
            }
        }
    }
}

// dx[r] = factor * (sum of the partial sums of r's slot + what rounding took off its target's entry of G times the target's
// row of W); zero for rows that are not counted
__global__ __launch_bounds__(256) void dx_kernel(const float* __restrict__ part, Splits splits, int rows, int Kp, int M, int K,
                                                 const int* __restrict__ slot, const int* __restrict__ tgt,
                                                 const float* __restrict__ rest, const void* W, int64_t ldw,
                                                 const Head* __restrict__ head, Upstream up, int split, void* out,
                                                 int64_t ldo, int dtype) {
    const float f = factor_of(up, head);
    const int ew = split ? -head->ew : 0;
    const int tiles = (head->count + 255) / 256, nsplit = splits_of(splits, tiles);
    const int64_t plane = (int64_t)(rows ? rows : tiles * 256) * Kp;
    const int cpr = (K + 3) / 4;
    for (int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x; t < (int64_t)M * cpr; t += (int64_t)gridDim.x * 256) {
        const int r = (int)(t / cpr), c = (int)(t - (int64_t)r * cpr) * 4;
        const int s = slot[r];
        f32x4 v = {0.f, 0.f, 0.f, 0.f};
        if (s >= 0) {
#pragma unroll 16
            for (int k = 0; k < nsplit; ++k) v += *reinterpret_cast<const f32x4*>(part + k * plane + (int64_t)s * Kp + c);
            const int w = tgt[s];
            if (rest && w >= 0) {
                const float q = rest[s];
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (c + e < K) v[e] = fmaf(q, load_as_f32(W, (int64_t)w * ldw + c + e, dtype), v[e]);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = ldexpf(v[e] * f, ew);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (c + e < K) store_as(out, (int64_t)r * ldo + c + e, v[e], dtype);
    }
}

// dW of one piece from its partial sums, and db from the row tiles' column sums
__global__ __launch_bounds__(256) void dw_kernel(const float* __restrict__ part, int64_t plane, int nsplit, int Kp, int rows,
                                                 int K, const Head* __restrict__ head, Upstream up, int split, void* dW,
                                                 int64_t ldw, int dtype, const float* __restrict__ dbp, int piece, int row_tile, void* db, int v0) {
    const float f = factor_of(up, head);
    const int ex = split ? -head->ex : 0;
    const int cpr = (K + 3) / 4;
    const int64_t nw = nsplit > 1 ? (int64_t)rows * cpr : 0;
    for (int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x; t < nw + (dbp ? rows : 0); t += (int64_t)gridDim.x * 256) {
        if (t >= nw) {
            const int v = (int)(t - nw), tiles = (head->count + row_tile - 1) / row_tile;
            float s = 0.f;
            for (int k = 0; k < tiles; ++k) s += dbp[(int64_t)k * piece + v];
            store_as(db, v0 + v, s * f, dtype);
            continue;
        }
        const int r = (int)(t / cpr), c = (int)(t - (int64_t)r * cpr) * 4;
        f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
        for (int k = 0; k < nsplit; ++k) v += *reinterpret_cast<const f32x4*>(part + k * plane + (int64_t)r * Kp + c);
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (c + e < K) store_as(dW, (int64_t)(v0 + r) * ldw + c + e, ldexpf(v[e] * f, ex), dtype);
    }
}

// ---- fp32 batches of at most 64 rows ------------------------------------------------------------------------------------
// There reading W and writing dW is nearly all of the work, and packing W would read it twice and write it once more.  So
// W goes from memory into fp32 matrix instructions (16 x 16 x 4), which keep up with memory for so few rows, and the logits,
// of which there are fewer than W has elements, are kept for the backward call instead of a packed W.  Slots in groups of
// 16, R groups; lane (r, g) = (lane & 15, lane >> 4) holds row or column r and, of 16 terms of a sum, terms 4 g to 4 g + 3:
// operands agree on the order of the terms, so that it may be any.
// W of 131072 x 512 (54 us a pass at the rate of a large copy): one row takes 56 us for the loss and 225 for loss and
// gradients (few_lse 86, 55 where W stays in the caches; few_dx 55, few_dw 51); 64 rows 143 and 460, where the split operands
// take 225 and 600 for 65 rows.  From 32 rows on the matrix instructions count (64 rows: 55 us of each product) and the
// kernels are bound by the two together.
__device__ __forceinline__ f32x4 mfma4(float a, float b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }

template <bool VEC>
__device__ __forceinline__ f32x4 load4(const float* p) {
    if (VEC) return *reinterpret_cast<const f32x4*>(p);
    return f32x4{p[0], p[1], p[2], p[3]};
}
// the first n of 4 values, zeros behind them
__device__ __forceinline__ f32x4 load_some(const float* p, int n) {
    f32x4 v;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = e < n ? p[e] : 0.f;
    return v;
}

struct FewArgs {
    const float* x; int64_t ldx;
    const float* W; int64_t ldw;
    const float* bias;
    int M, V, K, Vp;
    const Head* head;
    const int* order;
    int Kp;
    float* xs;                 // [slot][Kp], a copy of x for the backward call, zero behind the width and the counted rows
    float* z;                  // [slot][Vp], in units of log 2, -inf behind the vocabulary
    float2* part;              // [slot][Vp / 32]
    const int* tgt;
    float* zt;                 // [slot] the target's logit
};
// A wavefront makes the logits of 32 words, the four of a workgroup reading the same columns of x at about the same time; or,
// where that would leave CUs idle, a workgroup has 32 words and its wavefronts share out the sum over the width (SHARE; taken
// throughout, 64 x 50000 x 1024 is 125 instead of 110 us, 64 x 131072 x 512 154 instead of 149, one row the same).
template <int R, bool SHARE, bool VEC>
__global__ __launch_bounds__(256) void few_lse_kernel(FewArgs a) {
    const int count = a.head->count;
    for (int k = blockIdx.x; k < 16 * R; k += gridDim.x)
        for (int c = threadIdx.x; c < a.Kp; c += 256)
            a.xs[(int64_t)k * a.Kp + c] = k < count && c < a.K ? a.x[(int64_t)a.order[k] * a.ldx + c] : 0.f;
    if (count == 0) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
    const int tile = SHARE ? blockIdx.x : blockIdx.x * 4 + wave, w0 = tile * 32;
    const int q0 = SHARE ? wave : 0;
    constexpr int QS = SHARE ? 4 : 1;
    const float *wp[2], *xp[R];
#pragma unroll
    for (int t = 0; t < 2; ++t) wp[t] = a.W + (int64_t)min(w0 + 16 * t + r, a.V - 1) * a.ldw + 4 * g;
#pragma unroll
    for (int i = 0; i < R; ++i) xp[i] = a.x + (int64_t)a.order[min(16 * i + r, count - 1)] * a.ldx + 4 * g;
    f32x4 acc[2][R] = {};
    auto multiply = [&](const auto& wv, const auto& xv, int u) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int i = 0; i < R; ++i) acc[t][i] = mfma4(wv[t][u][e], xv[i][u][e], acc[t][i]);
    };
    constexpr int U = R == 4 ? 2 : 4, COLS = 16 * U;
    const int full = a.K / COLS;
    for (int q = q0; q < full; q += QS) {
        f32x4 wv[2][U], xv[R][U];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int u = 0; u < U; ++u) wv[t][u] = load4<VEC>(wp[t] + q * COLS + 16 * u);
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
            for (int u = 0; u < U; ++u) xv[i][u] = load4<VEC>(xp[i] + q * COLS + 16 * u);
#pragma unroll
        for (int u = 0; u < U; ++u) multiply(wv, xv, u);
    }
    if (full * COLS < a.K && (!SHARE || wave == (full & 3))) {
        f32x4 wv[2][U], xv[R][U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int c = full * COLS + 16 * u, n = a.K - c - 4 * g;
#pragma unroll
            for (int t = 0; t < 2; ++t) wv[t][u] = load_some(wp[t] + c, n);
#pragma unroll
            for (int i = 0; i < R; ++i) xv[i][u] = load_some(xp[i] + c, n);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) multiply(wv, xv, u);
    }
    // lane (r, g) has words 4 g to 4 g + 3 of both groups for slot r of row group i
    auto finish = [&](int i, const f32x4 (&d)[2]) {
        const int slot = 16 * i + r, t0 = slot < count ? a.tgt[slot] : -1;
        float v[2][4], m = -INFINITY;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int w = w0 + 16 * t + 4 * g + e;
                const float b = a.bias ? a.bias[min(w, a.V - 1)] : 0.f;
                v[t][e] = w < a.V ? fmaf(d[t][e], L2E, b * L2E) : -INFINITY;
                if (w == t0) a.zt[slot] = v[t][e];
                m = fmaxf(m, v[t][e]);
            }
            *reinterpret_cast<f32x4*>(a.z + (int64_t)slot * a.Vp + w0 + 16 * t + 4 * g) = f32x4{v[t][0], v[t][1], v[t][2], v[t][3]};
        }
        m = fmaxf(m, __shfl_xor(m, 16, 64));
        m = fmaxf(m, __shfl_xor(m, 32, 64));
        const float m0 = m == -INFINITY ? 0.f : m;
        float s = 0.f;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) s += __builtin_amdgcn_exp2f(v[t][e] - m0);
        s += __shfl_xor(s, 16, 64);
        s += __shfl_xor(s, 32, 64);
        if (g == 0) a.part[(int64_t)slot * (a.Vp / 32) + tile] = make_float2(m, s);
    };
    if (!SHARE) {
#pragma unroll
        for (int i = 0; i < R; ++i) finish(i, {acc[0][i], acc[1][i]});
        return;
    }
    __shared__ f32x4 sum[SHARE ? 4 : 1][2][R][64];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < R; ++i) sum[wave][t][i][lane] = acc[t][i];
    __syncthreads();
    if (wave >= R) return;
    f32x4 d[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        d[t] = sum[0][t][wave][lane];
#pragma unroll
        for (int k = 1; k < 4; ++k) d[t] += sum[k][t][wave][lane];
    }
    finish(wave, d);
}

template <int R>
void launch_few_lse(const FewArgs& a, bool vec, hipStream_t s) {
    const bool share = a.Vp / 32 < FEW_WAVES;
    const unsigned grid = share ? a.Vp / 32 : a.Vp / 128;
    if (share) vec ? few_lse_kernel<R, true, true><<<grid, 256, 0, s>>>(a) : few_lse_kernel<R, true, false><<<grid, 256, 0, s>>>(a);
    else vec ? few_lse_kernel<R, false, true><<<grid, 256, 0, s>>>(a) : few_lse_kernel<R, false, false><<<grid, 256, 0, s>>>(a);
}

struct FewGrad {
    const float* xs;           // [slot][Kp]
    const float* W; int64_t ldw;
    int M, V, K, Kp, Vp;
    const Head* head;
    const int* tgt;
    const float *z, *lse, *dlt, *rw;
    Upstream up;
    float* G;                  // [slot][Vp], zero behind the counted rows and behind the vocabulary
    int rows;                  // slots of z and G
    int words;                 // of a part of the dx contraction, a multiple of 128
    float* part;               // [part][slot][Kp]
    float* dW; int64_t lddw;
    float* db;
};
// G from the logits, and the bias gradient.  A thread has four words, a wavefront every fourth slot.
__global__ __launch_bounds__(256) void few_g_kernel(FewGrad a) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int w = (blockIdx.x * 64 + lane) * 4;               // Vp is a multiple of 256
    const int count = a.head->count;
    f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int s = wave; s < a.rows; s += 4) {
        f32x4 v = {0.f, 0.f, 0.f, 0.f};
        if (s < count) {
            const float l2 = a.lse[s], f = a.rw ? a.rw[s] : 1.f;
            const int t = a.tgt[s] - w;
            const f32x4 z = *reinterpret_cast<const f32x4*>(a.z + (int64_t)s * a.Vp + w);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = (t == e && a.tgt[s] >= 0 ? expm1f(a.dlt[s]) : __builtin_amdgcn_exp2f(z[e] - l2)) * f;
            sum += v;
        }
        *reinterpret_cast<f32x4*>(a.G + (int64_t)s * a.Vp + w) = v;
    }
    if (!a.db) return;
    __shared__ f32x4 part[4][64];
    part[wave][lane] = sum;
    __syncthreads();
    const float f = factor_of(a.up, a.head);
    const float* p = reinterpret_cast<const float*>(part);
    const int v = blockIdx.x * 256 + threadIdx.x;
    if (v < a.V) a.db[v] = ((p[threadIdx.x] + p[256 + threadIdx.x]) + (p[512 + threadIdx.x] + p[768 + threadIdx.x])) * f;
}

// Partial sums of dx = G W: a workgroup has 64 columns and one part of the words, of which its wavefronts take 16 at a time
// in turn.  A lane reads 4 columns of a word at once, which go to four products: column 4 r + c is column r of product c.
template <int R, bool VEC>
__global__ __launch_bounds__(256) void few_dx_kernel(FewGrad a) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
    const int c0 = blockIdx.x * 64 + 4 * r, first = blockIdx.y * a.words, last = min(a.Vp, first + a.words);
    f32x4 acc[R][4] = {};
    f32x4 b[2][4], v[2][R];                                   // the next words are on their way during a product
    auto load = [&](int k, int w) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float* row = a.W + (int64_t)min(w + 4 * g + e, a.V - 1) * a.ldw;      // G is zero behind the vocabulary
            if (VEC) b[k][e] = *reinterpret_cast<const f32x4*>(row + min(c0, a.K - 4));
            else
#pragma unroll
                for (int c = 0; c < 4; ++c) b[k][e][c] = row[min(c0 + c, a.K - 1)];
        }
#pragma unroll
        for (int i = 0; i < R; ++i) v[k][i] = *reinterpret_cast<const f32x4*>(a.G + (int64_t)(16 * i + r) * a.Vp + w + 4 * g);
    };
    auto multiply = [&](int k) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int c = 0; c < 4; ++c)
#pragma unroll
                for (int i = 0; i < R; ++i) acc[i][c] = mfma4(v[k][i][e], b[k][e][c], acc[i][c]);
    };
    load(0, first + 16 * wave);                               // a part has a multiple of 128 words
    for (int w = first + 16 * wave; w < last; w += 128) {
        load(1, w + 64);
        multiply(0);
        if (w + 128 < last) load(0, w + 128);
        multiply(1);
    }
    __shared__ f32x4 sum[4][R][4][64];
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c) sum[wave][i][c][lane] = acc[i][c];
    __syncthreads();
    if (wave >= R || c0 >= a.Kp) return;
    f32x4 d[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        d[c] = sum[0][wave][c][lane];
#pragma unroll
        for (int k = 1; k < 4; ++k) d[c] += sum[k][wave][c][lane];
    }
    float* out = a.part + ((int64_t)blockIdx.y * a.rows + 16 * wave + 4 * g) * a.Kp + c0;
#pragma unroll
    for (int e = 0; e < 4; ++e) *reinterpret_cast<f32x4*>(out + (int64_t)e * a.Kp) = f32x4{d[0][e], d[1][e], d[2][e], d[3][e]};
}

// dW = G^T x: a wavefront has T groups of 16 words and goes through the columns, 64 at a time.
template <int R, int T, bool VEC>
__global__ __launch_bounds__(256) void few_dw_kernel(FewGrad a) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
    const int w0 = (blockIdx.x * 4 + wave) * 16 * T;          // Vp is a multiple of 256
    const float f = factor_of(a.up, a.head);
    float v[T][4 * R];
#pragma unroll
    for (int st = 0; st < 4 * R; ++st)
#pragma unroll
        for (int t = 0; t < T; ++t) v[t][st] = a.G[(int64_t)(4 * st + g) * a.Vp + w0 + 16 * t + r];
    for (int c0 = blockIdx.y * 64 + 4 * r; c0 - 4 * r < a.K; c0 += 64 * gridDim.y) {
        f32x4 acc[T][4] = {};
#pragma unroll
        for (int st = 0; st < 4 * R; ++st) {
            const f32x4 b = *reinterpret_cast<const f32x4*>(a.xs + (int64_t)(4 * st + g) * a.Kp + min(c0, a.Kp - 4));
#pragma unroll
            for (int c = 0; c < 4; ++c)
#pragma unroll
                for (int t = 0; t < T; ++t) acc[t][c] = mfma4(v[t][st], b[c], acc[t][c]);
        }
#pragma unroll
        for (int t = 0; t < T; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int w = w0 + 16 * t + 4 * g + e;
                if (w >= a.V) continue;
                float* out = a.dW + (int64_t)w * a.lddw + c0;
                if (VEC) {
                    if (c0 < a.K) *reinterpret_cast<f32x4*>(out) = f32x4{acc[t][0][e] * f, acc[t][1][e] * f, acc[t][2][e] * f, acc[t][3][e] * f};
                } else {
#pragma unroll
                    for (int c = 0; c < 4; ++c)
                        if (c0 + c < a.K) out[c] = acc[t][c][e] * f;
                }
            }
    }
}

template <int R>
int few_backward(const FewGrad& a, int split, const int* slot, void* dx, int64_t lddx, hipStream_t s) {
    few_g_kernel<<<a.Vp / 256, 256, 0, s>>>(a);
    const bool even = a.K % 4 == 0;
    if (dx) {
        const dim3 grid((a.Kp + 63) / 64, split);
        if (even && capdec_aligned16(a.W) && a.ldw % 4 == 0) few_dx_kernel<R, true><<<grid, 256, 0, s>>>(a);
        else few_dx_kernel<R, false><<<grid, 256, 0, s>>>(a);
        Splits one;
        one.s[0] = (unsigned char)split;
        int64_t blocks = ((int64_t)a.M * ((a.K + 3) / 4) + 255) / 256;
        dx_kernel<<<(unsigned)(blocks < 8192 ? blocks : 8192), 256, 0, s>>>(a.part, one, a.rows, a.Kp, a.M, a.K, slot, a.tgt, nullptr,
                                                                          a.W, a.ldw, a.head, a.up, 0, dx, lddx, CAPDEC_F32);
    }
    if (a.dW) {
        // at least 2048 wavefronts where the columns allow it
        constexpr int T = 2;
        const int blocks = a.Vp / (64 * T), cols = (a.K + 63) / 64;
        const int y = blocks >= 512 ? 1 : 512 / blocks < cols ? 512 / blocks : cols;
        const dim3 grid(blocks, y);
        if (even && capdec_aligned16(a.dW) && a.lddw % 4 == 0) few_dw_kernel<R, T, true><<<grid, 256, 0, s>>>(a);
        else few_dw_kernel<R, T, false><<<grid, 256, 0, s>>>(a);
    }
    CAPDEC_LAUNCH_CHECK();
    return 0;
}

unsigned blocks_for(int64_t items, int64_t per, unsigned most) {
    int64_t b = (items + per - 1) / per;
    return (unsigned)(b < 1 ? 1 : b > (int64_t)most ? (int64_t)most : b);
}

template <class K>
int allow_lds(K kernel, int bytes) {
    if (bytes <= 64 * 1024) return 0;
    return (int)hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
}

template <class C, int ELT, bool SPLIT, bool BY_ROW = false>
int launch_lse(LogitArgs a, int words, int rows, hipStream_t s) {
    const unsigned grid = make_map(a.map, words / C::BI, rows / C::BJ, 1);
    CAPDEC_TRY(allow_lds(lse_kernel<C, ELT, SPLIT, BY_ROW>, C::LDS_BYTES));
    lse_kernel<C, ELT, SPLIT, BY_ROW><<<grid, C::THREADS, C::LDS_BYTES, s>>>(a);
    CAPDEC_LAUNCH_CHECK();
    return 0;
}
template <class C, int ELT, bool SPLIT>
int launch_dlogits(LogitArgs a, int words, int rows, hipStream_t s) {
    constexpr int turned = C::WAVES * 32 * (32 * C::TI * 2 + 8) * 2 + C::WJ * C::BI * 4;
    constexpr int bytes = turned > C::LDS_BYTES ? turned : C::LDS_BYTES;
    const unsigned grid = make_map(a.map, words / C::BI, rows / C::BJ, 1);
    CAPDEC_TRY(allow_lds(dlogits_kernel<C, ELT, SPLIT>, bytes));
    dlogits_kernel<C, ELT, SPLIT><<<grid, C::THREADS, bytes, s>>>(a);
    CAPDEC_LAUNCH_CHECK();
    return 0;
}
template <class C, int ELT, bool TP, bool SPLIT, int OUT>
int launch_grad(GradArgs a, int I, int J, int64_t most, hipStream_t s) {
    unsigned grid = make_map(a.map, (I + C::BI - 1) / C::BI, (J + C::BJ - 1) / C::BJ, a.nsplit);
    if (most) grid = (unsigned)((most + 7) / 8 * 8);          // dx: the kernel maps what is live
    CAPDEC_TRY(allow_lds(grad_kernel<C, ELT, TP, SPLIT, OUT>, C::LDS_BYTES));
    grad_kernel<C, ELT, TP, SPLIT, OUT><<<grid, C::THREADS, C::LDS_BYTES, s>>>(a);
    CAPDEC_LAUNCH_CHECK();
    return 0;
}

#define BY_TYPE(p, CALL)                                    \
    ((p).split ? CALL(F16, true) : (p).elt == BF16 ? CALL(BF16, false) : CALL(F16, false))

bool valid(const capdec_vocab_ce* a) {
    if (!a || !a->x || !a->W || !a->targets) return false;
    const bool rows = a->M > 1 ? a->ldx >= a->K : a->ldx >= 0;
    return rows && (a->V > 1 ? a->ldw >= a->K : a->ldw >= 0);
}

}  // namespace

extern "C" {

size_t capdec_vocab_ce_saved_bytes(const capdec_vocab_ce* a) {
    Plan p;
    return make_plan(a, p) ? p.saved : 0;
}
size_t capdec_vocab_ce_forward_workspace_bytes(const capdec_vocab_ce* a) {
    Plan p;
    return make_plan(a, p) ? p.fwd : 0;
}
size_t capdec_vocab_ce_backward_workspace_bytes(const capdec_vocab_ce* a) {
    Plan p;
    return make_plan(a, p) ? p.bwd : 0;
}

int capdec_vocab_ce_tiles(const capdec_vocab_ce* a, int32_t* tiles) {
    Plan p;
    CAPDEC_REQUIRE(tiles && make_plan(a, p));
    const int wide = Wide::BI * Wide::BJ, big = Big::BI * Big::BJ, mid = Mid::BI * Mid::BJ;
    tiles[0] = p.few ? 0 : p.few_z ? mid : p.wide_z ? wide : big;
    tiles[1] = p.few || a->loss_only ? 0 : p.wide_dx ? wide : big;
    tiles[2] = p.few || a->loss_only ? 0 : p.wide_dw ? wide : big;
    return 0;
}

int capdec_vocab_ce_forward(const capdec_vocab_ce* a, void* saved, size_t saved_bytes, void* workspace,
                            size_t workspace_bytes, float* nll, float* loss, void* stream) {
    Plan p;
    CAPDEC_REQUIRE(valid(a) && make_plan(a, p) && saved && workspace && nll);
    if (!capdec_aligned16(saved) || !capdec_aligned16(workspace)) return CAPDEC_EALIGN;
    if (saved_bytes < p.saved || workspace_bytes < p.fwd) return CAPDEC_ENOMEM;
    hipStream_t s = (hipStream_t)stream;
    char* sv = (char*)saved;
    Head* head = (Head*)sv;
    int* order = (int*)(sv + p.o_order);
    int* slot = (int*)(sv + p.o_slot);
    int* tgt = (int*)(sv + p.o_tgt);
    const int esz = p.split ? 4 : 2;
    const int vec = capdec_aligned16(a->x) && capdec_aligned16(a->W) && a->ldx * esz % 16 == 0 && a->ldw * esz % 16 == 0;
    if (p.few) {
        ScanArgs sc{a->targets, p.M, p.V, p.K, a->ignore_index, head, order, slot, tgt, nullptr, 0, nullptr, 0, 0, 0, nullptr};
        scan_kernel<<<1, 1024, 0, s>>>(sc);
        float2* part = (float2*)((char*)workspace + p.o_part);
        const FewArgs f{(const float*)a->x, a->ldx, (const float*)a->W, a->ldw, (const float*)a->bias, p.M, p.V, p.K, p.Vp, head,
                        order, p.Kp, (float*)(sv + p.o_x), (float*)(sv + p.o_z), part, tgt, (float*)(sv + p.o_dlt)};
        const bool v4 = vec && p.K % 4 == 0;
        if (p.few_rows == 16) launch_few_lse<1>(f, v4, s);
        else if (p.few_rows == 32) launch_few_lse<2>(f, v4, s);
        else launch_few_lse<4>(f, v4, s);
        nll_kernel<true><<<p.M, 1024, 0, s>>>(part, p.Vp / 32, 0, p.M, head, order, slot, tgt, (float*)(sv + p.o_lse),
                                              (float*)(sv + p.o_dlt), nll);
        if (loss) loss_kernel<<<1, 1024, 0, s>>>(nll, p.M, head, loss);
        CAPDEC_LAUNCH_CHECK();
        return 0;
    }
    PackArgs k{};
    ScanArgs sc{a->targets, p.M, p.V, p.K, a->ignore_index, head, order, slot, tgt, (const float*)a->x, a->ldx, (const float*)a->W,
                a->ldw, 0, vec && p.K % 4 == 0, (float2*)((char*)workspace + p.o_amax)};
    if (p.split && !p.by_row) sc.nparts = (int)blocks_for((int64_t)(p.V > p.M ? p.V : p.M), 16, AMAX_BLOCKS);
    scan_kernel<<<1 + 2 * sc.nparts, 1024, 0, s>>>(sc);
    k.nparts = sc.nparts;
    k.part = sc.part;
    k.x = a->x; k.ldx = a->ldx; k.W = a->W; k.ldw = a->ldw; k.bias = a->bias;
    k.M = p.M; k.V = p.V; k.K = p.K; k.Kp = p.Kp; k.xs = p.xs; k.dtype = a->dtype; k.split = p.split; k.Vp = p.Vp;
    k.pack_w = p.pack_w; k.vec = vec;
    k.head = head; k.order = order;
    k.px = (short*)(sv + p.o_x); k.pw = (short*)(sv + p.o_w); k.b2 = (float*)(sv + p.o_b2);
    k.nx = (int64_t)p.Mp * (p.Kp / 8);
    k.nw = p.pack_w ? (int64_t)p.V * (p.Kp / 8) : 0;
    const RowScales f{(float*)(sv + p.o_sx), (float*)(sv + p.o_sw)};
    if (p.by_row) {
        const unsigned grid = blocks_for((int64_t)p.M + p.V, 4, 8192);
        vec && p.K % 4 == 0 ? pack_rows_kernel<true><<<grid, 256, 0, s>>>(k, f) : pack_rows_kernel<false><<<grid, 256, 0, s>>>(k, f);
    } else {
        pack_kernel<<<blocks_for(k.nx + k.nw + p.Vp, 256, 8192), 256, 0, s>>>(k);
    }
    CAPDEC_LAUNCH_CHECK();

    LogitArgs g{};
    g.W = View{p.pack_w ? k.pw : (const short*)a->W, p.pack_w ? (int64_t)p.xs : a->ldw, p.V, 0};
    g.X = View{k.px, (int64_t)p.xs, p.Mp, 0};
    if (p.split) {
        g.W32 = View32{(const float*)a->W, a->ldw, nullptr, p.V};
        g.X32 = View32{(const float*)a->x, a->ldx, order, 0};              // (as many rows as are counted)
        g.K = p.K;
    }
    g.b2 = k.b2; g.head = head; g.kt = p.xs / 32; g.Mp = p.Mp;
    g.part = (float2*)((char*)workspace + p.o_part);
    g.tgt = tgt; g.zt = (float*)(sv + p.o_dlt);
#define LSE(E, S)                                                  \
    (p.few_z    ? launch_lse<Mid, E, S>(g, p.Vp, p.Mp, s)          \
     : p.wide_z ? launch_lse<Wide, E, S>(g, p.Vp, p.Mp, s)         \
                : launch_lse<Big, E, S>(g, p.Vp, p.Mp, s))
    if (p.by_row) {
        g.f = f;
        CAPDEC_TRY((p.few_z    ? launch_lse<Mid, F16, true, true>(g, p.Vp, p.Mp, s)
                    : p.wide_z ? launch_lse<Wide, F16, true, true>(g, p.Vp, p.Mp, s)
                               : launch_lse<Big, F16, true, true>(g, p.Vp, p.Mp, s)));
    } else {
        CAPDEC_TRY(BY_TYPE(p, LSE));
    }
#undef LSE
    nll_kernel<false><<<(p.M + 63) / 64, 1024, 0, s>>>(g.part, p.Vp / p.z_words, p.Mp, p.M, head, order, slot, tgt,
                                                       (float*)(sv + p.o_lse), (float*)(sv + p.o_dlt), nll);
    if (loss) loss_kernel<<<1, 1024, 0, s>>>(nll, p.M, head, loss);
    CAPDEC_LAUNCH_CHECK();
    return 0;
}

int capdec_vocab_ce_backward(const capdec_vocab_ce* a, const void* saved, size_t saved_bytes, void* workspace,
                             size_t workspace_bytes, const float* row_grad, const float* grad, int mean, void* dx,
                             int64_t lddx, void* dW, int64_t lddw, void* dbias, void* stream) {
    Plan p;
    CAPDEC_REQUIRE(valid(a) && !a->loss_only && make_plan(a, p) && saved && workspace && !(row_grad && grad));
    CAPDEC_REQUIRE(!dx || p.M == 1 || lddx >= p.K);
    CAPDEC_REQUIRE(!dW || p.V == 1 || lddw >= p.K);
    CAPDEC_REQUIRE(!dbias || a->bias);
    if (!capdec_aligned16(saved) || !capdec_aligned16(workspace)) return CAPDEC_EALIGN;
    if (saved_bytes < p.saved || workspace_bytes < p.bwd) return CAPDEC_ENOMEM;
    if (!dx && !dW && !dbias) return 0;
    hipStream_t s = (hipStream_t)stream;
    const char* sv = (const char*)saved;
    char* ws = (char*)workspace;
    const Head* head = (const Head*)sv;
    const int* order = (const int*)(sv + p.o_order);
    const int* slot = (const int*)(sv + p.o_slot);
    float* rw = row_grad ? (float*)(ws + p.o_rw) : nullptr;
    const int gexp = p.few || (!p.split && p.elt == BF16) ? 0 : G_EXP;
    const Upstream up{row_grad ? (const BwdHead*)ws : nullptr, grad, mean, gexp};
    float* rest = (float*)(ws + p.o_rest);
    if (row_grad) {
        weights_kernel<<<1, 1024, 0, s>>>(row_grad, head, order, p.Mp, gexp, rw, (BwdHead*)ws);
        CAPDEC_LAUNCH_CHECK();
    }
    if (p.few) {
        const FewGrad f{(const float*)(sv + p.o_x), (const float*)a->W, a->ldw, p.M, p.V, p.K, p.Kp, p.Vp, head,
                        (const int*)(sv + p.o_tgt), (const float*)(sv + p.o_z), (const float*)(sv + p.o_lse),
                        (const float*)(sv + p.o_dlt), rw, up, (float*)(ws + p.o_g), p.few_rows, p.few_words,
                        (float*)(ws + p.o_dx), (float*)dW, lddw, (float*)dbias};
        return p.few_rows == 16 ? few_backward<1>(f, p.few_split, slot, dx, lddx, s)
             : p.few_rows == 32 ? few_backward<2>(f, p.few_split, slot, dx, lddx, s)
                                : few_backward<4>(f, p.few_split, slot, dx, lddx, s);
    }
    const short* px = (const short*)(sv + p.o_x);
    const short* W = p.pack_w ? (const short*)(sv + p.o_w) : (const short*)a->W;
    const int64_t ldw = p.pack_w ? p.xs : a->ldw;
    const int kt = p.split ? 16 : 32, pl = p.split ? 2 : 1;
    short* G = (short*)(ws + p.o_g);
    float* dxp = (float*)(ws + p.o_dx);
    for (int v0 = 0; v0 < p.V; v0 += p.piece) {
        const int words = p.Vp - v0 < p.piece ? p.Vp - v0 : p.piece;      // a multiple of 256
        const int real = p.V - v0 < words ? p.V - v0 : words;
        LogitArgs g{};
        g.W = View{W, ldw, p.V, 0};
        g.X = View{px, (int64_t)p.xs, p.Mp, 0};
        if (p.split) {
            g.W32 = View32{(const float*)a->W, a->ldw, nullptr, p.V};
            g.X32 = View32{(const float*)px, p.Kp, nullptr, 0};
            g.K = p.K;
        }
        g.b2 = (const float*)(sv + p.o_b2); g.head = head; g.kt = p.xs / 32; g.Mp = p.Mp;
        g.lse = (const float*)(sv + p.o_lse); g.dlt = (const float*)(sv + p.o_dlt); g.rw = rw; g.tgt = (const int*)(sv + p.o_tgt);
        g.g = G; g.ldg = (int64_t)p.piece * pl; g.rest = rest; g.dbp = dbias ? (float*)(ws + p.o_db) : nullptr; g.v0 = v0; g.piece = p.piece; g.gexp = gexp;
#define DL(E, S)                                                   \
    (p.few_z    ? launch_dlogits<Mid, E, S>(g, words, p.Mp, s)     \
     : p.wide_z ? launch_dlogits<Wide, E, S>(g, words, p.Mp, s)    \
                : launch_dlogits<Big, E, S>(g, words, p.Mp, s))
        CAPDEC_TRY(BY_TYPE(p, DL));
#undef DL
        if (dx) {
            GradArgs d{};
            d.P = View{G, g.ldg, p.Mp, 0};
            d.Q = View{W + (int64_t)v0 * ldw, ldw, p.Kp, real};
            if (p.split) {
                d.P32 = View32{(const float*)G, p.piece, nullptr, p.Mp};
                d.Q32 = View32{(const float*)a->W + (int64_t)v0 * a->ldw, a->ldw, nullptr, p.K};
                d.k32 = real;
            }
            d.head = head; d.up = up; d.I = p.Mp; d.J = p.Kp; d.rows_live = 1; d.kt = words / kt; d.splits = p.sx;
            d.part = dxp; d.ldp = p.Kp; d.add = v0 > 0;
#define DX(E, S) (p.wide_dx ? launch_grad<Wide, E, false, S, 0>(d, p.Mp, p.Kp, p.dx_tiles, s) : launch_grad<Big, E, false, S, 0>(d, p.Mp, p.Kp, p.dx_tiles, s))
            CAPDEC_TRY(BY_TYPE(p, DX));
#undef DX
        }
        if (dW) {
            GradArgs d{};
            d.P = View{G, g.ldg, words, p.Mp};
            d.Q = View{px, (int64_t)p.xs, p.Kp, p.Mp};
            if (p.split) {
                d.P32 = View32{(const float*)G, p.piece, nullptr, words};
                d.Q32 = View32{(const float*)px, p.Kp, nullptr, p.Kp};
            }
            d.head = head; d.up = up; d.k_live = 1; d.nsplit = p.sw;
            d.tgt = g.tgt; d.rest = rest; d.v0 = v0;
            if (p.sw == 1) {
                d.I = real; d.J = p.K;
                d.out = (char*)dW + (int64_t)v0 * lddw * (p.split ? 4 : 2); d.ldo = lddw; d.dtype = a->dtype;
                d.vec = capdec_aligned16(dW) && lddw % 8 == 0 && p.K % 8 == 0;
#define DW(E, S) (p.wide_dw ? launch_grad<Wide, E, true, S, 1>(d, words, p.Kp, 0, s) : launch_grad<Big, E, true, S, 1>(d, words, p.Kp, 0, s))
                CAPDEC_TRY(BY_TYPE(p, DW));
#undef DW
            } else {
                d.I = real; d.J = p.Kp;
                d.part = (float*)(ws + p.o_dw); d.ldp = p.Kp; d.plane = (int64_t)p.piece * p.Kp;
#define DW(E, S) (p.wide_dw ? launch_grad<Wide, E, true, S, 0>(d, words, p.Kp, 0, s) : launch_grad<Big, E, true, S, 0>(d, words, p.Kp, 0, s))
                CAPDEC_TRY(BY_TYPE(p, DW));
#undef DW
            }
        }
        const int slabs = dW ? p.sw : 1;
        if (slabs > 1 || dbias) {
            const int64_t items = (slabs > 1 ? (int64_t)real * ((p.K + 3) / 4) : 0) + (dbias ? real : 0);
            dw_kernel<<<blocks_for(items, 256, 8192), 256, 0, s>>>((const float*)(ws + p.o_dw), (int64_t)p.piece * p.Kp, slabs,
                                                                   p.Kp, real, p.K, head, up, p.split, dW, lddw, a->dtype,
                                                                   g.dbp, p.piece, p.z_rows, dbias, v0);
            CAPDEC_LAUNCH_CHECK();
        }
    }
    if (dx) {
        dx_kernel<<<blocks_for((int64_t)p.M * ((p.K + 3) / 4), 256, 8192), 256, 0, s>>>(
            dxp, p.sx, 0, p.Kp, p.M, p.K, slot, (const int*)(sv + p.o_tgt), p.split ? nullptr : rest, a->W, a->ldw, head, up,
            p.split, dx, lddx, a->dtype);
        CAPDEC_LAUNCH_CHECK();
    }
    return 0;
}

}  // extern "C"
