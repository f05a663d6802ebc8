// Orthogonalised updates of weight matrices.
//
//   X_0 = U / (|U|_F + eps);   A = X X^T,  B = b A + c A^2,  X <- a X + B X     (steps times)
//
// on the shorter side: a tall matrix takes A = X^T X and X <- a X + X B, read through the transposing operand paths, so
// nothing is transposed in memory.  Three products per step, 2 (2 m^2 n + m^3) flops, m <= n: bound by the matrix cores
// from about 1000 x 1000 on, by launch and pipeline latency below.
// The iterate, A and B are kept as pairs of fp16 numbers times a power of two (SPLIT in mma16.h) with fp32 sums: an error
// made while r steps remain grows by up to a^r (3.4^r for the usual coefficients) in the directions whose singular
// values are still small, so the steps need fp32's digits whatever the matrices' type.  (Single fp16 numbers in the last
// two steps towards a bfloat16 result, a third of their products, made 1530 us of 1900 for 2048 x 8192, but left it up to
// 3.2e-3 off in norm, depending on the spectrum, where rounding alone is 1.7e-3; in the last step alone, 2.2e-3.)  The
// powers of two come from the exact maxima of the polynomials on the interval that the singular values can be in.
#include "mma16.h"
#include <math.h>

using namespace mma16;

namespace {

constexpr int MAX_BATCH = 32;             // matrices per launch (their descriptors are kernel arguments)
constexpr size_t BATCH_BYTES = (size_t)1 << 30;
constexpr int NORM_BLOCKS = 512;          // most partial sums of squares per matrix
constexpr int CHUNK = 1024;               // columns a wavefront reads of a row at a time

struct Item {
    const void* src;                      // orthogonalize: the matrix;  update: the gradient
    void* dst;                            // orthogonalize: the result;  update: the parameter
    float* mom;                           // update: the momentum
    int64_t lds, ldd, ldm;
};
struct Batch {
    Item it[MAX_BATCH];
};

// A and A^2 are symmetric: from 768 on, the upper triangle of 256 x 256 or 128 x 128 tiles, its contraction in parts where
// that fills the CUs better.  Times in us from measurements of split operands (a k-tile takes a CU 1.36 with one 256 x 256
// tile; 0.58, 0.80, 1.15 with one to three 128 x 128 tiles); the parts' sums go to memory and back at 4 TB/s.  (With 0.45 for
// one tile A^2 of 2048 stayed a whole square: 2048 x 2048 910 instead of 770 us, 2560 x 2560 1226 instead of 1263.)
// From 768 on: 16 matrices of 768 x 768 take 817 us as triangles and 987 whole, 768 x 4096 358 and 398; one square matrix would
// be faster whole up to 1024 (768: 249 and 187, 1024: 279 and 233), batches of 640 slower (16 of them: 568, as triangles 498).
struct Symmetric {
    bool on, wide;
    int nsplit;
    size_t slab;                   // bytes of partial sums for a batch
};
Symmetric symmetric_plan(int m, int kt, int nz) {
    Symmetric best{false, false, 1, 0};
    if (m < 768) return best;
    auto mids = [](int64_t n) {
        const int64_t per = (n + 255) / 256, left = per % 3;
        return (double)(per / 3) * 1.15 + (left == 2 ? 0.80 : left == 1 ? 0.58 : 0.0);
    };
    const int64_t w = (m + 255) / 256, h = (m + 127) / 128;
    // the whole square, by the rule of launch_sized
    double least = 0.9 * (w * w * nz >= 256 ? (double)((w * w * nz + 255) / 256) * 1.36 : mids(h * h * nz)) * kt;
    for (int wide = 0; wide < 2; ++wide)
        for (int s = 1; s <= 8 && kt / s >= 8; ++s) {
            const int64_t n = (wide ? w * (w + 1) / 2 : h * (h + 1) / 2) * nz * s;
            const size_t slab = s > 1 ? (size_t)n * (wide ? 256 * 256 : 128 * 128) * 4 : 0;
            if (slab > (size_t)512 << 20) break;
            const double t = (wide ? (double)((n + 255) / 256) * 1.36 : mids(n)) * ((kt + s - 1) / s) + (s > 1 ? 5 + 2e-6 * slab / 4 : 0);
            if (t < least) least = t, best = Symmetric{true, wide != 0, s, slab};
        }
    return best;
}

struct Dims {
    int rows, cols, rp, cp, m;            // rp, cp: rounded up to 32; m: the shorter of the two
    bool tall;
    size_t x_elems, a_elems;              // 16-bit elements of one matrix
    size_t per, norm, slab;               // workspace bytes: per matrix, of a batch's sums of squares, of partial products
    int batch;
};

bool make_dims(int count, int rows, int cols, Dims& d) {
    if (count < 1 || rows < 1 || cols < 1 || rows > (1 << 20) || cols > (1 << 20)) return false;
    if ((int64_t)rows * cols > (int64_t)1 << 31) return false;
    d.rows = rows; d.cols = cols;
    d.rp = (rows + 31) / 32 * 32;
    d.cp = (cols + 31) / 32 * 32;
    d.tall = rows > cols;
    d.m = d.tall ? d.cp : d.rp;
    d.x_elems = (size_t)d.rp * d.cp * 2;
    d.a_elems = (size_t)d.m * d.m * 2;
    d.per = (2 * d.x_elems + 2 * d.a_elems) * 2;
    size_t b = BATCH_BYTES / d.per;
    d.batch = b < 1 ? 1 : b > MAX_BATCH ? MAX_BATCH : (int)b;
    if (d.batch > count) d.batch = count;
    d.norm = (size_t)d.batch * NORM_BLOCKS * 8;
    d.slab = 0;                           // the most that a product of this batch, or of the rest of the matrices, may take
    const int n = d.tall ? d.rp : d.cp, rest = count % d.batch ? count % d.batch : d.batch;
    for (int nz : {d.batch, rest})
        for (int k : {n, d.m}) {
            const size_t b = symmetric_plan(d.m, k / 16, nz).slab;
            if (b > d.slab) d.slab = b;
        }
    return true;
}

__device__ __forceinline__ float load_as_f32(const void* p, int64_t i, int dtype) {
    if (dtype == CAPDEC_F32) return ((const float*)p)[i];
    const short b = ((const short*)p)[i];
    return dtype == CAPDEC_BF16 ? from_bits<BF16>(b) : from_bits<F16>(b);
}
__device__ __forceinline__ void store_as(void* p, int64_t i, float v, int dtype) {
    if (dtype == CAPDEC_F32) ((float*)p)[i] = v;
    else ((short*)p)[i] = dtype == CAPDEC_BF16 ? to_bits<BF16>(v) : to_bits<F16>(v);
}

// four consecutive elements, aligned to their own size
__device__ __forceinline__ void load4(const void* p, int64_t i, int dtype, float* v) {
    if (dtype == CAPDEC_F32) {
        const f32x4 q = *reinterpret_cast<const f32x4*>((const float*)p + i);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = q[e];
    } else {
        const s16x4 q = *reinterpret_cast<const s16x4*>((const short*)p + i);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = dtype == CAPDEC_BF16 ? from_bits<BF16>(q[e]) : from_bits<F16>(q[e]);
    }
}

struct Momentum {                         // update only (on != 0)
    int on, nesterov;
    float mu, grad_scale;
};

// the next momentum; u: the gradient in, U out
__device__ __forceinline__ float advance(const Momentum& mo, float m, float& u) {
    u *= mo.grad_scale;
    m = fmaf(mo.mu, m, u);
    u = mo.nesterov ? fmaf(mo.mu, m, u) : m;
    return m;
}

// Sums of squares of U in double (no square over- or underflows), one partial per block in a fixed order; an update
// advances its momentum here.  A wavefront per row and 1024 columns, four elements of each lane in flight when the
// rows are aligned.
__global__ __launch_bounds__(256) void norm_kernel(Batch b, int rows, int cols, int dtype, Momentum mo, int vec,
                                                   double* __restrict__ part) {
    const Item& it = b.it[blockIdx.y];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int cpr = (cols + CHUNK - 1) / CHUNK;
    double s = 0.0;
    for (int64_t t = (int64_t)blockIdx.x * 4 + wave; t < (int64_t)rows * cpr; t += (int64_t)gridDim.x * 4) {
        const int r = (int)(t / cpr), c0 = (int)(t - (int64_t)r * cpr) * CHUNK, c1 = min(cols, c0 + CHUNK);
        const int64_t src = (int64_t)r * it.lds, mom = (int64_t)r * it.ldm;
        if (vec) {
#pragma unroll
            for (int k = 0; k < CHUNK / 256; ++k) {
                const int c = c0 + k * 256 + lane * 4;
                if (c >= c1) break;
                float u[4];
                load4(it.src, src + c, dtype, u);
                if (mo.on) {
                    f32x4 m = *reinterpret_cast<const f32x4*>(it.mom + mom + c);
#pragma unroll
                    for (int e = 0; e < 4; ++e) m[e] = advance(mo, m[e], u[e]);
                    *reinterpret_cast<f32x4*>(it.mom + mom + c) = m;
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) s += (double)u[e] * (double)u[e];
            }
        } else {
            for (int c = c0 + lane; c < c1; c += 64) {
                float u = load_as_f32(it.src, src + c, dtype);
                if (mo.on) it.mom[mom + c] = advance(mo, it.mom[mom + c], u);
                s += (double)u * (double)u;
            }
        }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    __shared__ double ws[4];
    if (lane == 0) ws[wave] = s;
    __syncthreads();
    if (threadIdx.x == 0) part[blockIdx.y * NORM_BLOCKS + blockIdx.x] = (ws[0] + ws[1]) + (ws[2] + ws[3]);
}

// X_0 2^sx = U 2^sx / (|U| + eps) into the padded layout
__global__ __launch_bounds__(256) void normalise_kernel(Batch b, int rows, int cols, int rp, int cp, int dtype, Momentum mo,
                                                        int vec, const double* __restrict__ part, int nparts, float eps,
                                                        float scale, short* __restrict__ X, int64_t x_elems) {
    const Item& it = b.it[blockIdx.y];
    double s = 0.0;
    for (int k = threadIdx.x & 63; k < nparts; k += 64) s += part[blockIdx.y * NORM_BLOCKS + k];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    int e2 = 0;                        // 1 / (|U| + eps) may be more than an fp32 number holds
    const float inv = s == 0.0 ? 0.f : (float)frexp((double)scale / (sqrt(s) + (double)eps), &e2);
    short* x = X + blockIdx.y * x_elems;
    const int cpr = cp / 8;
    for (int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x; t < (int64_t)rp * cpr; t += (int64_t)gridDim.x * 256) {
        const int r = (int)(t / cpr), c = (int)(t - (int64_t)r * cpr) * 8;
        const int64_t src = (int64_t)r * it.lds + c, mom = (int64_t)r * it.ldm + c;
        float u[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, m[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (r < rows) {
            if (vec && c + 8 <= cols) {
                if (!mo.on || mo.nesterov) {
                    load4(it.src, src, dtype, u);
                    load4(it.src, src + 4, dtype, u + 4);
                }
                if (mo.on) {
                    load4(it.mom, mom, CAPDEC_F32, m);
                    load4(it.mom, mom + 4, CAPDEC_F32, m + 4);
                }
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (c + e < cols) {
                        u[e] = load_as_f32(it.src, src + e, dtype);
                        if (mo.on) m[e] = it.mom[mom + e];
                    }
            }
        }
        s16x8 hi, lo;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if (mo.on) u[e] = mo.nesterov ? fmaf(mo.mu, m[e], u[e] * mo.grad_scale) : m[e];
            short h, l;
            split16(ldexpf(u[e], e2) * inv, h, l);
            hi[e] = h;
            lo[e] = l;
        }
        short* d = x + (int64_t)r * cp * 2 + split_col(c);
        *reinterpret_cast<s16x8*>(d) = hi;
        *reinterpret_cast<s16x8*>(d + 16) = lo;
    }
}

// One product of a step for a batch of matrices: out = alpha P Q^T + beta R.
struct StepArgs {
    View P, Q;
    int64_t strideP, strideQ, strideR, strideO;   // 16-bit elements between the batch's matrices
    const short* R;                // stored like the operands, [i][j]; nullable
    int64_t ldr;
    float alpha, beta;
    int I, J, kt;
    int tri;                       // symmetric result: only the tiles on and above the diagonal, mirrored as they are stored
    int nsplit; float* slab;       // contraction in parts: partial sums [matrix][part][tile][accumulator][thread]
    Map map;
    short* out; int64_t ldo;       // inner products
    // last product of the last step
    Batch b; int dtype;
    float lr, decay, scale;        // update: p <- p (1 - lr decay) - lr scale out
    const capdec_train_state* st;  // nullable: lr is read from it
};
enum { INNER = 0, RESULT = 1, UPDATE = 2 };

// WHOLE: contraction and epilogue.  PART: the contraction of one of nsplit parts, its sums to the slab.  JOIN: the parts'
// sums added in order, then the epilogue; a workgroup per accumulator of a tile (blockIdx.y).
enum { WHOLE = 0, PART = 1, JOIN = 2 };

template <class C, bool TP, bool TQ, int OUT, int PHASE>
__global__ __launch_bounds__(C::THREADS, C::EU) void step_kernel(StepArgs a) {
    extern __shared__ __attribute__((aligned(16))) short lds[];
    int ti_, tj_, z;
    if (!tile_of(a.map, blockIdx.x, ti_, tj_, z)) return;
    const int tiles = a.map.ni * a.map.nj, tile = ti_ * a.map.nj + tj_;
    if (a.tri) {                   // the map runs over the triangle's tiles along one axis: column tj_ of it holds tj_ + 1
        tj_ = (int)((sqrtf(8.f * ti_ + 1.f) - 1.f) * 0.5f);
        while ((tj_ + 1) * (tj_ + 2) / 2 <= ti_) ++tj_;
        while (tj_ * (tj_ + 1) / 2 > ti_) --tj_;
        ti_ -= tj_ * (tj_ + 1) / 2;
    }
    const int i0 = ti_ * C::BI, j0 = tj_ * C::BJ;
    const int mat = PHASE == PART ? z / a.nsplit : z;
    constexpr int ACCS = C::TI * C::TJ;
    f32x16 acc[C::TI][C::TJ];
    if (PHASE != JOIN) {
        View P = a.P, Q = a.Q;
        P.p += mat * a.strideP;
        Q.p += mat * a.strideQ;
        const int part = z - mat * (PHASE == PART ? a.nsplit : 1), per = PHASE == PART ? (a.kt + a.nsplit - 1) / a.nsplit : a.kt;
        contract<C, F16, TP, TQ, true>(P, Q, i0, j0, part * per, min(a.kt, (part + 1) * per), lds, acc);
        if (threadIdx.x >= C::GROUP) return;
    }
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));
    if (PHASE == PART) {
        float* d = a.slab + ((int64_t)z * tiles + tile) * (ACCS * 16 * C::GROUP) + tid;
#pragma unroll
        for (int e = 0; e < ACCS * 16; ++e) d[e * C::GROUP] = acc[e / 16 / C::TJ][e / 16 % C::TJ][e % 16];
        return;
    }
    const int lane = tid & 63, wave = tid >> 6, wi = wave / C::WJ, wj = wave % C::WJ, h = lane >> 5;
    const short* R = a.R ? a.R + mat * a.strideR : nullptr;
    float lr = a.lr;
    if (OUT == UPDATE && a.st) lr = a.st->lr;
    auto finish = [&](int ti, int tj, const f32x16& sum) {
        const int j = j0 + (wj * C::TJ + tj) * 32 + (lane & 31), ib = i0 + (wi * C::TI + ti) * 32;
        if (j >= a.J) return;
        const int64_t js = split_col(j);
        float v[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) v[e] = a.alpha * sum[e];
        if (R) {                       // every load first, without branches: one round trip
            short hi[16], lo[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const short* q = R + (int64_t)min(ib + acc_row(e, h), a.I - 1) * a.ldr + js;
                hi[e] = q[0];
                lo[e] = q[16];
            }
#pragma unroll
            for (int e = 0; e < 16; ++e)
                v[e] = fmaf(a.beta, from_bits<F16>(hi[e]) + from_bits<F16>(lo[e]), v[e]);
        }
        if (OUT == INNER) {
            short* out = a.out + mat * a.strideO;
            s16x4 hi[4], lo[4];
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                short p, r;
                split16(v[e], p, r);
                hi[e / 4][e % 4] = p;
                lo[e / 4][e % 4] = r;
                const int i = ib + acc_row(e, h);
                if (i >= a.I) continue;
                short* d = out + (int64_t)i * a.ldo + js;
                d[0] = p;
                d[16] = r;
            }
            if (a.tri && ti_ != tj_) {
                // row j of the mirrored tile: four neighbours at a time (I is a multiple of 32)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int i = ib + 8 * q + 4 * h;
                    if (i >= a.I) continue;
                    short* d = out + (int64_t)j * a.ldo + split_col(i);
                    *reinterpret_cast<s16x4*>(d) = hi[q];
                    *reinterpret_cast<s16x4*>(d + 16) = lo[q];
                }
            }
            return;
        }
        const Item& it = a.b.it[mat];
        float old[16];
        if (OUT == UPDATE) {
#pragma unroll
            for (int e = 0; e < 16; ++e)
                old[e] = ((const float*)it.dst)[(int64_t)min(ib + acc_row(e, h), a.I - 1) * it.ldd + j];
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const int i = ib + acc_row(e, h);
            if (i >= a.I) continue;
            const int64_t at = (int64_t)i * it.ldd + j;
            if (OUT == RESULT) store_as(it.dst, at, v[e], a.dtype);
            else ((float*)it.dst)[at] = fmaf(-lr * a.scale, v[e], old[e] * (1.f - lr * a.decay));
        }
    };
    if (PHASE == JOIN) {
        const int ac = blockIdx.y;
        f32x16 sum;
#pragma unroll
        for (int e = 0; e < 16; ++e) sum[e] = 0.f;
        for (int k = 0; k < a.nsplit; ++k) {
            const float* d = a.slab + ((((int64_t)mat * a.nsplit + k) * tiles + tile) * ACCS + ac) * (16 * C::GROUP) + tid;
#pragma unroll
            for (int e = 0; e < 16; ++e) sum[e] += d[e * C::GROUP];
        }
        finish(ac / C::TJ, ac % C::TJ, sum);
    } else {
#pragma unroll
        for (int tj = 0; tj < C::TJ; ++tj)
#pragma unroll
            for (int ti = 0; ti < C::TI; ++ti) finish(ti, tj, acc[ti][tj]);
    }
}

template <class C, bool TP, bool TQ, int OUT, int PHASE>
int launch(const StepArgs& a0, int nz, hipStream_t s) {
    StepArgs a = a0;
    int ni = (a.I + C::BI - 1) / C::BI, nj = (a.J + C::BJ - 1) / C::BJ;
    if (a.tri) {
        ni = ni * (ni + 1) / 2;
        nj = 1;
    }
    const unsigned grid = make_map(a.map, ni, nj, PHASE == PART ? nz * a.nsplit : nz);
    constexpr int bytes = PHASE == JOIN ? 0 : C::LDS_BYTES;
    if (bytes > 64 * 1024)
        CAPDEC_TRY((int)hipFuncSetAttribute(reinterpret_cast<const void*>(step_kernel<C, TP, TQ, OUT, PHASE>),
                                            hipFuncAttributeMaxDynamicSharedMemorySize, bytes));
    step_kernel<C, TP, TQ, OUT, PHASE><<<dim3(grid, PHASE == JOIN ? C::TI * C::TJ : 1), PHASE == JOIN ? C::GROUP : C::THREADS, bytes, s>>>(a);
    CAPDEC_LAUNCH_CHECK();
    return 0;
}

// the largest tiles that give every CU one, from 256x256 to 64x64; fewer than two of those for each: four groups to a tile
template <bool TP, bool TQ, int OUT>
int launch_sized(const StepArgs& a, int nz, hipStream_t s) {
    auto tiles = [&](int bi, int bj) { return (int64_t)((a.I + bi - 1) / bi) * ((a.J + bj - 1) / bj) * nz; };
    if (tiles(256, 256) >= 256) return launch<Wide, TP, TQ, OUT, WHOLE>(a, nz, s);
    if (tiles(256, 128) >= 256) return launch<Big, TP, TQ, OUT, WHOLE>(a, nz, s);
    if (tiles(128, 128) >= 256) return launch<Mid, TP, TQ, OUT, WHOLE>(a, nz, s);
    if (tiles(64, 64) >= 512) return launch<Small, TP, TQ, OUT, WHOLE>(a, nz, s);
    return launch<Deep, TP, TQ, OUT, WHOLE>(a, nz, s);
}

// A symmetric product of a batch, into planes of the operands' layout.
template <bool T>
int launch_symmetric(StepArgs a, int nz, float* slab, hipStream_t s) {
    const Symmetric p = symmetric_plan(a.I, a.kt, nz);
    a.tri = p.on; a.nsplit = p.nsplit; a.slab = slab;
    if (!p.on) return launch_sized<T, T, INNER>(a, nz, s);
    if (p.nsplit == 1) return p.wide ? launch<Wide, T, T, INNER, WHOLE>(a, nz, s) : launch<Mid, T, T, INNER, WHOLE>(a, nz, s);
    CAPDEC_TRY((p.wide ? launch<Wide, T, T, INNER, PART>(a, nz, s) : launch<Mid, T, T, INNER, PART>(a, nz, s)));
    return p.wide ? launch<Wide, T, T, INNER, JOIN>(a, nz, s) : launch<Mid, T, T, INNER, JOIN>(a, nz, s);
}

// Largest |p(x)| on [0, top] of a x + b x^3 + c x^5 (odd) or b x + c x^2: ends and stationary points.
double top_of_step(double a, double b, double c, double top) {
    auto f = [&](double x) { return fabs(x * (a + x * x * (b + x * x * c))); };
    double best = f(top);
    auto root = [&](double y) {                   // y = x^2 of a stationary point: a + 3 b y + 5 c y^2 = 0
        if (y > 0 && y < top * top) best = fmax(best, f(sqrt(y)));
    };
    if (c != 0) {
        const double q = 9 * b * b - 20 * a * c;
        if (q >= 0) {
            root((-3 * b + sqrt(q)) / (10 * c));
            root((-3 * b - sqrt(q)) / (10 * c));
        }
    } else if (b != 0) {
        root(-a / (3 * b));
    }
    return best;
}
double top_of_poly(double b, double c, double top) {
    double best = fabs(top * (b + c * top));
    if (c != 0) {
        const double x = -b / (2 * c);
        if (x > 0 && x < top) best = fmax(best, fabs(x * (b + c * x)));
    }
    return best;
}
// power of two that brings values up to `top` below 2^15 (fp16 ends at 65504), with room for rounding
int exponent_for(double top) {
    if (!(top > 0)) return 14;
    int e;
    frexp(top * 1.01, &e);                        // top < 2^e
    return e < -45 ? 60 : 15 - e;                 // an iterate that shrinks away needs no more
}

struct Iteration {
    int steps;
    float a, b, c, eps;
};

int run_batch(const Batch& b, int nz, const Dims& d, const Iteration& n, int dtype, const Momentum& mo, char* ws,
              const StepArgs& last, hipStream_t s) {
    double* part = (double*)ws;
    short* X[2];
    X[0] = (short*)(ws + ((d.norm + 255) & ~(size_t)255));
    X[1] = X[0] + (size_t)d.batch * d.x_elems;
    short* A = X[1] + (size_t)d.batch * d.x_elems;
    short* B = A + (size_t)d.batch * d.a_elems;
    float* slab = (float*)(B + (size_t)d.batch * d.a_elems);
    double sigma = 1.0;                           // bound of the iterate's singular values
    int sx = exponent_for(sigma);
    int vec = d.cols % 4 == 0;                    // every row of every matrix starts on four elements
    for (int z = 0; z < nz && vec; ++z) {
        const Item& it = b.it[z];
        vec = it.lds % 4 == 0 && reinterpret_cast<uintptr_t>(it.src) % (dtype == CAPDEC_F32 ? 16 : 8) == 0 &&
              (!mo.on || (it.ldm % 4 == 0 && capdec_aligned16(it.mom)));
    }
    const int64_t chunks = (int64_t)d.rows * ((d.cols + CHUNK - 1) / CHUNK);
    const int nparts = (int)(chunks < 4 * NORM_BLOCKS ? (chunks + 3) / 4 : NORM_BLOCKS);
    norm_kernel<<<dim3(nparts, nz), 256, 0, s>>>(b, d.rows, d.cols, dtype, mo, vec, part);
    const int64_t items = (int64_t)d.rp * (d.cp / 8);
    const unsigned blocks = (unsigned)(items / 256 + 1 < 1024 ? items / 256 + 1 : 1024);
    normalise_kernel<<<dim3(blocks, nz), 256, 0, s>>>(b, d.rows, d.cols, d.rp, d.cp, dtype, mo, vec, part, nparts, n.eps,
                                                      ldexpf(1.f, sx), X[0], (int64_t)d.x_elems);
    CAPDEC_LAUNCH_CHECK();
    for (int k = 0; k < n.steps; ++k) {
        const double lambda = sigma * sigma;
        const int sa = exponent_for(lambda), sb = exponent_for(top_of_poly(n.b, n.c, lambda));
        const int64_t ldx = (int64_t)d.cp * 2, lda = (int64_t)d.m * 2;
        StepArgs g{};
        g.strideP = g.strideQ = (int64_t)d.x_elems;
        g.P = g.Q = View{X[k & 1], ldx, d.m, d.rp};
        g.alpha = ldexpf(1.f, sa - 2 * sx);
        g.I = g.J = d.m; g.kt = (d.tall ? d.rp : d.cp) / 16;
        g.out = A; g.ldo = lda; g.strideO = (int64_t)d.a_elems;
        if (d.tall) CAPDEC_TRY(launch_symmetric<true>(g, nz, slab, s));
        else CAPDEC_TRY(launch_symmetric<false>(g, nz, slab, s));

        g.strideP = g.strideQ = g.strideR = (int64_t)d.a_elems;
        g.P = g.Q = View{A, lda, d.m, d.m};
        g.R = A; g.ldr = lda;
        g.alpha = (float)ldexp((double)n.c, sb - 2 * sa);
        g.beta = (float)ldexp((double)n.b, sb - sa);
        g.kt = d.m / 16;
        g.out = B;
        CAPDEC_TRY(launch_symmetric<false>(g, nz, slab, s));

        const bool end = k + 1 == n.steps;
        const double next = top_of_step(n.a, n.b, n.c, sigma);
        const int sn = end ? 0 : exponent_for(next);
        StepArgs h = end ? last : StepArgs{};
        h.b = b;
        const View vx{X[k & 1], ldx, d.cp, d.rp}, vb{B, lda, d.m, d.m};
        h.alpha = ldexpf(1.f, sn - sb - sx);
        h.beta = (float)ldexp((double)n.a, sn - sx);
        h.R = X[k & 1]; h.ldr = ldx; h.strideR = (int64_t)d.x_elems;
        h.I = end ? d.rows : d.rp;
        h.J = end ? d.cols : d.cp;
        h.kt = d.m / 16;
        h.out = X[~k & 1]; h.ldo = ldx; h.strideO = (int64_t)d.x_elems;
        if (d.tall) {
            h.P = View{X[k & 1], ldx, d.rp, d.rp}; h.strideP = (int64_t)d.x_elems;
            h.Q = vb; h.strideQ = (int64_t)d.a_elems;
            if (!end) CAPDEC_TRY((launch_sized<false, false, INNER>(h, nz, s)));
            else if (mo.on) CAPDEC_TRY((launch_sized<false, false, UPDATE>(h, nz, s)));
            else CAPDEC_TRY((launch_sized<false, false, RESULT>(h, nz, s)));
        } else {
            h.P = vb; h.strideP = (int64_t)d.a_elems;
            h.Q = vx; h.strideQ = (int64_t)d.x_elems;
            if (!end) CAPDEC_TRY((launch_sized<false, true, INNER>(h, nz, s)));
            else if (mo.on) CAPDEC_TRY((launch_sized<false, true, UPDATE>(h, nz, s)));
            else CAPDEC_TRY((launch_sized<false, true, RESULT>(h, nz, s)));
        }
        sigma = next;
        sx = sn;
    }
    return 0;
}

// the iterate's bound must leave the powers of two in fp32's and fp16's range
bool iteration_fits(const float* coeffs, int steps) {
    if (!coeffs || steps < 1 || steps > 32) return false;
    double sigma = 1.0;
    for (int k = 0; k < 3; ++k)
        if (!(fabs((double)coeffs[k]) <= 1e3)) return false;
    for (int k = 0; k < steps; ++k) {
        sigma = top_of_step(coeffs[0], coeffs[1], coeffs[2], sigma);
        if (!(sigma <= 64.0)) return false;
    }
    return true;
}

}  // namespace

extern "C" {

size_t capdec_orthogonalize_workspace_bytes(int count, int rows, int cols) {
    Dims d;
    if (!make_dims(count, rows, cols, d)) return 0;
    return ((d.norm + 255) & ~(size_t)255) + d.per * d.batch + d.slab;
}

int capdec_orthogonalize(const capdec_matrix* mats, int count, int rows, int cols, int dtype, int steps, const float* coeffs,
                         float eps, void* workspace, size_t workspace_bytes, void* stream) {
    Dims d;
    CAPDEC_REQUIRE(mats && make_dims(count, rows, cols, d) && dtype >= 0 && dtype <= 2 && iteration_fits(coeffs, steps));
    CAPDEC_REQUIRE(workspace && eps >= 0.f);
    for (int k = 0; k < count; ++k)
        CAPDEC_REQUIRE(mats[k].src && mats[k].dst && (rows == 1 || (mats[k].ld_src >= cols && mats[k].ld_dst >= cols)));
    if (!capdec_aligned16(workspace)) return CAPDEC_EALIGN;
    if (workspace_bytes < capdec_orthogonalize_workspace_bytes(count, rows, cols)) return CAPDEC_ENOMEM;
    const Iteration n{steps, coeffs[0], coeffs[1], coeffs[2], eps};
    for (int k = 0; k < count; k += d.batch) {
        const int nz = count - k < d.batch ? count - k : d.batch;
        Batch b{};
        for (int e = 0; e < nz; ++e)
            b.it[e] = Item{mats[k + e].src, mats[k + e].dst, nullptr, mats[k + e].ld_src, mats[k + e].ld_dst, 0};
        StepArgs last{};
        last.dtype = dtype;
        CAPDEC_TRY(run_batch(b, nz, d, n, dtype, Momentum{}, (char*)workspace, last, (hipStream_t)stream));
    }
    return 0;
}

int capdec_muon_step(const capdec_muon_param* params, int count, int rows, int cols, float lr, const capdec_train_state* st,
                     float momentum, int nesterov, float weight_decay, float update_scale, float grad_scale, int steps,
                     const float* coeffs, float eps, void* workspace, size_t workspace_bytes, void* stream) {
    Dims d;
    CAPDEC_REQUIRE(params && make_dims(count, rows, cols, d) && iteration_fits(coeffs, steps));
    CAPDEC_REQUIRE(workspace && eps >= 0.f);
    for (int k = 0; k < count; ++k) {
        const capdec_muon_param& q = params[k];
        CAPDEC_REQUIRE(q.p && q.g && q.m && (rows == 1 || (q.ldp >= cols && q.ldg >= cols && q.ldm >= cols)));
    }
    if (!capdec_aligned16(workspace)) return CAPDEC_EALIGN;
    if (workspace_bytes < capdec_orthogonalize_workspace_bytes(count, rows, cols)) return CAPDEC_ENOMEM;
    const Iteration n{steps, coeffs[0], coeffs[1], coeffs[2], eps};
    const Momentum mo{1, nesterov, momentum, grad_scale};
    for (int k = 0; k < count; k += d.batch) {
        const int nz = count - k < d.batch ? count - k : d.batch;
        Batch b{};
        for (int e = 0; e < nz; ++e) {
            const capdec_muon_param& q = params[k + e];
            b.it[e] = Item{q.g, q.p, q.m, q.ldg, q.ldp, q.ldm};
        }
        StepArgs last{};
        last.lr = lr; last.st = st; last.decay = weight_decay; last.scale = update_scale;
        CAPDEC_TRY(run_batch(b, nz, d, n, CAPDEC_F32, mo, (char*)workspace, last, (hipStream_t)stream));
    }
    return 0;
}

}  // extern "C"
