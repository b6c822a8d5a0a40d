// Orthogonalised matrix updates: Newton-Schulz iterations on lists of matrices, and the optimiser step built on them.
//
//   u  = x                                            (orthogonalize)
//   m <- mu m + (1 - mu) s g,  u = (1 - mu) s g + mu m or m    (optimiser step; s scales the gradient)
//   X  = u / (|u|_F + eps), transposed if it has more rows than columns: m x n with m <= n
//   `steps` times:  A = X X^T,  B = b A + c A A,  X <- a X + B X
//   out = X                                           p <- (1 - lr wd) p - lr k X
//
// Arithmetic.  The three products of a step are all the work: 4 m^2 n + 2 m^3 flops, for which float32 MFMA has 1/16 of
// the float16 rate.  Each operand is therefore held as two float16 numbers, v S = hi + lo with hi = f16(v S) and
// lo = f16(v S - hi): 22 bits and the sign of lo, a representation error of 2^-24 as float32's own.  A product is
// hi hi + hi lo + lo hi, exact in each term and summed in float32 (the dropped lo lo is below 2^-24 of the product):
// three float16 MFMAs for one of float32, 16 / 3 of its rate at float32's accuracy.  S is a power of two that keeps
// hi below 2^15 for the largest singular value the coefficients can reach (the caller's interval bound), so nothing
// overflows, and a value's lo part leaves float16's normal range only 2^-13 below the largest.  A matrix whose norm is
// far below eps starts far below 1: its S is larger by the power of two that all steps together cannot grow back
// (ns_scale; A needs none, it only corrects a X there).  a X is added to the
// sum in float32, not folded into B: folded, the large term makes every partial sum of the product round at its size
// (2 to 3 times the float32 error).
//
// Layout.  X is kept as hi / lo planes [mp][np] and transposed [np][mp], A and B as [mp][mp], all padded with zeros to
// the tile, so that every product is one of rows with rows (K contiguous on both sides) and no tile checks bounds.
// A and B are symmetric: only tiles on and above the diagonal are computed, and written twice.
#include <math.h>

#include <algorithm>

#include "kernels.h"

namespace pcx {
namespace {

typedef __bf16 bf16;
typedef _Float16 f16;
typedef f16 f16x4 __attribute__((ext_vector_type(4)));
typedef f16 f16x8 __attribute__((ext_vector_type(8)));

constexpr int NS_LIST = 24;      // entries per launch (their table is a kernel argument)
constexpr int NS_TILE = 64;      // rows and columns of a tile; X, A, B are padded to it
constexpr int NS_K = 32;         // K values staged at a time

struct NsMat {
    const void* x;               // orthogonalize: the matrices; step: gradients
    void* out;                   // orthogonalize: the result; step: parameters
    float* mom;                  // step: momentum
    int64_t xb, xr, xc;          // strides of x in elements: matrix, row, column
    int rows, cols, batch;
    int m, n, mp, np;            // short and long side, and padded
    float step;                  // step: lr k
    int64_t ws;                  // byte offset of the entry's planes in the workspace
    int norm;                    // first of its partial sums of squares
};

struct NsTable {
    NsMat e[NS_LIST];
    int first[NS_LIST + 1];      // blocks of the launch up to each entry
    int count, mats;
};

struct NsArgs {
    char* ws;
    double* part;                // [.] partial sums of squares, NS_PART per matrix
    int dtype;                   // orthogonalize: type of x and out
    int is_step, nesterov;
    float mu, gs, decay;         // momentum, gradient scale, 1 - lr wd
    float eps;
    float sx, sa;                // S of X (of a matrix that starts near 1) and of A, B
    double growth;               // most that all steps together enlarge a small singular value
    float* unit;                 // [matrices] 1 / S of X
    float a, b, c;               // this step's coefficients
    int src;                     // which X buffer the step reads
};

constexpr int NS_PART = 64;      // partial sums per matrix

// planes of one matrix, in float16 numbers from its workspace: X hi, lo, X^T hi, lo (two buffers), A hi, lo, B hi, lo
struct Planes {
    f16* base;
    int64_t mn, mm;
    __device__ f16* x(int buf, int lo) const { return base + (4 * buf + lo) * mn; }
    __device__ f16* xt(int buf, int lo) const { return base + (4 * buf + 2 + lo) * mn; }
    __device__ f16* a(int lo) const { return base + 8 * mn + lo * mm; }
    __device__ f16* b(int lo) const { return base + 8 * mn + (2 + lo) * mm; }
};
__host__ __device__ inline int64_t plane_bytes(int mp, int np) {
    return 2 * (8 * (int64_t)mp * np + 4 * (int64_t)mp * mp);
}
__device__ __forceinline__ Planes planes_of(const NsArgs& q, const NsMat& e, int bat) {
    Planes p;
    p.mn = (int64_t)e.mp * e.np;
    p.mm = (int64_t)e.mp * e.mp;
    p.base = reinterpret_cast<f16*>(q.ws + e.ws + bat * plane_bytes(e.mp, e.np));
    return p;
}

__device__ __forceinline__ int find_entry(const NsTable& t, int blk) {
    int i = 0;
    while (i + 1 < t.count && blk >= t.first[i + 1]) ++i;
    return i;
}

__device__ __forceinline__ float load_any(const void* p, int64_t i, int dtype) {
    if (dtype == PCX_F32) return static_cast<const float*>(p)[i];
    if (dtype == PCX_BF16) return (float)static_cast<const bf16*>(p)[i];
    return (float)static_cast<const f16*>(p)[i];
}
__device__ __forceinline__ void split(float v, f16& hi, f16& lo) {
    hi = (f16)v;
    lo = (f16)(v - (float)hi);
}

// the momentum update of one element -> u (the same operations in both passes that need u)
__device__ __forceinline__ float nesterov_u(const NsArgs& q, float g, float m) {
    return q.nesterov ? fmaf(1.f - q.mu, g * q.gs, q.mu * m) : m;
}

// ---------------------------------------------------------------- u, and the sums of its squares (in float64: no range)
__global__ __launch_bounds__(256) void ns_norm_kernel(NsTable t, NsArgs q) {
    __shared__ double red[4];
    const int ei = find_entry(t, blockIdx.x);
    const NsMat& e = t.e[ei];
    const int bat = (blockIdx.x - t.first[ei]) / NS_PART, blk = (blockIdx.x - t.first[ei]) % NS_PART;
    const int64_t n = (int64_t)e.rows * e.cols;
    const int64_t per = (n + NS_PART - 1) / NS_PART, i0 = blk * per, i1 = i0 + per < n ? i0 + per : n;
    double s = 0.;
    if (q.is_step) {
        const float* g = static_cast<const float*>(e.x);
        for (int64_t i = i0 + threadIdx.x; i < i1; i += 256) {
            const float gv = g[i], mv = fmaf(1.f - q.mu, gv * q.gs, q.mu * e.mom[i]);
            e.mom[i] = mv;
            const float u = nesterov_u(q, gv, mv);
            s += (double)u * u;
        }
    } else {
        for (int64_t i = i0 + threadIdx.x; i < i1; i += 256) {
            const int64_t r = i / e.cols, c = i - r * e.cols;
            const float u = load_any(e.x, bat * e.xb + r * e.xr + c * e.xc, q.dtype);
            s += (double)u * u;
        }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) q.part[(int64_t)(e.norm + bat) * NS_PART + blk] = (red[0] + red[1]) + (red[2] + red[3]);
}

// exponent of the power of two above sx: 0 unless |X|_F times the growth of all steps stays below 1
__device__ __forceinline__ int ns_scale(double fro, double growth) {
    const double far = 1. / (fro * growth);
    if (!(far >= 2.)) return 0;  // (NaN too)
    return far > 1e27 ? 90 : ilogb(far);
}

// ---------------------------------------------------------------- X = u S / (|u| + eps) as planes, both ways round
__global__ __launch_bounds__(256) void ns_split_kernel(NsTable t, NsArgs q) {
    __shared__ float tile[64][65];
    __shared__ double scale_s;
    const int ei = find_entry(t, blockIdx.x);
    const NsMat& e = t.e[ei];
    const int tm = e.mp / 64, tn = e.np / 64, per = tm * tn;
    const int rel = blockIdx.x - t.first[ei], bat = rel / per, tl = rel % per;
    const int i0 = (tl / tn) * 64, j0 = (tl % tn) * 64;  // of X (m x n)
    const Planes P = planes_of(q, e, bat);
    if (threadIdx.x < 64) {
        double s = q.part[(int64_t)(e.norm + bat) * NS_PART + threadIdx.x];
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
        if (threadIdx.x == 0) {
            const double norm = sqrt(s), inv = 1. / (norm + (double)q.eps);
            const int k = ns_scale(norm * inv, q.growth);
            scale_s = ldexp(q.sx * inv, k);
            if (tl == 0) q.unit[e.norm + bat] = ldexpf(1.f / q.sx, -k);
        }
    }
    __syncthreads();
    const double scale = scale_s;
    const bool tall = e.rows > e.cols;
    // read with the source's columns across the threads
    for (int k = threadIdx.x; k < 64 * 64; k += 256) {
        const int sr = k >> 6, sc = k & 63;
        const int r = (tall ? j0 : i0) + sr, c = (tall ? i0 : j0) + sc;
        float v = 0.f;
        if (r < e.rows && c < e.cols) {
            if (q.is_step) {
                const int64_t i = (int64_t)r * e.cols + c;
                v = nesterov_u(q, static_cast<const float*>(e.x)[i], e.mom[i]);
            } else {
                v = load_any(e.x, bat * e.xb + r * e.xr + c * e.xc, q.dtype);
            }
        }
        tile[tall ? sc : sr][tall ? sr : sc] = (float)(v * scale);
    }
    __syncthreads();
    for (int k = threadIdx.x; k < 64 * 16; k += 256) {
        const int r = k >> 4, c = (k & 15) * 4;
        f16x4 h, l, ht, lt;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            f16 a, b;
            split(tile[r][c + j], a, b);
            h[j] = a;
            l[j] = b;
            split(tile[c + j][r], a, b);
            ht[j] = a;
            lt[j] = b;
        }
        const int64_t o = (int64_t)(i0 + r) * e.np + j0 + c, ot = (int64_t)(j0 + r) * e.mp + i0 + c;
        *reinterpret_cast<f16x4*>(P.x(0, 0) + o) = h;
        *reinterpret_cast<f16x4*>(P.x(0, 1) + o) = l;
        *reinterpret_cast<f16x4*>(P.xt(0, 0) + ot) = ht;
        *reinterpret_cast<f16x4*>(P.xt(0, 1) + ot) = lt;
    }
}

// ---------------------------------------------------------------- the products
// 64 x 64 tile of C[r][c] = sum_k P[r][k] Q[c][k], four waves of 32 x 32 each; P, Q: hi / lo planes with row length ld.
// On return lane l of wave w holds rows r = 32 (w & 1) + acc_row(i, l >> 5), column c = 32 (w >> 1) + (l & 31) of the
// tile, so four consecutive i are four consecutive rows of one column.
struct Operand {
    const f16* hi;
    const f16* lo;
    int64_t ld;
};

__device__ __forceinline__ f32x16 mfma16(f16x8 a, f16x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

__device__ __forceinline__ void tile_product(const Operand& P, const Operand& Q, int K, f16* sm, f32x16& acc) {
    constexpr int RS = NS_K + 8;  // padded row (16-byte aligned)
    f16* sp[2] = {sm, sm + 64 * RS};
    f16* sq[2] = {sm + 2 * 64 * RS, sm + 3 * 64 * RS};
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int row = tid >> 2, kc = (tid & 3) * 8;
    const int wr = (wave & 1) * 32 + (lane & 31), wc = (wave >> 1) * 32 + (lane & 31), kh = (lane >> 5) * 8;
    for (int k0 = 0; k0 < K; k0 += NS_K) {
        const f16x8 p0 = *reinterpret_cast<const f16x8*>(P.hi + row * P.ld + k0 + kc);
        const f16x8 p1 = *reinterpret_cast<const f16x8*>(P.lo + row * P.ld + k0 + kc);
        const f16x8 q0 = *reinterpret_cast<const f16x8*>(Q.hi + row * Q.ld + k0 + kc);
        const f16x8 q1 = *reinterpret_cast<const f16x8*>(Q.lo + row * Q.ld + k0 + kc);
        __syncthreads();
        *reinterpret_cast<f16x8*>(sp[0] + row * RS + kc) = p0;
        *reinterpret_cast<f16x8*>(sp[1] + row * RS + kc) = p1;
        *reinterpret_cast<f16x8*>(sq[0] + row * RS + kc) = q0;
        *reinterpret_cast<f16x8*>(sq[1] + row * RS + kc) = q1;
        __syncthreads();
#pragma unroll
        for (int k = 0; k < NS_K; k += 16) {
            const f16x8 ph = *reinterpret_cast<const f16x8*>(sp[0] + wr * RS + k + kh);
            const f16x8 pl = *reinterpret_cast<const f16x8*>(sp[1] + wr * RS + k + kh);
            const f16x8 qh = *reinterpret_cast<const f16x8*>(sq[0] + wc * RS + k + kh);
            const f16x8 ql = *reinterpret_cast<const f16x8*>(sq[1] + wc * RS + k + kh);
            acc = mfma16(ph, ql, acc);
            acc = mfma16(pl, qh, acc);
            acc = mfma16(ph, qh, acc);
        }
    }
}

// C[c][r .. r+3] and, transposed, C[r .. r+3][c] of four values
__device__ __forceinline__ void store_planes(f16* hi, f16* lo, int64_t ld, int r, int c, const f16x4& h, const f16x4& l) {
    *reinterpret_cast<f16x4*>(hi + c * ld + r) = h;
    *reinterpret_cast<f16x4*>(lo + c * ld + r) = l;
}
__device__ __forceinline__ void store_planes_t(f16* hi, f16* lo, int64_t ld, int r, int c, const f16x4& h, const f16x4& l) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        hi[(r + j) * ld + c] = h[j];
        lo[(r + j) * ld + c] = l[j];
    }
}

// PHASE 0: A = X X^T.  1: B = b A + c A A.  Tiles (ti <= tj), the mirrored one written too.
template <int PHASE> __global__ __launch_bounds__(256) void ns_sym_kernel(NsTable t, NsArgs q) {
    __shared__ __attribute__((aligned(16))) f16 sm[4 * 64 * (NS_K + 8)];
    const int ei = find_entry(t, blockIdx.x);
    const NsMat& e = t.e[ei];
    const int tm = e.mp / 64, per = tm * (tm + 1) / 2;
    const int rel = blockIdx.x - t.first[ei], bat = rel / per;
    int tj = 0, tl = rel % per;
    while (tl > tj) tl -= ++tj;  // column tj holds tiles 0 .. tj
    const int i0 = tl * 64, j0 = tj * 64;
    const Planes p = planes_of(q, e, bat);
    f32x16 acc{};
    if (PHASE == 0) {
        const Operand P{p.x(q.src, 0) + (int64_t)i0 * e.np, p.x(q.src, 1) + (int64_t)i0 * e.np, e.np};
        const Operand Q{p.x(q.src, 0) + (int64_t)j0 * e.np, p.x(q.src, 1) + (int64_t)j0 * e.np, e.np};
        tile_product(P, Q, e.np, sm, acc);
    } else {
        const Operand P{p.a(0) + (int64_t)i0 * e.mp, p.a(1) + (int64_t)i0 * e.mp, e.mp};
        const Operand Q{p.a(0) + (int64_t)j0 * e.mp, p.a(1) + (int64_t)j0 * e.mp, e.mp};
        tile_product(P, Q, e.mp, sm, acc);
    }
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int c = j0 + (wave >> 1) * 32 + (lane & 31);
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        const int r = i0 + (wave & 1) * 32 + acc_row(4 * g, lane >> 5);
        f16x4 h, l;
        if (PHASE == 0) {
            const float unit = q.unit[e.norm + bat], k = q.sa * unit * unit;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                f16 a, b;
                split(acc[4 * g + j] * k, a, b);
                h[j] = a;
                l[j] = b;
            }
            store_planes(p.a(0), p.a(1), e.mp, r, c, h, l);
            if (i0 != j0) store_planes_t(p.a(0), p.a(1), e.mp, r, c, h, l);
        } else {
            const f16x4 ah = *reinterpret_cast<const f16x4*>(p.a(0) + (int64_t)c * e.mp + r);
            const f16x4 al = *reinterpret_cast<const f16x4*>(p.a(1) + (int64_t)c * e.mp + r);
            const float k = q.c / q.sa;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                f16 a, b;
                split(fmaf(q.b, (float)ah[j] + (float)al[j], acc[4 * g + j] * k), a, b);
                h[j] = a;
                l[j] = b;
            }
            store_planes(p.b(0), p.b(1), e.mp, r, c, h, l);
            if (i0 != j0) store_planes_t(p.b(0), p.b(1), e.mp, r, c, h, l);
        }
    }
}

// X <- a X + B X, as planes both ways round; LAST: to the caller's matrices instead
template <bool LAST> __global__ __launch_bounds__(256) void ns_apply_kernel(NsTable t, NsArgs q) {
    __shared__ __attribute__((aligned(16))) f16 sm[4 * 64 * (NS_K + 8)];
    const int ei = find_entry(t, blockIdx.x);
    const NsMat& e = t.e[ei];
    const int tm = e.mp / 64, tn = e.np / 64, per = tm * tn;
    const int rel = blockIdx.x - t.first[ei], bat = rel / per, tl = rel % per;
    const int i0 = (tl / tn) * 64, j0 = (tl % tn) * 64;
    const Planes p = planes_of(q, e, bat);
    const Operand B{p.b(0) + (int64_t)i0 * e.mp, p.b(1) + (int64_t)i0 * e.mp, e.mp};
    const Operand X{p.xt(q.src, 0) + (int64_t)j0 * e.mp, p.xt(q.src, 1) + (int64_t)j0 * e.mp, e.mp};
    // the accumulator's rows (four adjacent per lane) run along the output's rows in memory
    const bool tall = LAST && e.rows > e.cols;
    f32x16 acc{};
    if (tall) tile_product(B, X, e.mp, sm, acc);
    else tile_product(X, B, e.mp, sm, acc);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int c = (tall ? j0 : i0) + (wave >> 1) * 32 + (lane & 31);
    const float k = 1.f / q.sa;
    const f16* xh = tall ? p.xt(q.src, 0) : p.x(q.src, 0);
    const f16* xl = tall ? p.xt(q.src, 1) : p.x(q.src, 1);
    const int64_t ld = tall ? e.mp : e.np;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        const int r = (tall ? i0 : j0) + (wave & 1) * 32 + acc_row(4 * g, lane >> 5);
        const f16x4 oh = *reinterpret_cast<const f16x4*>(xh + c * ld + r);
        const f16x4 ol = *reinterpret_cast<const f16x4*>(xl + c * ld + r);
        float v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = fmaf(q.a, (float)oh[j] + (float)ol[j], acc[4 * g + j] * k);
        if (!LAST) {
            f16x4 h, l;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                f16 a, b;
                split(v[j], a, b);
                h[j] = a;
                l[j] = b;
            }
            store_planes(p.x(1 - q.src, 0), p.x(1 - q.src, 1), e.np, r, c, h, l);
            store_planes_t(p.xt(1 - q.src, 0), p.xt(1 - q.src, 1), e.mp, r, c, h, l);
        } else {
            const float u = q.unit[e.norm + bat];
            if (c >= e.rows) continue;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (r + j >= e.cols) continue;
                const int64_t o = (int64_t)c * e.cols + r + j;
                if (q.is_step) {
                    float* w = static_cast<float*>(e.out);
                    w[o] = fmaf(q.decay, w[o], -e.step * (v[j] * u));
                } else {
                    const int64_t ob = (int64_t)bat * e.rows * e.cols + o;
                    if (q.dtype == PCX_F32) static_cast<float*>(e.out)[ob] = v[j] * u;
                    else if (q.dtype == PCX_BF16) static_cast<bf16*>(e.out)[ob] = (bf16)(v[j] * u);
                    else static_cast<f16*>(e.out)[ob] = (f16)(v[j] * u);
                }
            }
        }
    }
}

// ---------------------------------------------------------------- host
int round_up(int v, int k) { return (v + k - 1) / k * k; }

void set_shape(NsMat& e, int64_t rows, int64_t cols) {
    e.rows = (int)rows;
    e.cols = (int)cols;
    e.m = (int)std::min(rows, cols);
    e.n = (int)std::max(rows, cols);
    e.mp = round_up(e.m, NS_TILE);
    e.np = round_up(e.n, NS_TILE);
}

// largest singular value any step can leave, starting in [0, 1], and the largest of |b s^2 + c s^4| on the way: by
// dense sampling of the interval each step maps into (the polynomials are smooth: 1 % covers the gaps)
void ns_bounds(const float* coef, int steps, double* smax, double* bmax, double* growth) {
    double hi = 1.0;
    *smax = 1.0;
    *bmax = 0.0;
    *growth = 1.0;
    for (int k = 0; k < steps; ++k) {
        const double a = coef[3 * k], b = coef[3 * k + 1], c = coef[3 * k + 2];
        double next = 0.0, grow = 1.0;
        for (int i = 0; i <= 4096; ++i) {
            const double s = hi * i / 4096, l = s * s, bb = b * l + c * l * l;
            next = std::max(next, fabs(s * (a + bb)));
            grow = std::max(grow, 1.01 * fabs(a + bb));
            *bmax = std::max(*bmax, std::max(fabs(bb), l));
        }
        hi = next * 1.01;
        *growth *= grow;
        *smax = std::max(*smax, hi);
        if (!(hi < 1e6)) break;
    }
}

// One launch table's workspace: the partial sums and the unit of every matrix, then the planes, 256-byte aligned.
int64_t ns_place(NsTable& t) {
    int64_t mats = 0;
    for (int i = 0; i < t.count; ++i) {
        t.e[i].norm = (int)mats;
        mats += t.e[i].batch;
    }
    t.mats = (int)mats;
    int64_t off = mats * (NS_PART * (int64_t)sizeof(double) + (int64_t)sizeof(float));
    for (int i = 0; i < t.count; ++i) {
        off = (off + 255) / 256 * 256;
        t.e[i].ws = off;
        off += t.e[i].batch * plane_bytes(t.e[i].mp, t.e[i].np);
    }
    return off;
}

int ns_scales(NsArgs& q, const float* coef, int steps) {
    double smax, bmax;
    ns_bounds(coef, steps, &smax, &bmax, &q.growth);
    PCX_CHECK_ARG(smax <= 8.0 && bmax <= 64.0,
                  "orthogonalize: the coefficients take singular values in [0, 1] to %g (8 at most)", smax);
    q.sx = (float)exp2(floor(log2(32768.0 / smax)));
    q.sa = (float)exp2(floor(log2(32768.0 / std::max(1.0, bmax))));
    return PCX_OK;
}

int ns_run(NsTable& t, NsArgs q, const float* coef, int steps, hipStream_t s) {
    q.unit = reinterpret_cast<float*>(q.part + (int64_t)t.mats * NS_PART);
    auto blocks = [&](auto per) {
        int64_t n = 0;
        for (int i = 0; i < t.count; ++i) {
            t.first[i] = (int)n;
            n += per(t.e[i]) * t.e[i].batch;
        }
        t.first[t.count] = (int)n;
        return (unsigned)n;
    };
    const auto full = [](const NsMat& e) { return (int64_t)(e.mp / 64) * (e.np / 64); };
    const auto half = [](const NsMat& e) { return (int64_t)(e.mp / 64) * (e.mp / 64 + 1) / 2; };
    unsigned n = blocks([](const NsMat&) { return (int64_t)NS_PART; });
    ns_norm_kernel<<<n, 256, 0, s>>>(t, q);
    PCX_LAUNCH_CHECK("ns_norm_kernel");
    n = blocks(full);
    ns_split_kernel<<<n, 256, 0, s>>>(t, q);
    PCX_LAUNCH_CHECK("ns_split_kernel");
    for (int k = 0; k < steps; ++k) {
        q.a = coef[3 * k];
        q.b = coef[3 * k + 1];
        q.c = coef[3 * k + 2];
        q.src = k & 1;
        n = blocks(half);
        ns_sym_kernel<0><<<n, 256, 0, s>>>(t, q);
        PCX_LAUNCH_CHECK("ns_sym_kernel");
        ns_sym_kernel<1><<<n, 256, 0, s>>>(t, q);
        PCX_LAUNCH_CHECK("ns_sym_kernel");
        n = blocks(full);
        if (k + 1 < steps) ns_apply_kernel<false><<<n, 256, 0, s>>>(t, q);
        else ns_apply_kernel<true><<<n, 256, 0, s>>>(t, q);
        PCX_LAUNCH_CHECK("ns_apply_kernel");
    }
    return PCX_OK;
}

// Adam (coupled decay, as pcx_adam_step) on a list of segments of flat buffers
constexpr int SEG_LIST = 64;
struct SegTable {
    pcx_segment e[SEG_LIST];
    int first[SEG_LIST + 1];
    int count;
};
__global__ __launch_bounds__(256) void adam_segments_kernel(float* __restrict__ p, const float* __restrict__ g,
                                                            float* __restrict__ m, float* __restrict__ v, SegTable t,
                                                            float lr_bc1, float b1, float b2, float inv_sqrt_bc2,
                                                            float eps, float wd, float gs) {
    int i = 0;
    while (i + 1 < t.count && (int)blockIdx.x >= t.first[i + 1]) ++i;
    const int64_t k = (int64_t)(blockIdx.x - t.first[i]) * 256 + threadIdx.x;
    if (k >= t.e[i].n) return;
    const int64_t o = t.e[i].offset + k, ov = t.e[i].v_offset + k;
    const float gg = g[o] * gs + wd * p[o];
    const float mm = b1 * m[o] + (1.f - b1) * gg, vv = b2 * v[ov] + (1.f - b2) * gg * gg;
    m[o] = mm;
    v[ov] = vv;
    p[o] -= lr_bc1 * mm / (sqrtf(vv) * inv_sqrt_bc2 + eps);
}

bool ns_shape_ok(int64_t batch, int64_t rows, int64_t cols) {
    // tile and block counts stay in 32 bits
    if (batch < 0 || rows < 1 || cols < 1 || std::max(rows, cols) > 1 << 20 || std::min(rows, cols) > 1 << 14) return false;
    const int64_t tiles = ((rows + 63) / 64) * ((cols + 63) / 64) + NS_PART;
    return rows * cols <= (int64_t)1 << 31 && batch < (int64_t)1 << 24 && batch * tiles < (int64_t)1 << 30;
}

int ns_check(const char* what, int steps, const float* coef, float eps) {
    PCX_CHECK_ARG(steps >= 1 && steps <= 64, "%s: 1 to 64 steps (got %d)", what, steps);
    PCX_CHECK_ARG(coef, "%s: no coefficients", what);
    for (int i = 0; i < 3 * steps; ++i) PCX_CHECK_ARG(isfinite(coef[i]), "%s: coefficient %d is not finite", what, i);
    PCX_CHECK_ARG(eps > 0.f && isfinite(eps), "%s: eps must be positive (got %g)", what, (double)eps);
    return PCX_OK;
}

void ns_single(NsTable& t, int64_t batch, int64_t rows, int64_t cols) {
    t.count = 1;
    set_shape(t.e[0], rows, cols);
    t.e[0].batch = (int)batch;
}

// the matrices [at, at + NS_LIST) of a step's list; one workspace serves the launches of every such part in turn
int muon_part(const pcx_muon_matrix* mats, int n, int at, NsTable& t) {
    t.count = std::min(NS_LIST, n - at);
    for (int i = 0; i < t.count; ++i) {
        const pcx_muon_matrix& a = mats[at + i];
        PCX_CHECK_ARG(ns_shape_ok(1, a.rows, a.cols), "muon_step: a matrix of %lld x %lld is not supported",
                      (long long)a.rows, (long long)a.cols);
        NsMat& e = t.e[i];
        set_shape(e, a.rows, a.cols);
        e.batch = 1;
        e.x = a.grad;
        e.out = a.param;
        e.mom = a.momentum;
    }
    return PCX_OK;
}

}  // namespace
}  // namespace pcx

using namespace pcx;

extern "C" size_t pcx_orthogonalize_workspace_bytes(int64_t batch, int64_t rows, int64_t cols) {
    if (!ns_shape_ok(batch, rows, cols) || batch == 0) return 0;
    NsTable t{};
    ns_single(t, batch, rows, cols);
    return (size_t)ns_place(t);
}

extern "C" int pcx_orthogonalize(int dtype, int64_t batch, int64_t rows, int64_t cols, const void* x, int64_t batch_stride,
                                 int64_t row_stride, int64_t col_stride, void* out, int steps, const float* coef, float eps,
                                 void* ws, size_t ws_bytes, hipStream_t stream) {
    PCX_CHECK_ARG(dtype == PCX_F32 || dtype == PCX_BF16 || dtype == PCX_F16, "orthogonalize: unknown element type %d", dtype);
    int rc = ns_check("orthogonalize", steps, coef, eps);
    if (rc) return rc;
    PCX_CHECK_ARG(ns_shape_ok(batch, rows, cols), "orthogonalize: %lld matrices of %lld x %lld are not supported",
                  (long long)batch, (long long)rows, (long long)cols);
    NsArgs q{};
    rc = ns_scales(q, coef, steps);
    if (rc || batch == 0) return rc;
    PCX_CHECK_ARG(x && out, "orthogonalize: NULL buffer");
    NsTable t{};
    ns_single(t, batch, rows, cols);
    const int64_t need = ns_place(t);
    if (!ws || (int64_t)ws_bytes < need) {
        set_error("orthogonalize: workspace of %zu bytes, %lld needed", ws_bytes, (long long)need);
        return PCX_EWORKSPACE;
    }
    NsMat& e = t.e[0];
    e.x = x;
    e.xb = batch_stride;
    e.xr = row_stride;
    e.xc = col_stride;
    e.out = out;
    q.ws = static_cast<char*>(ws);
    q.part = static_cast<double*>(ws);
    q.dtype = dtype;
    q.eps = eps;
    return ns_run(t, q, coef, steps, stream);
}

extern "C" size_t pcx_muon_workspace_bytes(const pcx_muon_matrix* mats, int n) {
    if (n <= 0 || !mats) return 0;
    int64_t most = 0;
    for (int at = 0; at < n; at += NS_LIST) {
        NsTable t{};
        if (muon_part(mats, n, at, t) != PCX_OK) return 0;
        most = std::max(most, ns_place(t));
    }
    return (size_t)most;
}

extern "C" int pcx_muon_step(const pcx_muon_matrix* mats, int n, float lr, float momentum, int nesterov, float weight_decay,
                             float grad_scale, int steps, const float* coef, float eps, void* ws, size_t ws_bytes,
                             hipStream_t stream) {
    int rc = ns_check("muon_step", steps, coef, eps);
    if (rc) return rc;
    PCX_CHECK_ARG(n >= 0 && (mats || n == 0), "muon_step: no matrices");
    PCX_CHECK_ARG(momentum >= 0.f && momentum < 1.f, "muon_step: momentum must be in [0, 1) (got %g)", (double)momentum);
    NsArgs q{};
    rc = ns_scales(q, coef, steps);
    if (rc) return rc;
    for (int at = 0; at < n; at += NS_LIST) {  // every matrix is checked before the first launch
        NsTable t{};
        rc = muon_part(mats, n, at, t);
        if (rc) return rc;
        for (int i = 0; i < t.count; ++i)
            PCX_CHECK_ARG(t.e[i].x && t.e[i].out && t.e[i].mom, "muon_step: NULL buffer of matrix %d", at + i);
        const int64_t need = ns_place(t);
        if (!ws || (int64_t)ws_bytes < need) {
            set_error("muon_step: workspace of %zu bytes, %lld needed", ws_bytes, (long long)need);
            return PCX_EWORKSPACE;
        }
    }
    q.ws = static_cast<char*>(ws);
    q.part = static_cast<double*>(ws);
    q.is_step = 1;
    q.nesterov = nesterov != 0;
    q.mu = momentum;
    q.gs = grad_scale;
    q.decay = (float)(1.0 - (double)lr * (double)weight_decay);
    q.eps = eps;
    for (int at = 0; at < n; at += NS_LIST) {
        NsTable t{};
        rc = muon_part(mats, n, at, t);
        if (rc) return rc;
        ns_place(t);
        for (int i = 0; i < t.count; ++i) t.e[i].step = lr * mats[at + i].scale;
        rc = ns_run(t, q, coef, steps, stream);
        if (rc) return rc;
    }
    return PCX_OK;
}

extern "C" int pcx_adam_segments(float* p, const float* g, float* m, float* v, const pcx_segment* segs, int n, int64_t step,
                                 float lr, float beta1, float beta2, float eps, float weight_decay, float grad_scale,
                                 hipStream_t stream) {
    PCX_CHECK_ARG(n >= 0 && (segs || n == 0), "adam_segments: no segments");
    PCX_CHECK_ARG(n == 0 || (p && g && m && v), "adam_segments: NULL buffer");
    PCX_CHECK_ARG(step >= 1, "adam_segments: step must be >= 1");
    for (int i = 0; i < n; ++i)
        PCX_CHECK_ARG(segs[i].n >= 0 && segs[i].offset >= 0 && segs[i].v_offset >= 0 && segs[i].n < (int64_t)1 << 36,
                      "adam_segments: bad segment %d", i);
    const double bc1 = 1.0 - pow((double)beta1, (double)step), bc2 = 1.0 - pow((double)beta2, (double)step);
    for (int at = 0; at < n; at += SEG_LIST) {
        SegTable t{};
        t.count = std::min(SEG_LIST, n - at);
        int64_t blocks = 0;
        for (int i = 0; i < t.count; ++i) {
            t.e[i] = segs[at + i];
            t.first[i] = (int)blocks;
            blocks += (t.e[i].n + 255) / 256;
        }
        t.first[t.count] = (int)blocks;
        PCX_CHECK_ARG(blocks < (int64_t)1 << 31, "adam_segments: too many elements");
        if (blocks == 0) continue;
        adam_segments_kernel<<<(unsigned)blocks, 256, 0, stream>>>(p, g, m, v, t, (float)(lr / bc1), beta1, beta2,
                                                                  (float)(1.0 / sqrt(bc2)), eps, weight_decay, grad_scale);
        PCX_LAUNCH_CHECK("adam_segments_kernel");
    }
    return PCX_OK;
}
