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
// three float16 MFMAs for one of float32, 16 / 3 of its rate.  Long sums round more than that (errors of 0.5 to 0.8 of
// float32 arithmetic's from 40 rows on), short ones less (1.9 times its error at 1 x 50), so matrices of at most 32 rows are
// in float32: tile_step in one block, ns_long_kernel in many.  (In a list with others they go by the planes
// too, unless blocks hold the whole list: launches of their own would add 7 to its 17.)  S is a power of two that keeps
// hi below 2^15 for the largest singular value the coefficients can reach (the caller's interval bound), so nothing
// overflows, and a value's lo part leaves float16's normal range only 2^-13 below the largest.  A matrix whose norm is
// far below eps starts far below 1: its S is larger by the power of two that all steps together cannot grow back
// (ns_scale; A needs none, it only corrects a X there).  a X is added to the sum in float32, not folded into B: folded,
// the large term makes every partial sum of the product round at its size (2 to 3 times the float32 error).
//
// Layout.  X is kept as hi / lo planes and transposed, A and B once, all padded with zeros to 64, so that every product is
// one of rows with rows.  A plane is stored as [K / 8][rows][8]: 8 values of K, a lane's operand of an MFMA, lie together,
// and the lanes' rows behind each other, so every load of an operand is one run of memory, and copied to LDS as it lies it
// is read without conflicts.  (4096 x 4096 in bfloat16: 5160 us row by row, where the rows of a tile lie a power of two
// apart more often than not and queue at one L2 channel; 4836 us as [K / 32][rows][32], all else alike; that with its runs
// swizzled in LDS 4059 us at a later step, 3948 as it is now.)
// A and B are symmetric: only tiles on and below the diagonal are computed, and written twice.
//
// What bounds it.  Large matrices: the MFMA rate.  4096 x 4096 in bfloat16, five steps: 3.64 to 4.06 ms (one card and
// another), 0.51 to 0.57 PFLOP/s of the three products' definition and 1.02 to 1.12 executed (three terms, half of the
// tiles of A and B), where a float16 product of the library reaches 1.08 at that size.  Of a few hundred tiles: LDS, which
// feeds the MFMAs of 64 x 64 tiles at half their rate, the traffic from L2, and a launch's fixed parts (addresses, first
// stages, the epilogue's passes).  Small ones: those fixed parts, 5 to 8 us a launch of which 2 to 3 compute.
#include <limits.h>
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "kernels.h"

namespace pcx {
namespace {

typedef __bf16 bf16;
typedef _Float16 f16;
typedef f16 f16x4 __attribute__((ext_vector_type(4)));
typedef f16 f16x8 __attribute__((ext_vector_type(8)));

constexpr int NS_LIST = 16;      // entries per launch (their table is the first kernel's argument)
constexpr int NS_PAD = 64;       // X, A, B are padded to it; tiles that reach over the padding read their last rows again
constexpr int NS_K = 32;         // K values of a stage
constexpr int NS_STEPS = 64;     // most steps
constexpr int NS_PART = 512;     // most partial sums of squares per matrix
constexpr int NS_ROUND = 768;    // tiles up to here are on the card together, or nearly so

struct NsMat {
    const void* x;               // orthogonalize: the matrices; step: gradients
    void* out;                   // orthogonalize: the result; step: parameters
    float* mom;                  // step: momentum
    int64_t xb, xr, xc;          // strides of x in elements: matrix, row, column
    int rows, cols, batch;
    int mp, np;                  // short and long side, padded
    float step;                  // step: lr k
    int64_t ws;                  // byte offset of the entry's planes in the workspace
    int mat, parts;              // first of its matrices in the launch, partial sums of each
};

struct NsTable {
    NsMat e[NS_LIST];
    int count, mats;
};

// Work units of a launch up to each entry; behind the last, more than there are.
struct NsFirst {
    int first[NS_LIST];
    int count;
};
// Those of a product, per entry: its tiles in order, the first `whole` over all of K, the others in `split` parts each
// (joined by whichever unit of a tile ends last, in part order).
struct NsUnits : NsFirst {
    int tiles[NS_LIST];          // tiles of one matrix of the entry
    int whole[NS_LIST];          // of the entry's tiles times batch
    int split[NS_LIST];
    int tail[NS_LIST];           // first counter of the entry's split tiles
    int joint[NS_LIST];          // first of their parts' sums
};

struct NsCoef {
    int steps;
    float c[3 * NS_STEPS];
};

struct NsArgs {
    char* ws;
    double* part;                // [matrices][NS_PART] partial sums of squares
    float* unit;                 // [matrices] 1 / S of X
    unsigned* done;              // [split tiles] parts that have been written
    float* joint;                // [split tiles][parts][tile] their sums
    int ndone;
    int slices;                  // long matrices of one tile's rows: blocks of their launches
    int dtype;                   // orthogonalize: type of x and out
    int is_step, nesterov;
    float mu, gs, decay;         // momentum, gradient scale, 1 - lr wd
    float eps;
    float sx, sa;                // S of X (of a matrix that starts near 1) and of A, B
    double growth;               // most that all steps together enlarge a small singular value
};

// What all launches of a list need.  The first is given it and leaves it in the workspace: the others' arguments stay short
// (a launch of 3 KB of arguments costs the host 4.3 us, of 64 bytes 2.8).
struct NsJob {
    NsTable t;
    NsArgs q;
    NsFirst norm, split;
    NsUnits product[4];          // by phase
};
static_assert(sizeof(NsJob) <= 4096, "a kernel's arguments");
// (in the constant address space, as arguments are: scalar loads wherever they stand)
__device__ __forceinline__ const NsJob& job_at(const void* p) {
    return *(const NsJob*)(const __attribute__((address_space(4))) NsJob*)(uintptr_t)p;
}

struct NsStep {
    float a, b, c;
    int src;                     // which X buffer it reads
};

// slices of a matrix of `tiles` tiles of 32 columns (ns_long_kernel): of 16 tiles, two to a wave, at most 256 of them
__host__ __device__ inline int long_slices(int tiles) {
    return tiles >= 256 * 16 ? 256 : (tiles + 15) / 16;
}

// planes of one matrix, in float16 numbers from its workspace: X hi, lo, X^T hi, lo (two buffers), A hi, lo, B hi, lo
struct Planes {
    f16* base;
    int64_t mn, mm;
    __device__ f16* x(int buf, int lo) const { return base + (4 * buf + lo) * mn; }
    __device__ f16* xt(int buf, int lo) const { return base + (4 * buf + 2 + lo) * mn; }
    __device__ f16* a(int lo) const { return base + 8 * mn + lo * mm; }
    __device__ f16* b(int lo) const { return base + 8 * mn + (2 + lo) * mm; }
};
// value (row, k) of a plane of `rows` rows
__device__ __forceinline__ int64_t at_panel(int row, int k, int rows) {
    return ((int64_t)(k >> 3) * rows + row) * 8 + (k & 7);
}
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

// (all of the table at once: searched in a loop, each look waits for the one before)
__device__ __forceinline__ int find_entry(const int* first, int count, int blk) {
    if (count == 1) return 0;
    int i = 0;
#pragma unroll
    for (int k = 1; k < NS_LIST; ++k) i += blk >= first[k];
    return __builtin_amdgcn_readfirstlane(i);
}

// blocks go to the 8 XCDs in turn: block b of n works as unit xcd_order(b, n), which gives each XCD (its own L2) adjacent
// units
__device__ __forceinline__ int xcd_order(int b, int n) {
    const int q = n >> 3, r = n & 7, x = b & 7;
    return (x < r ? x * (q + 1) : r * (q + 1) + (x - r) * q) + (b >> 3);
}

__device__ __forceinline__ float load_any(const void* p, int64_t i, int dtype) {
    if (dtype == PCX_F32) return static_cast<const float*>(p)[i];
    if (dtype == PCX_BF16) return (float)static_cast<const bf16*>(p)[i];
    return (float)static_cast<const f16*>(p)[i];
}
// v = hi + lo to 2^-24 of v: hi by pairs in one conversion, lo = f16(v - hi) in one mixed-precision instruction each
typedef f16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ void split2(float a, float b, f16x2& hi, f16x2& lo) {
    hi = __builtin_convertvector((f32x2{a, b}), f16x2);
    lo = f16x2{(f16)fmaf((float)hi[0], -1.f, a), (f16)fmaf((float)hi[1], -1.f, b)};
}
__device__ __forceinline__ void split4(const float* v, f16x4& hi, f16x4& lo) {
    f16x2 h0, l0, h1, l1;
    split2(v[0], v[1], h0, l0);
    split2(v[2], v[3], h1, l1);
    hi = f16x4{h0[0], h0[1], h1[0], h1[1]};
    lo = f16x4{l0[0], l0[1], l1[0], l1[1]};
}

// the momentum update of one element -> u (the same operations in both passes that need u)
__device__ __forceinline__ float nesterov_u(const NsArgs& q, float g, float m) {
    return q.nesterov ? fmaf(1.f - q.mu, g * q.gs, q.mu * m) : m;
}

// ---------------------------------------------------------------- u, and the sums of its squares (in float64: no range)
__global__ __launch_bounds__(256) void ns_norm_kernel(NsJob job) {
    __shared__ double red[4];
    const NsTable& t = job.t;
    const NsArgs& q = job.q;
    const NsFirst& un = job.norm;
    if (blockIdx.x == 0) {
        for (int i = threadIdx.x; i < (int)(sizeof(NsJob) / 4); i += 256)
            reinterpret_cast<unsigned*>(q.ws)[i] = reinterpret_cast<const unsigned*>(&job)[i];
        for (int i = threadIdx.x; i < q.ndone; i += 256) q.done[i] = 0;
    }
    const int ei = find_entry(un.first, un.count, blockIdx.x);
    const NsMat& e = t.e[ei];
    const int bat = (blockIdx.x - un.first[ei]) / e.parts, blk = (blockIdx.x - un.first[ei]) % e.parts;
    double s = 0.;
    const int64_t n = (int64_t)e.rows * e.cols;
    if (q.is_step || (e.xc == 1 && e.xr == e.cols)) {  // adjacent values
        const int64_t per = (n + e.parts - 1) / e.parts, i0 = blk * per, i1 = i0 + per < n ? i0 + per : n;
        if (q.is_step) {
            const float* g = static_cast<const float*>(e.x);
#pragma unroll 8
            for (int64_t i = i0 + threadIdx.x; i < i1; i += 256) {
                const float gv = g[i], mv = fmaf(1.f - q.mu, gv * q.gs, q.mu * e.mom[i]);
                e.mom[i] = mv;
                const float u = nesterov_u(q, gv, mv);
                s += (double)u * u;
            }
        } else {
            const auto run = [&](auto kind) {
                const auto* x = static_cast<const decltype(kind)*>(e.x) + bat * e.xb;
#pragma unroll 8
                for (int64_t i = i0 + threadIdx.x; i < i1; i += 256) {
                    const double u = (float)x[i];
                    s += u * u;
                }
            };
            if (q.dtype == PCX_F32) run(float());
            else if (q.dtype == PCX_BF16) run(bf16());
            else run(f16());
        }
    } else {  // along the axis of the smaller stride
        const bool turn = llabs(e.xr) < llabs(e.xc);
        const int no = turn ? e.cols : e.rows, ni = turn ? e.rows : e.cols;
        const int64_t so = turn ? e.xc : e.xr, si = turn ? e.xr : e.xc;
        for (int r = blk; r < no; r += e.parts)
            for (int c = threadIdx.x; c < ni; c += 256) {
                const double u = load_any(e.x, bat * e.xb + r * so + c * si, q.dtype);
                s += u * u;
            }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) q.part[(int64_t)(e.mat + bat) * NS_PART + blk] = (red[0] + red[1]) + (red[2] + red[3]);
}

// exponent of the power of two above sx: 0 unless |X|_F times the growth of all steps stays below 1
__device__ __forceinline__ int ns_scale(double fro, double growth) {
    if (!(fro * growth <= 0.5)) return 0;  // (NaN too)
    const double far = 1. / (fro * growth);
    return far > 1e27 ? 90 : ilogb(far);
}

// ---------------------------------------------------------------- X = u S / (|u| + eps) as planes, both ways round
__global__ __launch_bounds__(256) void ns_split_kernel(const void* job) {
    const NsTable& t = job_at(job).t;
    const NsArgs& q = job_at(job).q;
    const NsFirst& un = job_at(job).split;
    __shared__ float tile[64][65];
    __shared__ double red[4];
    __shared__ double scale_s;
    const int ei = find_entry(un.first, un.count, blockIdx.x);
    const NsMat& e = t.e[ei];
    const int tn = e.np / 64, per = (e.mp / 64) * tn;
    // (adjacent tiles to one XCD, as in the products: rows off line boundaries share lines, whole in one L2.  us of this pass
    // in turn / so, three runs each: 6 x 1000 x 333 bfloat16 16.6 / 14.1, 333 x 1000 11.0 / 10.9; where rows are whole
    // lines it costs: 512 x 4608 float32 10.0 / 11.2, 4096 x 4096 bfloat16 35.3 / 36.4)
    const int rel = xcd_order(blockIdx.x - un.first[ei], per * e.batch), bat = rel / per, tl = rel % per;
    const int i0 = (tl / tn) * 64, j0 = (tl % tn) * 64;  // of X (m x n)
    const Planes P = planes_of(q, e, bat);
    const bool tall = e.rows > e.cols;
    // 16 values a thread, the source's columns across the threads, on their way while the norm is formed
    const int sc = threadIdx.x & 63, c = (tall ? i0 : j0) + sc;
    float v[16];
    const auto fetch = [&](auto kind) {
        const auto* x = static_cast<const decltype(kind)*>(e.x) + bat * e.xb + c * e.xc;
#pragma unroll
        for (int k = 0; k < 16; ++k) {
            const int r = (tall ? j0 : i0) + (threadIdx.x >> 6) + 4 * k;
            v[k] = r < e.rows && c < e.cols ? (float)x[r * e.xr] : 0.f;
        }
    };
    if (q.is_step) {
        fetch(float());
        float m[16];
#pragma unroll
        for (int k = 0; k < 16; ++k) {
            const int r = (tall ? j0 : i0) + (threadIdx.x >> 6) + 4 * k;
            m[k] = r < e.rows && c < e.cols ? e.mom[(int64_t)r * e.cols + c] : 0.f;
        }
#pragma unroll
        for (int k = 0; k < 16; ++k) v[k] = nesterov_u(q, v[k], m[k]);
    } else if (q.dtype == PCX_F32) {
        fetch(float());
    } else if (q.dtype == PCX_BF16) {
        fetch(bf16());
    } else {
        fetch(f16());
    }
    {
        double s = 0.;
        for (int i = threadIdx.x; i < e.parts; i += 256) s += q.part[(int64_t)(e.mat + bat) * NS_PART + i];
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
        __syncthreads();
        if (threadIdx.x == 0) {
            const double norm = sqrt((red[0] + red[1]) + (red[2] + red[3])), inv = 1. / (norm + (double)q.eps);
            const int k = ns_scale(norm * inv, q.growth);
            scale_s = ldexp(q.sx * inv, k);
            if (tl == 0) q.unit[e.mat + bat] = ldexpf(1.f / q.sx, -k);
        }
    }
    __syncthreads();
    const double scale = scale_s;
#pragma unroll
    for (int k = 0; k < 16; ++k) {
        const int sr = (threadIdx.x >> 6) + 4 * k;
        tile[tall ? sc : sr][tall ? sr : sc] = (float)(v[k] * scale);
    }
    __syncthreads();
    for (int k = threadIdx.x; k < 64 * 16; k += 256) {
        const int r = (k >> 1) & 63, c = (k & 1) * 4 + (k >> 7) * 8;
        f16x4 h, l, ht, lt;
        const float va[4] = {tile[r][c], tile[r][c + 1], tile[r][c + 2], tile[r][c + 3]};
        const float vt[4] = {tile[c][r], tile[c + 1][r], tile[c + 2][r], tile[c + 3][r]};
        split4(va, h, l);
        split4(vt, ht, lt);
        const int64_t o = at_panel(i0 + r, j0 + c, e.mp), ot = at_panel(j0 + r, i0 + c, e.np);
        *reinterpret_cast<f16x4*>(P.x(0, 0) + o) = h;
        *reinterpret_cast<f16x4*>(P.x(0, 1) + o) = l;
        *reinterpret_cast<f16x4*>(P.xt(0, 0) + ot) = ht;
        *reinterpret_cast<f16x4*>(P.xt(0, 1) + ot) = lt;
    }
}

// ---------------------------------------------------------------- the products
// C[r][c] = sum_k P[r][k] Q[c][k] on tiles of TM = 64 WM rows by TN = 64 WN columns, four waves of 32 WM x 32 WN each.
// The operands' four plane tiles (32 K values of TM + TN rows, hi and lo) are copied to LDS by global_load_lds, 16 bytes
// per lane, NB stages deep.  One barrier per stage, half a stage ahead of its first read: while the first half's MFMAs
// run, the second half's operands are read; then the next stage has landed, its first half is read under the second
// half's MFMAs.  (64 x 64 tiles whose waves take a part of K each, with operands straight to registers and no barrier,
// read every operand once where here LDS gives it to two waves: no faster, 22.0 us against 20.3 for B X of 512 x 4608.)
typedef __attribute__((address_space(3))) void lds_void;

__device__ __forceinline__ f32x16 mfma16(f16x8 a, f16x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ const char* uniform(const void* p) {
    const uint64_t v = (uint64_t)(uintptr_t)p;
    const unsigned lo = __builtin_amdgcn_readfirstlane((unsigned)v), hi = __builtin_amdgcn_readfirstlane((unsigned)(v >> 32));
    return (const char*)(uintptr_t)(((uint64_t)hi << 32) | lo);
}
// (inline asm: behind the builtin, every later LDS read would wait for all copies in flight)
__device__ __forceinline__ void copy16(const char* base, unsigned off, unsigned lds) {
    const unsigned m0 = __builtin_amdgcn_readfirstlane(lds);
    asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "{m0}"(m0) : "memory");
}
template <int N> __device__ __forceinline__ void wait_copies() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// Values exchanged between blocks of one launch.  Each XCD has an L2 of its own: these go past it, store and load by
// store and load, where a fence would write back and drop the whole L2 (measured: a 6 x 333 x 1000 batch in 4 parts per
// tile took 2850 us with fences around the exchange).
__device__ __forceinline__ void put_shared(uint64_t* p, float a, float b) {
    const uint64_t v = (uint64_t)__float_as_uint(a) | (uint64_t)__float_as_uint(b) << 32;
    __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float2 get_shared(const uint64_t* p) {
    const uint64_t v = __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return make_float2(__uint_as_float((unsigned)v), __uint_as_float((unsigned)(v >> 32)));
}

struct Rows {  // the rows of an operand's tile: its planes, first row, rows of the planes
    const f16* hi;
    const f16* lo;
    int first, rows;
};

template <int WM, int WN> struct Frags {
    f16x8 ph[WM], pl[WM], qh[WN], ql[WN];
};

template <int WM, int WN, int NB> struct Product {
    static constexpr int TM = 64 * WM, TN = 64 * WN;
    static constexpr int PB = TM * 64, QB = TN * 64;        // bytes of a plane's tile
    static constexpr int STAGE = 2 * (PB + QB);
    static constexpr int LDS = NB * STAGE > (TM + 8) * TN * 4 ? NB * STAGE : (TM + 8) * TN * 4;  // (the epilogue's tile)
    static constexpr int COPIES = 2 * (WM + WN);            // of a wave and stage

    static constexpr int READS = 2 * (WM + WN), MFMAS = 3 * WM * WN;

    // operand t of a stage's half, this lane's 8 values
    __device__ static const char* operand_at(const char* st, int half) {
        const int lane = threadIdx.x & 63;
        return st + (2 * half + (lane >> 5)) * TM * 16 + (lane & 31) * 16;
    }
    template <int T> __device__ static void read(const char* at, Frags<WM, WN>& f) {
        const int wave = threadIdx.x >> 6;
        const char* p = at + (wave & 1) * 512 * WM;
        const char* c = at + 2 * PB + (wave >> 1) * 512 * WN;
        if constexpr (T < WM) f.ph[T] = *reinterpret_cast<const f16x8*>(p + 512 * T);
        else if constexpr (T < WM + WN) f.ql[T - WM] = *reinterpret_cast<const f16x8*>(c + QB + 512 * (T - WM));
        else if constexpr (T < 2 * WM + WN) f.pl[T - WM - WN] = *reinterpret_cast<const f16x8*>(p + PB + 512 * (T - WM - WN));
        else f.qh[T - 2 * WM - WN] = *reinterpret_cast<const f16x8*>(c + 512 * (T - 2 * WM - WN));
    }
    // MFMA t of a half: the small terms first, neighbours in different accumulators
    template <int T> __device__ static void mfma(const Frags<WM, WN>& f, f32x16 (&acc)[WM][WN]) {
        constexpr int term = T / (WM * WN), i = T / WN % WM, j = T % WN;
        acc[i][j] = mfma16(term == 1 ? f.pl[i] : f.ph[i], term == 0 ? f.ql[j] : f.qh[j], acc[i][j]);
    }
    // One half's MFMAs with the next half's operand reads (and a stage's copies, `fetch`) spread between them: all the
    // reads in one run fill the LDS queue, and a wave's MFMAs wait behind its own reads.
    template <int T = 0, typename F>
    __device__ __forceinline__ static void half_step(const Frags<WM, WN>& f, f32x16 (&acc)[WM][WN], const char* next, Frags<WM, WN>& g, F fetch) {
        if constexpr (T < READS) {
            read<T>(next, g);
            fetch(std::integral_constant<int, T>());
            mfmas<T * MFMAS / READS, (T + 1) * MFMAS / READS>(f, acc);
            __builtin_amdgcn_sched_barrier(0);
            half_step<T + 1>(f, acc, next, g, fetch);
        }
    }
    template <int A, int B> __device__ static void mfmas(const Frags<WM, WN>& f, f32x16 (&acc)[WM][WN]) {
        if constexpr (A < B) {
            mfma<A>(f, acc);
            mfmas<A + 1, B>(f, acc);
        }
    }
    template <int T = 0> __device__ static void read_all(const char* at, Frags<WM, WN>& f) {
        if constexpr (T < READS) {
            read<T>(at, f);
            read_all<T + 1>(at, f);
        }
    }

    // stages [s0, s1) of K
    __device__ static void run(const Rows& P, const Rows& Q, int s0, int s1, char* sm, f32x16 (&acc)[WM][WN]) {
        const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        const unsigned lds0 = (unsigned)(uintptr_t)(lds_void*)sm;
        unsigned offp[WM], offq[WN];  // (rows behind the planes' last: that one again, for sums that nobody stores)
#pragma unroll
        for (int i = 0; i < WM; ++i) offp[i] = (unsigned)(wave * P.rows + min(64 * i + lane, P.rows - P.first - 1)) * 16;
#pragma unroll
        for (int i = 0; i < WN; ++i) offq[i] = (unsigned)(wave * Q.rows + min(64 * i + lane, Q.rows - Q.first - 1)) * 16;
        const char* base[4] = {uniform(P.hi + P.first * 8), uniform(P.lo + P.first * 8), uniform(Q.hi + Q.first * 8),
                               uniform(Q.lo + Q.first * 8)};
        // copy T of this wave for a stage
        const auto copy = [&](auto t, int s, int buf) {
            constexpr int T = decltype(t)::value, pl = T / (WM + WN), x = T % (WM + WN);
            const unsigned at = lds0 + (unsigned)(buf * STAGE + wave * TM * 16);
            if constexpr (x < WM) copy16(base[pl] + (int64_t)s * P.rows * 64, offp[x], at + pl * PB + x * 1024);
            else copy16(base[2 + pl] + (int64_t)s * Q.rows * 64, offq[x - WM], at + 2 * PB + pl * QB + (x - WM) * 1024);
        };
        const int n = s1 - s0;
        copies(copy, s0, 0);
        if (n > 1) copies(copy, s0 + 1, 1);
        if (NB > 2 && n > 2) copies(copy, s0 + 2, 2);
        if (NB > 2 && n > 2) wait_copies<2 * COPIES>();
        else if (n > 1) wait_copies<COPIES>();
        else wait_copies<0>();
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        Frags<WM, WN> f0, f1;
        read_all(operand_at(sm, 0), f0);
        int buf = 0, s = 0;
        // (two loops and no branch inside: a join would move all accumulators)
        for (; s + NB < n; ++s) {
            half_step(f0, acc, operand_at(sm + buf * STAGE, 1), f1, [](auto) {});
            turn<(NB - 2) * COPIES>();
            const int freed = buf;
            buf = buf + 1 == NB ? 0 : buf + 1;
            half_step(f1, acc, operand_at(sm + buf * STAGE, 0), f0, [&](auto t) { copy(t, s0 + s + NB, freed); });
        }
        for (; s < n; ++s) {  // (the operands read behind the last stage are not used)
            half_step(f0, acc, operand_at(sm + buf * STAGE, 1), f1, [](auto) {});
            turn<0>();
            buf = buf + 1 == NB ? 0 : buf + 1;
            half_step(f1, acc, operand_at(sm + buf * STAGE, 0), f0, [](auto) {});
        }
    }
    // every wave is done with the stage's buffer, and the next stage has landed
    template <int N> __device__ __forceinline__ static void turn() {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        wait_copies<N>();
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    }
    template <int T = 0, typename F> __device__ static void copies(F copy, int s, int buf) {
        if constexpr (T < COPIES) {
            copy(std::integral_constant<int, T>(), s, buf);
            copies<T + 1>(copy, s, buf);
        }
    }
};

// what is stored for a result v: itself, or the parameter `old` moved by it
template <typename T> struct Plain {
    __device__ static T old(const T*) { return T(); }
    __device__ T operator()(T, float v) const { return (T)v; }
};
struct Descend {
    float decay, step;
    __device__ static float old(const float* p) { return *p; }
    __device__ float operator()(float w, float v) const { return fmaf(decay, w, -step * v); }
};

enum NsPhase { NS_GRAM = 0, NS_POLY = 1, NS_APPLY = 2, NS_LAST = 3 };

// NS_GRAM: A = X X^T.  NS_POLY: B = b A + c A A.  Both symmetric: of each pair of 64-blocks across the diagonal one is
// computed and written twice.  NS_APPLY: X <- a X + B X, both ways round.  NS_LAST: that to the caller's matrices.
template <int PHASE, int WM, int WN, int NB> __global__ __launch_bounds__(256) void ns_product_kernel(const void* job, NsStep st) {
    const NsTable& t = job_at(job).t;
    const NsArgs& q = job_at(job).q;
    const NsUnits& un = job_at(job).product[PHASE];
    using G = Product<WM, WN, NB>;
    constexpr bool SYM = PHASE <= NS_POLY;
    extern __shared__ __attribute__((aligned(16))) char sm[];
    __shared__ int last;
    const int ei = find_entry(un.first, un.count, blockIdx.x);
    const NsMat& e = t.e[ei];
    const unsigned rel = blockIdx.x - un.first[ei], whole = un.whole[ei], split = un.split[ei], tiles = un.tiles[ei];
    const unsigned cut = tiles * e.batch - whole;
    // Adjacent units to one XCD: split tiles in part order share their K range there, whole tiles their rows (X <- a X + B X
    // of 512 x 4608 20.3 -> 17.5 us; units in turn give each XCD one column of tiles and all of X).  Where the tiles fill the
    // card more than once, in turn is better: 372 us against 397 at 4096 x 4096.
    const int over = rel < whole ? -1 : xcd_order(rel - whole, cut * split);
    const int part = over < 0 ? 0 : (unsigned)over / cut;
    const unsigned tile = over < 0 ? (whole <= NS_ROUND ? xcd_order(rel, whole) : rel) : whole + over - part * cut;
    const int bat = e.batch == 1 ? 0 : tile / tiles;
    int tl = tile - bat * tiles;
    const Planes p = planes_of(q, e, bat);
    // rows r0 .., columns c0 .. of the product, and its operands.  The accumulators hold four adjacent rows per lane, so
    // the side that lies along memory in the output gives the rows.
    const bool tall = PHASE == NS_LAST && e.rows > e.cols;
    int r0, c0;
    Rows P, Q;
    if (SYM) {
        int ti = 0;
        for (;; ++ti) {
            if (tl <= ti) break;
            tl -= ti + 1;
        }
        r0 = ti * G::TM;
        c0 = tl * G::TN;
        const f16* hi = PHASE == NS_GRAM ? p.x(st.src, 0) : p.a(0);
        const f16* lo = PHASE == NS_GRAM ? p.x(st.src, 1) : p.a(1);
        P = Rows{hi, lo, r0, e.mp};
        Q = Rows{hi, lo, c0, e.mp};
    } else {
        const int tc = ((tall ? e.np : e.mp) + G::TN - 1) / G::TN;
        const int tr = (unsigned)tl / (unsigned)tc;
        r0 = tr * G::TM;
        c0 = (tl - tr * tc) * G::TN;
        const Rows B{p.b(0), p.b(1), tall ? r0 : c0, e.mp};
        const Rows X{p.xt(st.src, 0), p.xt(st.src, 1), tall ? c0 : r0, e.np};
        P = tall ? B : X;
        Q = tall ? X : B;
    }
    const int stages = (int)((PHASE == NS_GRAM ? e.np : e.mp) / NS_K);
    // the old values of small tiles are on their way during the product (these are latency, not throughput)
    const f16* oldh = PHASE == NS_POLY ? p.a(0) : tall ? p.xt(st.src, 0) : p.x(st.src, 0);
    const f16* oldl = PHASE == NS_POLY ? p.a(1) : tall ? p.xt(st.src, 1) : p.x(st.src, 1);
    const int orow = tall ? e.np : e.mp;  // rows of the old values' and the output's planes: the product's columns
    const int nr = min(G::TM, (SYM || tall ? e.mp : e.np) - r0), nc = min(G::TN, (SYM ? e.mp : tall ? e.np : e.mp) - c0);
    constexpr bool EARLY = WM * WN == 1 && PHASE != NS_GRAM;
    f16x4 eh[EARLY ? 4 : 1], el[EARLY ? 4 : 1];
    if (EARLY) {
#pragma unroll
        for (int y = 0; y < 4; ++y) {
            const int x = threadIdx.x + 256 * y, c = x / 2 % G::TN, r = x % 2 * 4 + x / (2 * G::TN) * 8;
            const int64_t o = at_panel(c0 + c, r0 + r, orow);  // (64 x 64: nothing reaches over the padding)
            eh[y] = *reinterpret_cast<const f16x4*>(oldh + o);
            el[y] = *reinterpret_cast<const f16x4*>(oldl + o);
        }
    }
    const float unit = q.unit[e.mat + bat];
    f32x16 acc[WM][WN];
#pragma unroll
    for (int i = 0; i < WM; ++i)
#pragma unroll
        for (int j = 0; j < WN; ++j) acc[i][j] = f32x16{};
    // (a matrix of 2^20 columns has 2^15 stages, and at most 16 parts)
    const int s0 = over < 0 ? 0 : (int)((unsigned)(stages * part) / (unsigned)split);
    const int s1 = over < 0 ? stages : (int)((unsigned)(stages * (part + 1)) / (unsigned)split);
    G::run(P, Q, s0, s1, sm, acc);
    if (over >= 0) {
        {
            // the tile's parts meet in memory; the unit that ends last adds them in part order
            constexpr int SZ = G::TM * G::TN;
            uint64_t* mine = reinterpret_cast<uint64_t*>(q.joint + (int64_t)(un.joint[ei] + over) * SZ) + threadIdx.x;
#pragma unroll
            for (int i = 0; i < WM; ++i)
#pragma unroll
                for (int j = 0; j < WN; ++j)
#pragma unroll
                    for (int g = 0; g < 8; ++g)
                        put_shared(mine + ((i * WN + j) * 8 + g) * 256, acc[i][j][2 * g], acc[i][j][2 * g + 1]);
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // (they have reached what every XCD reads)
            __syncthreads();
            unsigned* done = q.done + un.tail[ei] + over % cut;
            if (threadIdx.x == 0)
                last = __hip_atomic_fetch_add(done, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (unsigned)split - 1u;
            __syncthreads();
            if (!last) return;
            if (threadIdx.x == 0) __hip_atomic_store(done, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);  // for the next launch
#pragma unroll
            for (int i = 0; i < WM; ++i)
#pragma unroll
                for (int j = 0; j < WN; ++j) acc[i][j] = f32x16{};
            const uint64_t* from = reinterpret_cast<const uint64_t*>(q.joint + (int64_t)(un.joint[ei] + over % cut) * SZ) + threadIdx.x;
            constexpr int FLY = WM * WN == 1 ? 5 : 2;  // parts in flight (8 would cost a CU its third block: 17 -> 19 us at 512 x 4608)
            for (int k = 0; k < split; k += FLY) {
#pragma unroll
                for (int i = 0; i < WM; ++i)
#pragma unroll
                    for (int j = 0; j < WN; ++j) {
                        float2 v[FLY][8];
#pragma unroll
                        for (int f = 0; f < FLY; ++f)
#pragma unroll
                            for (int g = 0; g < 8; ++g)
                                v[f][g] = get_shared(from + (int64_t)min(k + f, split - 1) * cut * (SZ / 2) + ((i * WN + j) * 8 + g) * 256);
#pragma unroll
                        for (int f = 0; f < FLY; ++f)
                            if (k + f < split) {
#pragma unroll
                                for (int g = 0; g < 8; ++g) {
                                    acc[i][j][2 * g] += v[f][g].x;
                                    acc[i][j][2 * g + 1] += v[f][g].y;
                                }
                            }
                    }
            }
        }
    }
    // The tile goes through LDS, [column][row], so that both passes over it touch whole lines of memory: along the rows
    // first, where the old values are added, then across.
    constexpr int LS = G::TM + 8;  // (two float4 of a column, then the next: 8 columns share no bank)
    float* tv = reinterpret_cast<float*>(sm);
    {
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
        const float k = PHASE == NS_GRAM ? q.sa * unit * unit : PHASE == NS_POLY ? st.c / q.sa : 1.f / q.sa;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < WM; ++i)
#pragma unroll
            for (int j = 0; j < WN; ++j) {
                float* at = tv + ((wave >> 1) * 32 * WN + 32 * j + (lane & 31)) * LS + (wave & 1) * 32 * WM + 32 * i;
#pragma unroll
                for (int g = 0; g < 4; ++g)
                    st4(at + acc_row(4 * g, lane >> 5), make_float4(acc[i][j][4 * g] * k, acc[i][j][4 * g + 1] * k,
                                                                    acc[i][j][4 * g + 2] * k, acc[i][j][4 * g + 3] * k));
            }
        __syncthreads();
    }
    f16* outh = PHASE == NS_GRAM ? p.a(0) : PHASE == NS_POLY ? p.b(0) : p.x(1 - st.src, 0);
    f16* outl = PHASE == NS_GRAM ? p.a(1) : PHASE == NS_POLY ? p.b(1) : p.x(1 - st.src, 1);
#pragma unroll 8
    for (int x0 = 0; x0 < G::TM * G::TN / 4; x0 += 256) {
        const int x = x0 + threadIdx.x, c = x / 2 % G::TN, r = x % 2 * 4 + x / (2 * G::TN) * 8;
        if (r >= nr || c >= nc) continue;
        if (SYM && (r0 + r) / 64 < (c0 + c) / 64) continue;  // (the mirrored block writes it)
        float* at = tv + c * LS + r;
        const float4 was = ld4(at);
        float v[4] = {was.x, was.y, was.z, was.w};
        const int64_t o = at_panel(c0 + c, r0 + r, orow);
        if (PHASE != NS_GRAM) {
            const f16x4 oh = EARLY ? eh[EARLY ? x0 / 256 : 0] : *reinterpret_cast<const f16x4*>(oldh + o);
            const f16x4 ol = EARLY ? el[EARLY ? x0 / 256 : 0] : *reinterpret_cast<const f16x4*>(oldl + o);
            const float f = PHASE == NS_POLY ? st.b : st.a;
#pragma unroll
            for (int y = 0; y < 4; ++y) v[y] = fmaf(f, (float)oh[y] + (float)ol[y], v[y]);
        }
        if (PHASE != NS_LAST) {
            f16x4 h, l;
            split4(v, h, l);
            *reinterpret_cast<f16x4*>(outh + o) = h;
            *reinterpret_cast<f16x4*>(outl + o) = l;
        }
        if (PHASE >= NS_POLY) st4(at, make_float4(v[0], v[1], v[2], v[3]));
    }
    __syncthreads();
    if (PHASE != NS_LAST) {
        f16* acrh = PHASE == NS_APPLY ? p.xt(1 - st.src, 0) : outh;
        f16* acrl = PHASE == NS_APPLY ? p.xt(1 - st.src, 1) : outl;
#pragma unroll 4
        for (int x = threadIdx.x; x < G::TM * G::TN / 4; x += 256) {
            const int r = x / 2 % G::TM, c = x % 2 * 4 + x / (2 * G::TM) * 8;
            if (r >= nr || c >= nc) continue;
            if (SYM && (r0 + r) / 64 <= (c0 + c) / 64) continue;
            const float* at = tv + c * LS + r;
            const float v[4] = {at[0], at[LS], at[2 * LS], at[3 * LS]};
            f16x4 h, l;
            split4(v, h, l);
            const int64_t o = at_panel(r0 + r, c0 + c, PHASE == NS_APPLY ? e.np : e.mp);
            *reinterpret_cast<f16x4*>(acrh + o) = h;
            *reinterpret_cast<f16x4*>(acrl + o) = l;
        }
        return;
    }
    const auto finish = [&](auto kind, auto put) {
        using T = decltype(kind);
        T* out = static_cast<T*>(e.out) + (int64_t)bat * e.rows * e.cols;
        // (16 values a thread at a time: the parameters are read from HBM)
        const int r = threadIdx.x % G::TM, cs = threadIdx.x / G::TM;
        if (r0 + r >= e.cols) return;
        T* o = out + (int64_t)(c0 + cs) * e.cols + r0 + r;
        const float* at = tv + cs * LS + r;
        constexpr int STEP = 256 / G::TM;
#pragma unroll 1
        for (int x0 = 0; x0 < G::TN; x0 += 16 * STEP) {
            T old[16];
#pragma unroll
            for (int x = 0; x < 16; ++x) {
                const int c = x0 + x * STEP;
                if (c0 + cs + c < e.rows) old[x] = put.old(o + (int64_t)c * e.cols);
            }
#pragma unroll
            for (int x = 0; x < 16; ++x) {
                const int c = x0 + x * STEP;
                if (c0 + cs + c < e.rows) o[(int64_t)c * e.cols] = put(old[x], at[c * LS] * unit);
            }
        }
    };
    if (q.is_step) finish(float(), Descend{q.decay, e.step});
    else if (q.dtype == PCX_F32) finish(float(), Plain<float>());
    else if (q.dtype == PCX_BF16) finish(bf16(), Plain<bf16>());
    else finish(f16(), Plain<f16>());
}

// ---------------------------------------------------------------- products of few tiles
// 32 x 32 tiles, all waves of a block on one of them, each on every W-th stage of K: nothing is shared between waves, so
// operands go from memory straight to registers, three stages ahead, with no barrier until the waves' sums meet in LDS.
// Four times the blocks of 64 x 64 tiles and a quarter of the epilogue for each, for launches that are all latency.
constexpr int NSF_WAVES = 8;

template <int PHASE> __global__ __launch_bounds__(64 * NSF_WAVES) void ns_few_kernel(const void* job, NsStep st) {
    const NsTable& t = job_at(job).t;
    const NsArgs& q = job_at(job).q;
    const NsUnits& un = job_at(job).product[PHASE];
    constexpr bool SYM = PHASE <= NS_POLY;
    constexpr int W = NSF_WAVES, LS = 40, AHEAD = 3;
    __shared__ __attribute__((aligned(16))) float tv[W][32 * LS];
    const int ei = find_entry(un.first, un.count, blockIdx.x);
    const NsMat& e = t.e[ei];
    const unsigned rel = blockIdx.x - un.first[ei], tiles = un.tiles[ei];
    const int bat = e.batch == 1 ? 0 : rel / tiles;
    int tl = rel - bat * tiles;
    const Planes p = planes_of(q, e, bat);
    const bool tall = PHASE == NS_LAST && e.rows > e.cols;
    int r0, c0;
    Rows P, Q;
    if (SYM) {
        int ti = 0;
        for (; tl > ti; ++ti) tl -= ti + 1;
        r0 = ti * 32;
        c0 = tl * 32;
        const f16* hi = PHASE == NS_GRAM ? p.x(st.src, 0) : p.a(0);
        const f16* lo = PHASE == NS_GRAM ? p.x(st.src, 1) : p.a(1);
        P = Rows{hi, lo, r0, e.mp};
        Q = Rows{hi, lo, c0, e.mp};
    } else {
        const int tc = (tall ? e.np : e.mp) / 32, tr = (unsigned)tl / (unsigned)tc;
        r0 = tr * 32;
        c0 = (tl - tr * tc) * 32;
        const Rows B{p.b(0), p.b(1), tall ? r0 : c0, e.mp};
        const Rows X{p.xt(st.src, 0), p.xt(st.src, 1), tall ? c0 : r0, e.np};
        P = tall ? B : X;
        Q = tall ? X : B;
    }
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int stages = (PHASE == NS_GRAM ? e.np : e.mp) / NS_K;
    // each thread's four values of the result: rows r .. r + 3 of column c
    const int c = (threadIdx.x >> 1) & 31, r = (threadIdx.x & 1) * 4 + (threadIdx.x >> 6 & 3) * 8;
    const bool mine = threadIdx.x < 256;
    const f16* oldh = PHASE == NS_POLY ? p.a(0) : tall ? p.xt(st.src, 0) : p.x(st.src, 0);
    const f16* oldl = PHASE == NS_POLY ? p.a(1) : tall ? p.xt(st.src, 1) : p.x(st.src, 1);
    const int64_t o = at_panel(c0 + c, r0 + r, tall ? e.np : e.mp);
    f16x4 oh{}, ol{};
    if (PHASE != NS_GRAM) {
        oh = *reinterpret_cast<const f16x4*>(oldh + o);
        ol = *reinterpret_cast<const f16x4*>(oldl + o);
    }
    const float unit = q.unit[e.mat + bat];

    const unsigned offp = ((lane & 31) + (lane >> 5) * P.rows) * 16, offq = ((lane & 31) + (lane >> 5) * Q.rows) * 16;
    const char* base[4] = {uniform(P.hi + P.first * 8), uniform(P.lo + P.first * 8), uniform(Q.hi + Q.first * 8),
                           uniform(Q.lo + Q.first * 8)};
    const int64_t kp = (int64_t)P.rows * 64, kq = (int64_t)Q.rows * 64;
    f16x8 f[AHEAD][2][4];  // [stage][half][P hi, P lo, Q hi, Q lo]
    const auto fetch = [&](int s, f16x8 (&g)[2][4]) {
        const int k = min(s, stages - 1);  // (behind the end: not used)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int y = 0; y < 4; ++y)
                g[h][y] = *reinterpret_cast<const f16x8*>(base[y] + k * (y < 2 ? kp : kq) + h * (y < 2 ? kp : kq) / 2 + (y < 2 ? offp : offq));
    };
    f32x16 a0{}, a1{}, a2{};
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) fetch(wave + i * W, f[i]);
    for (int s = wave; s < stages; s += AHEAD * W) {
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            if (s + i * W < stages) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    a0 = mfma16(f[i][h][0], f[i][h][3], a0);
                    a1 = mfma16(f[i][h][1], f[i][h][2], a1);
                    a2 = mfma16(f[i][h][0], f[i][h][2], a2);
                }
            }
            if (s + (i + AHEAD) * W < stages) fetch(s + (i + AHEAD) * W, f[i]);
        }
    }
    a2 += a0 + a1;
#pragma unroll
    for (int g = 0; g < 4; ++g)
        st4(&tv[wave][(lane & 31) * LS + acc_row(4 * g, lane >> 5)],
            make_float4(a2[4 * g], a2[4 * g + 1], a2[4 * g + 2], a2[4 * g + 3]));
    __syncthreads();
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    if (mine) {
        const int used = min(W, stages);
        for (int w = 0; w < used; ++w) {
            const float4 x = ld4(&tv[w][c * LS + r]);
            v[0] += x.x;
            v[1] += x.y;
            v[2] += x.z;
            v[3] += x.w;
        }
        const float k = PHASE == NS_GRAM ? q.sa * unit * unit : PHASE == NS_POLY ? st.c / q.sa : 1.f / q.sa;
        const float fo = PHASE == NS_POLY ? st.b : st.a;
#pragma unroll
        for (int y = 0; y < 4; ++y) v[y] = PHASE == NS_GRAM ? v[y] * k : fmaf(fo, (float)oh[y] + (float)ol[y], v[y] * k);
    }
    if (PHASE != NS_LAST) {
        f16* outh = PHASE == NS_GRAM ? p.a(0) : PHASE == NS_POLY ? p.b(0) : p.x(1 - st.src, 0);
        f16* outl = PHASE == NS_GRAM ? p.a(1) : PHASE == NS_POLY ? p.b(1) : p.x(1 - st.src, 1);
        f16x4 h, l;
        split4(v, h, l);
        if (mine) {
            *reinterpret_cast<f16x4*>(outh + o) = h;
            *reinterpret_cast<f16x4*>(outl + o) = l;
        }
        if (SYM && r0 == c0) return;  // (the same for the block)
        __syncthreads();
        if (mine) st4(&tv[0][c * LS + r], make_float4(v[0], v[1], v[2], v[3]));
        __syncthreads();
        if (!mine) return;
        f16* acrh = PHASE == NS_APPLY ? p.xt(1 - st.src, 0) : outh;
        f16* acrl = PHASE == NS_APPLY ? p.xt(1 - st.src, 1) : outl;
        const float w[4] = {tv[0][r * LS + c], tv[0][(r + 1) * LS + c], tv[0][(r + 2) * LS + c], tv[0][(r + 3) * LS + c]};
        split4(w, h, l);
        const int64_t oa = at_panel(r0 + c, c0 + r, PHASE == NS_APPLY ? e.np : e.mp);
        *reinterpret_cast<f16x4*>(acrh + oa) = h;
        *reinterpret_cast<f16x4*>(acrl + oa) = l;
        return;
    }
    if (!mine || c0 + c >= e.rows) return;
    const auto finish = [&](auto kind, auto put) {
        using T = decltype(kind);
        T* out = static_cast<T*>(e.out) + (int64_t)bat * e.rows * e.cols + (int64_t)(c0 + c) * e.cols + r0 + r;
        T old[4];
#pragma unroll
        for (int y = 0; y < 4; ++y)
            if (r0 + r + y < e.cols) old[y] = put.old(out + y);
#pragma unroll
        for (int y = 0; y < 4; ++y)
            if (r0 + r + y < e.cols) out[y] = put(old[y], v[y] * unit);
    };
    if (q.is_step) finish(float(), Descend{q.decay, e.step});
    else if (q.dtype == PCX_F32) finish(float(), Plain<float>());
    else if (q.dtype == PCX_BF16) finish(bf16(), Plain<bf16>());
    else finish(f16(), Plain<f16>());
}

// ---------------------------------------------------------------- small matrices: all steps in one block
// X of up to 32 tiles of 32 x 32 stays in the registers of eight waves (in float32, T tiles a wave); its planes, X for the
// gram product and then X^T, and the planes of A and then B pass through LDS.  A launch per product costs 5 us and more
// however small it is, and there are 3 per step: 128 x 128 took 96 us that way, 57 us here (of a step's 10 us 4.4 are
// MFMAs, the rest LDS traffic, the splitting into hi and lo, and barriers).
constexpr int NSB_WAVES = 8, NSB_LDS = 159 * 1024;

// float16 number (row, k) of an LDS plane of `rows` rows: panels of 32 K values, runs of 8 swizzled over the slots
__device__ __forceinline__ int at_lds(int row, int k, int rows) {
    return ((k >> 5) * rows + row) * 32 + 8 * (((k >> 3) & 3) ^ ((row >> 2) & 3)) + (k & 7);
}

struct LdsRows {  // planes in LDS: hi, lo `d` numbers further, rows of a panel
    const f16* hi;
    int d, rows;
};
// two 32 x 32 tiles of sum_k P[p0 + r][k] Q[q + c][k], k < 16 n, for q = q0 and q1: the P operands are read once (the
// kernel is bound by its LDS reads).  The small terms have sums of their own: an MFMA does not wait for its neighbour.
__device__ __forceinline__ void block_product(const LdsRows& P, int p0, const LdsRows& Q, int q0, int q1, int n, int l32, int h,
                                              f32x16 (&c)[2]) {
    f32x16 s[2] = {};
    c[0] = c[1] = f32x16{};
    const int slot[2] = {8 * (h ^ ((l32 >> 2) & 3)), 8 * ((2 + h) ^ ((l32 >> 2) & 3))};
    const f16* pp = P.hi + (p0 + l32) * 32;
    const f16* qq = Q.hi + (q0 + l32) * 32;
    const int dq = (q1 - q0) * 32;
    for (int k = 0; k < n; k += 2, pp += P.rows * 32, qq += Q.rows * 32) {
#pragma unroll
        for (int y = 0; y < 2; ++y) {
            const f16x8 ph = *reinterpret_cast<const f16x8*>(pp + slot[y]), pl = *reinterpret_cast<const f16x8*>(pp + slot[y] + P.d);
            f16x8 qh[2], ql[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                qh[i] = *reinterpret_cast<const f16x8*>(qq + slot[y] + i * dq);
                ql[i] = *reinterpret_cast<const f16x8*>(qq + slot[y] + i * dq + Q.d);
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) s[i] = mfma16(ph, ql[i], s[i]);
#pragma unroll
            for (int i = 0; i < 2; ++i) c[i] = mfma16(ph, qh[i], c[i]);
#pragma unroll
            for (int i = 0; i < 2; ++i) s[i] = mfma16(pl, qh[i], s[i]);
        }
    }
    c[0] += s[0];
    c[1] += s[1];
}
// a tile's value (r, c) as plane element (row c, k r): four adjacent k at a time
__device__ __forceinline__ void put_along(f16* pl, int d, int rows, int r0, int c, int h, const f32x16& v) {
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        const float x[4] = {v[4 * g], v[4 * g + 1], v[4 * g + 2], v[4 * g + 3]};
        f16x4 hi, lo;
        split4(x, hi, lo);
        f16* at = pl + at_lds(c, r0 + acc_row(4 * g, h), rows);
        *reinterpret_cast<f16x4*>(at) = hi;
        *reinterpret_cast<f16x4*>(at + d) = lo;
    }
}

// and as (row r, k c): adjacent lanes swap rows first, so that each writes two adjacent k
__device__ __forceinline__ void put_across(f16* pl, int d, int rows, int r0, int c0, int l32, int h, const f32x16& v) {
    const bool odd = l32 & 1;
    // rows 16 apart are swizzled alike, and the lane's row of a pair (odd: the second) in the same slot
    f16* at[2] = {pl + at_lds(r0 + 4 * h, c0 + (l32 & ~1), rows) + 32 * odd,
                  pl + at_lds(r0 + 4 * h + 8, c0 + (l32 & ~1), rows) + 32 * odd - 8 * 32};
#pragma unroll
    for (int k = 0; k < 16; k += 2) {
        // of rows k, k + 1 the even lane keeps the first and gets its neighbour's, the odd one the second
        float first = v[k], second = v[k + 1];
        asm("" : "+v"(first), "+v"(second));  // (or the choice becomes an index into v)
        const float give = odd ? first : second, keep = odd ? second : first;
        const float got = __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(give), 0xb1, 0xf, 0xf, true));
        f16x2 hi, lo;
        split2(odd ? got : keep, odd ? keep : got, hi, lo);
        f16* to = at[(k >> 2) & 1] + acc_row(k, 0) * 32;
        *reinterpret_cast<f16x2*>(to) = hi;
        *reinterpret_cast<f16x2*>(to + d) = lo;
    }
}

// One step of a matrix whose short side is one tile, in float32 throughout: its sums are short, and the 22 bits of two
// float16 numbers were most of its error (medians of 40 gradients, times float32 arithmetic's own: 3 x 5 1.7 with planes,
// 0.8 here; 1 x 50 1.5 and 1.0; 32 x 288 1.1 and 0.9).  It is no slower, as its operands need no splitting and its step two
// barriers: 9 x 32 21.7 and 17.0 us, 32 x 288 39.7 and 34.3, 32 x 1000 92 and 70.
// `n`: tiles of X from the wave's first on; it has numbers 0, 1, 16 and 17 of them, as far as they exist.
// A lane holds rows acc_row(k, h) of its column, which are values of K to B X as they stand, and, symmetric, A and B are
// their own operands; only X X^T takes X through LDS, a tile at a time and the wave's own.
constexpr int NSB_TILE = 32 * 33;
// g += x x^T, through the wave's own tile in LDS
__device__ __forceinline__ void tile_gram(float* own, const f32x16& x, int l32, int h, f32x16& g) {
#pragma unroll
    for (int k = 0; k < 16; ++k) own[l32 * 33 + acc_row(k, h)] = x[k];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
    for (int k = 0; k < 16; ++k) {
        const float v = own[(2 * k + h) * 33 + l32];
        g = mfma32(v, v, g);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
}
// B = b A + c A A as an operand, from A in LDS
__device__ __forceinline__ void tile_poly(const float* A, int l32, int h, float b, float c, float (&v)[16]) {
    f32x16 p{};
#pragma unroll
    for (int k = 0; k < 16; ++k) v[k] = A[l32 * 33 + acc_row(k, h)];
#pragma unroll
    for (int k = 0; k < 16; ++k) p = mfma32(v[k], v[k], p);
#pragma unroll
    for (int k = 0; k < 16; ++k) v[k] = fmaf(c, p[k], b * v[k]);
}
// a x + B x
__device__ __forceinline__ f32x16 tile_apply(const float (&v)[16], const f32x16& x, float a) {
    f32x16 y{};
#pragma unroll
    for (int k = 0; k < 16; ++k) y = mfma32(v[k], x[k], y);
    return x * a + y;
}
template <int T> __device__ __forceinline__ void tile_step(float* lds, f32x16 (&x)[T / 2][2], int n, int waves, int l32, int h,
                                                           float unit2, float a, float b, float c) {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    float* own = lds + wave * NSB_TILE;
    float* all = lds + waves * NSB_TILE;
    f32x16 g{};
    if (n > 0) {
#pragma unroll
        for (int i = 0; i < T; ++i) {
            if (2 * NSB_WAVES * (i / 2) + i % 2 < n) tile_gram(own, x[i / 2][i % 2], l32, h, g);
        }
#pragma unroll
        for (int k = 0; k < 16; ++k) own[acc_row(k, h) * 33 + l32] = g[k];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 32 * 32; i += 64 * NSB_WAVES) {
        const int at = (i >> 5) * 33 + (i & 31);
        float s = 0.f;
        for (int w = 0; w < waves; ++w) s += lds[w * NSB_TILE + at];
        all[at] = s * unit2;
    }
    __syncthreads();
    if (n <= 0) return;
    float v[16];
    tile_poly(all, l32, h, b, c, v);
#pragma unroll
    for (int i = 0; i < T; ++i)
        if (2 * NSB_WAVES * (i / 2) + i % 2 < n) x[i / 2][i % 2] = tile_apply(v, x[i / 2][i % 2], a);
}

// kinds of matrices in a launch: short sides of one tile, of more, or some of each (with the code of both, a wave of 4 tiles
// has too few registers: 64 x 512 78 -> 88 us)
enum NsKind { NSB_ONE = 1, NSB_MORE = 2, NSB_BOTH = 3 };
template <int T, int KIND> __global__ __launch_bounds__(64 * NSB_WAVES) void ns_block_kernel(NsTable t, NsFirst un, NsArgs q, NsCoef coef) {
    extern __shared__ __attribute__((aligned(16))) char sm[];
    __shared__ double red[NSB_WAVES + 2];
    const int ei = find_entry(un.first, un.count, blockIdx.x);
    const NsMat& e = t.e[ei];
    const int bat = blockIdx.x - un.first[ei];
    const bool tall = e.rows > e.cols;
    const int m = tall ? e.cols : e.rows, n = tall ? e.rows : e.cols;
    const int mb = (m + 31) / 32, nb = (n + 31) / 32, mp = 32 * mb, np = 32 * nb;
    f16* X = reinterpret_cast<f16*>(sm);
    f16* A = X + 2 * mp * np;
    const int dx = mp * np, da = mp * mp;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l32 = threadIdx.x & 31, h = (threadIdx.x >> 5) & 1;
    // u comes in through LDS, whole rows at a time: [rows][cols | 1]
    float* raw = reinterpret_cast<float*>(sm);
    const int pitch = e.cols | 1, total = e.rows * e.cols;
    double s = 0.;
    constexpr int THREADS = 64 * NSB_WAVES, FLY = 16;
    const bool linear = e.xc == 1 && e.xr == e.cols;
    const float by_cols = 1.f / (float)e.cols;  // (i + 1/2 is 2^-11 of a column away from the next row: i < 2^15)
    const auto fetch = [&](auto kind) {
        const auto* src = static_cast<const decltype(kind)*>(e.x) + bat * e.xb;
        for (int i0 = threadIdx.x; i0 < total; i0 += FLY * THREADS) {
            float u[FLY], mo[FLY];
            int at[FLY];
#pragma unroll
            for (int y = 0; y < FLY; ++y) {
                const int i = min(i0 + y * THREADS, total - 1), r = (int)((i + 0.5f) * by_cols), c = i - r * e.cols;
                at[y] = r * pitch + c;
                u[y] = (float)src[linear ? i : r * e.xr + c * e.xc];
                if (q.is_step) mo[y] = e.mom[i];
            }
#pragma unroll
            for (int y = 0; y < FLY; ++y) {
                if (i0 + y * THREADS >= total) break;
                if (q.is_step) {
                    const float mv = fmaf(1.f - q.mu, u[y] * q.gs, q.mu * mo[y]);
                    e.mom[i0 + y * THREADS] = mv;
                    u[y] = nesterov_u(q, u[y], mv);
                }
                raw[at[y]] = u[y];
                s += (double)u[y] * u[y];
            }
        }
    };
    if (q.dtype == PCX_F32) fetch(float());
    else if (q.dtype == PCX_BF16) fetch(bf16());
    else fetch(f16());
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    if ((threadIdx.x & 63) == 0) red[wave] = s;
    __syncthreads();
    if (wave == 0) {  // (64-bit roots and quotients: once)
        s = 0.;
#pragma unroll
        for (int w = 0; w < NSB_WAVES; ++w) s += red[w];
        const double norm = sqrt(s), inv = 1. / (norm + (double)q.eps);
        if (threadIdx.x == 0) {
            const int k = ns_scale(norm * inv, q.growth);
            red[NSB_WAVES] = ldexp(q.sx * inv, k);
            red[NSB_WAVES + 1] = (double)k;
        }
    }
    __syncthreads();
    const int lift = (int)red[NSB_WAVES + 1];
    const double scale = red[NSB_WAVES];  // (up to 2^248 where norm and eps are float32's smallest: no float32 holds it)
    const float unit = ldexpf(1.f / q.sx, -lift);
    // The wave's tiles of X, in pairs along n: of pair i rows 32 tr[i] of m, columns 32 tc[i] of n and the next 32 (a pair
    // at an odd end has no second tile: it computes one that is not stored).  And its pair of tiles of A.
    const int pr = tall ? 1 : pitch, pc = tall ? pitch : 1, row_pairs = (nb + 1) / 2, a_pairs = (mb + 1) / 2;
    int tr[T / 2], tc[T / 2];
    f32x16 x[T / 2][2];
#pragma unroll
    for (int i = 0; i < T / 2; ++i) {
        const int pair = wave + NSB_WAVES * i;
        tr[i] = pair / row_pairs;
        tc[i] = 2 * (pair % row_pairs);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int r0 = 32 * tr[i] + 4 * h, c = 32 * (tc[i] + j) + l32;
            const float* at = raw + r0 * pr + c * pc;
#pragma unroll
            for (int k = 0; k < 16; ++k)
                x[i][j][k] = r0 + acc_row(k, 0) < m && c < n ? (float)(at[acc_row(k, 0) * pr] * scale) : 0.f;
        }
    }
    const int ar = wave / a_pairs, ac = 2 * (wave % a_pairs);
    __syncthreads();

    for (int step = 0; step < coef.steps; ++step) {
        const float a = coef.c[3 * step], b = coef.c[3 * step + 1], c = coef.c[3 * step + 2];
        int lane = threadIdx.x & 63;
        asm volatile("" : "+v"(lane));  // (addresses are formed anew: kept over the steps, they take the registers of X)
        const int l32 = lane & 31, h = lane >> 5;
        if (KIND == NSB_ONE || (KIND == NSB_BOTH && mb == 1)) {
            tile_step<T>(reinterpret_cast<float*>(sm), x, tr[0] == 0 ? nb - tc[0] : 0, min(NSB_WAVES, row_pairs), l32, h,
                         unit * unit, a, b, c);
            continue;
        }
        if (step) __syncthreads();  // (X^T and B of the last step are read)
#pragma unroll
        for (int i = 0; i < T; ++i) {  // X planes: rows of m, K along n
            if (tr[i / 2] < mb && tc[i / 2] + i % 2 < nb)
                put_across(X, dx, mp, 32 * tr[i / 2], 32 * (tc[i / 2] + i % 2), l32, h, x[i / 2][i % 2]);
            __builtin_amdgcn_sched_barrier(0);
        }
        __syncthreads();
        f32x16 g[2], p[2];
        if (ar < mb) {
            const LdsRows XR{X, dx, mp};
            block_product(XR, 32 * ar, XR, 32 * ac, 32 * min(ac + 1, mb - 1), 2 * nb, l32, h, g);
            const float k = q.sa * unit * unit;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                g[j] *= k;
                if (ac + j < mb) put_along(A, da, mp, 32 * ar, 32 * (ac + j) + l32, h, g[j]);
            }
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < T; ++i) {  // X^T planes: rows of n, K along m
            if (tr[i / 2] < mb && tc[i / 2] + i % 2 < nb)
                put_along(X, dx, np, 32 * tr[i / 2], 32 * (tc[i / 2] + i % 2) + l32, h, x[i / 2][i % 2]);
            __builtin_amdgcn_sched_barrier(0);
        }
        if (ar < mb) {
            const LdsRows AR{A, da, mp};
            block_product(AR, 32 * ar, AR, 32 * ac, 32 * min(ac + 1, mb - 1), 2 * mb, l32, h, p);
#pragma unroll
            for (int j = 0; j < 2; ++j) g[j] = g[j] * b + p[j] * (c / q.sa);
        }
        __syncthreads();
        if (ar < mb) {
#pragma unroll
            for (int j = 0; j < 2; ++j)
                if (ac + j < mb) put_along(A, da, mp, 32 * ar, 32 * (ac + j) + l32, h, g[j]);
        }
        __syncthreads();
        const LdsRows BR{A, da, mp}, XR{X, dx, np};
        const float k = 1.f / q.sa;
#pragma unroll
        for (int i = 0; i < T / 2; ++i) {
            if (tr[i] < mb) {
                block_product(BR, 32 * tr[i], XR, 32 * tc[i], 32 * min(tc[i] + 1, nb - 1), 2 * mb, l32, h, p);
#pragma unroll
                for (int j = 0; j < 2; ++j) x[i][j] = x[i][j] * a + p[j] * k;
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < T; ++i) {
        const int r0 = 32 * tr[i / 2] + 4 * h, c = 32 * (tc[i / 2] + i % 2) + l32;
        float* at = raw + r0 * pr + c * pc;
#pragma unroll
        for (int k = 0; k < 16; ++k)
            if (r0 + acc_row(k, 0) < m && c < n) at[acc_row(k, 0) * pr] = x[i / 2][i % 2][k] * unit;
    }
    __syncthreads();
    const auto finish = [&](auto kind, auto put) {
        using V = decltype(kind);
        V* out = static_cast<V*>(e.out) + (int64_t)bat * total;
#pragma unroll 8
        for (int i = threadIdx.x; i < total; i += 64 * NSB_WAVES) {
            const int r = (int)((i + 0.5f) * by_cols), c = i - r * e.cols;
            out[i] = put(put.old(out + i), raw[r * pitch + c]);
        }
    };
    if (q.is_step) finish(float(), Descend{q.decay, e.step});
    else if (q.dtype == PCX_F32) finish(float(), Plain<float>());
    else if (q.dtype == PCX_BF16) finish(bf16(), Plain<bf16>());
    else finish(f16(), Plain<f16>());
}

// ---------------------------------------------------------------- long matrices of at most 32 rows
// The same steps in float32 where the long side has more than a block's registers: X lies in memory, in tiles of 32 columns
// as the registers hold them, a block works on a slice of its tiles, and a launch per step takes A from the slices' sums
// of the last one (two sets of them, in turn) and leaves its own: X is read and written once a step, and A, B cost every
// block 32 MFMAs.  Launches: the norm, X with its first sums, and one a step.  As products of planes 22 bits were most of the
// error, and 17 launches most of the time: 4 x 3999 1.7e-6 and 100 us, 0.6e-6 and 54 us so; 1 x 2000 0.66e-6 and 89 us, 0.44e-6
// and 57; 32 x 1100 78 and 51 us, 32 x 8192 116 and 60, 32 x 2^20 5.1 and 0.46 ms (1.74 GB move: 3.8 TB/s).
enum NsLong { NSL_FIRST, NSL_STEP, NSL_LAST };

template <int PHASE> __global__ __launch_bounds__(64 * NSB_WAVES) void ns_long_kernel(const void* job, NsStep st) {
    const NsTable& t = job_at(job).t;
    const NsArgs& q = job_at(job).q;
    const NsFirst& un = job_at(job).split;
    __shared__ float lds[(NSB_WAVES + 1) * NSB_TILE];
    __shared__ double red[NSB_WAVES];
    const int ei = find_entry(un.first, un.count, blockIdx.x);
    const NsMat& e = t.e[ei];
    const bool tall = e.rows > e.cols;
    const int m = tall ? e.cols : e.rows, n = tall ? e.rows : e.cols, tiles = (n + 31) / 32;
    const int slices = long_slices(tiles), rel = blockIdx.x - un.first[ei], bat = rel / slices, slice = rel - bat * slices;
    const int each = (tiles + slices - 1) / slices, t0 = slice * each, t1 = min(t0 + each, tiles);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l32 = threadIdx.x & 31, h = (threadIdx.x >> 5) & 1;
    float* X = reinterpret_cast<float*>(q.ws + e.ws) + (int64_t)bat * tiles * 1024 + (threadIdx.x & 63) * 4;
    float* own = lds + wave * NSB_TILE;
    float* all = lds + NSB_WAVES * NSB_TILE;
    const auto sums = [&](int set) { return q.joint + ((int64_t)set * q.slices + blockIdx.x) * 1024; };
    float v[16];
    double scale = 0.;
    float unit = 1.f;
    if (PHASE == NSL_FIRST) {
        double s = 0.;
        for (int i = threadIdx.x; i < e.parts; i += 64 * NSB_WAVES) s += q.part[(int64_t)(e.mat + bat) * NS_PART + i];
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
        if ((threadIdx.x & 63) == 0) red[wave] = s;
        __syncthreads();
        s = 0.;
#pragma unroll
        for (int w = 0; w < NSB_WAVES; ++w) s += red[w];
        const double norm = sqrt(s), inv = 1. / (norm + (double)q.eps);
        const int k = ns_scale(norm * inv, q.growth);
        scale = ldexp(inv, k);
        if (slice == 0 && threadIdx.x == 0) q.unit[e.mat + bat] = ldexpf(1.f, -k);
    } else {
        unit = q.unit[e.mat + bat];
        const float* from = sums(st.src) - (int64_t)slice * 1024;
        for (int i = threadIdx.x; i < 1024; i += 64 * NSB_WAVES) {
            float s = 0.f;
#pragma unroll 8
            for (int w = 0; w < slices; ++w) s += from[w * 1024 + i];
            all[(i >> 5) * 33 + (i & 31)] = s * unit * unit;
        }
        __syncthreads();
        tile_poly(all, l32, h, st.b, st.c, v);
    }
    f32x16 g{};
    for (int at = t0 + wave; at < t1; at += NSB_WAVES) {
        const int c = 32 * at + l32;
        f32x16 x;
        float* to = X + (int64_t)at * 1024;
        if (PHASE == NSL_FIRST) {
            const auto fetch = [&](auto kind) {
                const auto* src = static_cast<const decltype(kind)*>(e.x) + bat * e.xb;
#pragma unroll
                for (int k = 0; k < 16; ++k) {
                    const int r = acc_row(k, h), row = tall ? c : r, col = tall ? r : c;
                    float u = 0.f;
                    if (r < m && c < n) {
                        u = (float)src[row * e.xr + col * e.xc];
                        if (q.is_step) u = nesterov_u(q, u, e.mom[(int64_t)row * e.cols + col]);
                    }
                    x[k] = (float)(u * scale);
                }
            };
            if (q.dtype == PCX_F32) fetch(float());
            else if (q.dtype == PCX_BF16) fetch(bf16());
            else fetch(f16());
        } else {
#pragma unroll
            for (int k = 0; k < 16; k += 4) {
                const float4 w = ld4(to + 64 * k);
                x[k] = w.x;
                x[k + 1] = w.y;
                x[k + 2] = w.z;
                x[k + 3] = w.w;
            }
            x = tile_apply(v, x, st.a);
        }
        if (PHASE != NSL_LAST) {
#pragma unroll
            for (int k = 0; k < 16; k += 4) st4(to + 64 * k, make_float4(x[k], x[k + 1], x[k + 2], x[k + 3]));
            tile_gram(own, x, l32, h, g);
            continue;
        }
        const auto finish = [&](auto kind, auto put) {
            using T = decltype(kind);
            T* out = static_cast<T*>(e.out) + (int64_t)bat * e.rows * e.cols;
#pragma unroll
            for (int k = 0; k < 16; ++k) {
                const int r = acc_row(k, h);
                if (r >= m || c >= n) continue;
                T* o = out + (int64_t)(tall ? c : r) * e.cols + (tall ? r : c);
                *o = put(put.old(o), x[k] * unit);
            }
        };
        if (q.is_step) finish(float(), Descend{q.decay, e.step});
        else if (q.dtype == PCX_F32) finish(float(), Plain<float>());
        else if (q.dtype == PCX_BF16) finish(bf16(), Plain<bf16>());
        else finish(f16(), Plain<f16>());
    }
    if (PHASE == NSL_LAST) return;
#pragma unroll
    for (int k = 0; k < 16; ++k) own[acc_row(k, h) * 33 + l32] = g[k];
    __syncthreads();
    float* to = sums(PHASE == NSL_FIRST ? 0 : 1 - st.src);
    for (int i = threadIdx.x; i < 1024; i += 64 * NSB_WAVES) {
        float s = 0.f;
#pragma unroll
        for (int w = 0; w < NSB_WAVES; ++w) s += lds[w * NSB_TILE + (i >> 5) * 33 + (i & 31)];
        to[i] = s;
    }
}

// ---------------------------------------------------------------- host
int round_up(int v, int k) { return (v + k - 1) / k * k; }

void set_shape(NsMat& e, int64_t rows, int64_t cols) {
    e.rows = (int)rows;
    e.cols = (int)cols;
    e.mp = round_up((int)std::min(rows, cols), NS_PAD);
    e.np = round_up((int)std::max(rows, cols), NS_PAD);
    e.parts = (int)std::min<int64_t>(NS_PART, (rows * cols + 2047) / 2048);
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

constexpr int NS_TM[3] = {64, 128, 32}, NS_PER_CU[3] = {3, 2, 1};  // of NsConfig: tile edges; blocks a CU holds

// tiles of one matrix of an entry in a phase
int64_t ns_tiles(const NsMat& e, int phase, int edge) {
    const int64_t tm = (e.mp + edge - 1) / edge, tn = (e.np + edge - 1) / edge;
    return phase <= NS_POLY ? tm * (tm + 1) / 2 : tm * tn;
}
int ns_stages(const NsMat& e, int phase) { return (phase == NS_GRAM ? e.np : e.mp) / NS_K; }

// 128 x 128 tiles do the same work with half the LDS reads per MFMA and half the traffic from L2, 64 x 64 tiles spread it
// over four times the blocks.  us for 64 / 128 of X <- a X + B X (tiles of 128, stages of K): 1024 x 4096 (256, 32) 45 / 39,
// 4 x 1024 x 1024 (256, 32) 45 / 38, 16 x 256 x 1024 (256, 8) 21 / 21, 768 x 6144 (288, 24) 39 / 41, 4 x 512 x 4608
// (576, 16) 61 / 52; of X X^T: 4 x 1024 x 1024 (144, 32) 26 / 29, 3 x 1536 x 1536 (234, 48) 54 / 54, 8 x 1024 x 1024
// (288, 32) 50 / 47, 32 x 512 x 512 (320, 16) 44 / 30.  Large tiles from one per CU on if K is long, else from five per
// four CUs, counted by the longest: the deep network's weights (310 tiles, worth 258 of the longest) take 26 / 30.
// 32 x 32 tiles are for launches that are all latency.  us for 32 / 64: A A of 512 x 512 (36 tiles of 64) 6.3 / 8.2,
// B X of 512 x 512 (64) 7.9 / 9.6, X X^T of 512 x 2048 (36, 64 stages) 11.5 / 12.4 but of 512 x 4608 (144 stages)
// 20.4 / 16.9, A A of 6 x 333 x 333 (126) 11.3 / 8.2: up to a 64 x 64 tile per four CUs and 64 stages.
enum NsConfig { NS_TILE64, NS_TILE128, NS_TILE32 };
NsConfig ns_config(const NsTable& t, int phase) {
    int64_t small = 0, work = 0, most = 0;  // 64 x 64 tiles; stages of all 128 x 128 tiles, and of one
    for (int i = 0; i < t.count; ++i) {
        const int64_t stages = ns_stages(t.e[i], phase);
        small += ns_tiles(t.e[i], phase, 64) * t.e[i].batch;
        work += ns_tiles(t.e[i], phase, 128) * t.e[i].batch * stages;
        most = std::max(most, stages);
    }
    if (4 * small <= num_cus() && most <= 64) return NS_TILE32;
    const int64_t each = num_cus() * most;
    return 4 * work >= 5 * each || (most >= 32 && work >= each) ? NS_TILE128 : NS_TILE64;
}

struct NsPlan {
    NsUnits un;
    NsConfig cfg;
    unsigned blocks;
    int64_t counters, joint;  // split tiles, floats of their parts
};

// Units of a product launch: as many as the card holds at a time (`slots`), of about the same number of stages.
NsPlan ns_plan(const NsTable& t, int phase) {
    NsPlan p{};
    p.cfg = ns_config(t, phase);
    const int edge = NS_TM[p.cfg];
    const int64_t slots = (int64_t)num_cus() * NS_PER_CU[p.cfg];
    int64_t units = 0, parts = 0;
    int stages[NS_LIST];
    for (int i = 0; i < t.count; ++i) {
        p.un.tiles[i] = (int)ns_tiles(t.e[i], phase, edge);
        stages[i] = ns_stages(t.e[i], phase);
    }
    p.un.count = t.count;
    int64_t all = 0;
    for (int i = 0; i < t.count; ++i) all += (int64_t)p.un.tiles[i] * t.e[i].batch;
    for (int i = 0; i < t.count; ++i) {
        const int64_t n = (int64_t)p.un.tiles[i] * t.e[i].batch;
        int64_t whole = 0, split = 1;
        if (t.count == 1 && n >= slots) {  // full rounds of whole tiles, the rest in parts
            whole = n / slots * slots;
            if (n > whole) split = std::max<int64_t>(1, std::min<int64_t>(slots / (n - whole), stages[i] / 16));
        } else if (stages[i] >= 48) {
            // a stage takes about 0.17 us, meeting in memory 4 us and 0.3 us a part: sqrt(0.6 stages) parts are the best,
            // and no meeting pays for K of less than 48 stages.  (More parts of the longest K in a list, up to as many
            // units as the card holds: 22.8 us against 20.9 for X X^T of the deep network's weights.)
            split = std::min<int64_t>((int64_t)(sqrt(0.6 * stages[i]) + 0.5), std::max<int64_t>(1, slots / all));
        }
        split = p.cfg == NS_TILE32 ? 1 : std::min<int64_t>(split, 16);  // (there the waves share K)
        if (split == 1) whole = n;
        p.un.whole[i] = (int)whole;
        p.un.split[i] = (int)split;
        p.un.tail[i] = (int)p.counters;
        p.un.joint[i] = (int)parts;
        p.un.first[i] = (int)units;
        p.counters += n - whole;
        parts += (n - whole) * split;
        units += whole + (n - whole) * split;
    }
    for (int i = t.count; i < NS_LIST; ++i) p.un.first[i] = INT_MAX;
    p.blocks = (unsigned)units;
    p.joint = parts * edge * edge;
    return p;
}

// Units of the passes over values: `per` blocks to a matrix of an entry.
template <typename F> unsigned ns_blocks(const NsTable& t, NsFirst& un, F per) {
    int64_t n = 0;
    un.count = t.count;
    for (int i = 0; i < t.count; ++i) {
        un.first[i] = (int)n;
        n += per(t.e[i]) * t.e[i].batch;
    }
    for (int i = t.count; i < NS_LIST; ++i) un.first[i] = INT_MAX;
    return (unsigned)n;
}

// pairs of tiles along the long side, and the bytes of a matrix's planes in LDS if one block holds it (0 if not): at most
// two pairs a wave, and one of A's
int ns_block_pairs(const NsMat& e) {
    return ((std::min(e.rows, e.cols) + 31) / 32) * ((std::max(e.rows, e.cols) + 63) / 64);
}
int ns_block_bytes(const NsMat& e) {
    if (std::min(e.rows, e.cols) > 128 || std::max(e.rows, e.cols) > 1024 || ns_block_pairs(e) > 2 * NSB_WAVES) return 0;
    const int64_t mp = round_up(std::min(e.rows, e.cols), 32), np = round_up(std::max(e.rows, e.cols), 32);
    int64_t bytes = 4 * (mp * np + (int64_t)mp * mp);
    if (mp == 32) bytes = std::max<int64_t>(bytes, 4 * NSB_TILE * (std::min(NSB_WAVES, ns_block_pairs(e)) + 1));
    return bytes <= NSB_LDS ? (int)bytes : 0;
}

// the launch's matrices in blocks of their own: bytes of LDS and pairs of the largest, and their kinds (0: one does not fit)
int ns_in_blocks(const NsTable& t, int* bytes, int* pairs) {
    int kind = 0;
    *bytes = *pairs = 0;
    for (int i = 0; i < t.count; ++i) {
        const int b = ns_block_bytes(t.e[i]);
        if (!b) return 0;
        *bytes = std::max(*bytes, b);
        *pairs = std::max(*pairs, ns_block_pairs(t.e[i]));
        kind |= std::min(t.e[i].rows, t.e[i].cols) <= 32 ? NSB_ONE : NSB_MORE;
    }
    return kind;
}

// the launch's matrices are all of at most 32 rows or columns (and too long for blocks of their own)
bool ns_all_short(const NsTable& t) {
    for (int i = 0; i < t.count; ++i)
        if (std::min(t.e[i].rows, t.e[i].cols) > 32) return false;
    return true;
}
int long_tiles(const NsMat& e) { return (std::max(e.rows, e.cols) + 31) / 32; }

// One launch table's workspace: the job, partial sums and unit of every matrix, counters and partial products of split tiles,
// then the planes.  Fills in the places; returns its size.
int64_t ns_place(NsTable& t, NsArgs& q, void* ws) {
    int64_t mats = 0, counters = 0, joint = 0;
    for (int i = 0; i < t.count; ++i) {
        t.e[i].mat = (int)mats;
        mats += t.e[i].batch;
    }
    t.mats = (int)mats;
    int bytes, pairs;
    if (ns_in_blocks(t, &bytes, &pairs)) return 256;  // (nothing passes through memory)
    const bool all_short = ns_all_short(t);
    if (all_short) {
        int64_t slices = 0;
        for (int i = 0; i < t.count; ++i) slices += (int64_t)long_slices(long_tiles(t.e[i])) * t.e[i].batch;
        q.slices = (int)slices;
        joint = 2 * slices * 1024;
    } else {
        for (int ph = NS_GRAM; ph <= NS_LAST; ++ph) {
            const NsPlan p = ns_plan(t, ph);
            counters = std::max(counters, p.counters);
            joint = std::max(joint, p.joint);
        }
    }
    int64_t off = 0;
    const auto take = [&](int64_t bytes) {
        const int64_t at = off;
        off = (off + bytes + 255) / 256 * 256;
        return reinterpret_cast<char*>(reinterpret_cast<uintptr_t>(ws) + (uintptr_t)at);
    };
    q.ws = static_cast<char*>(ws);
    take(sizeof(NsJob));
    q.ndone = (int)counters;
    char* a = take(mats * NS_PART * (int64_t)sizeof(double));
    char* b = take(mats * (int64_t)sizeof(float));
    char* c = take(counters * (int64_t)sizeof(unsigned));
    char* d = take(joint * (int64_t)sizeof(float));
    q.part = reinterpret_cast<double*>(a);
    q.unit = reinterpret_cast<float*>(b);
    q.done = reinterpret_cast<unsigned*>(c);
    q.joint = reinterpret_cast<float*>(d);
    for (int i = 0; i < t.count; ++i) {
        t.e[i].ws = off;
        take(t.e[i].batch * (all_short ? (int64_t)long_tiles(t.e[i]) * 4096 : plane_bytes(t.e[i].mp, t.e[i].np)));
    }
    return off;
}

template <int PHASE, int WM, int WN, int NB> int ns_product_as(const NsPlan& p, const void* job, const NsStep& st, hipStream_t s) {
    constexpr int sm = Product<WM, WN, NB>::LDS;
    if (sm > 64 * 1024)
        (void)hipFuncSetAttribute((const void*)ns_product_kernel<PHASE, WM, WN, NB>, hipFuncAttributeMaxDynamicSharedMemorySize, sm);
    ns_product_kernel<PHASE, WM, WN, NB><<<p.blocks, 256, sm, s>>>(job, st);
    PCX_LAUNCH_CHECK("ns_product_kernel");
    return PCX_OK;
}
template <int PHASE> int ns_product(const NsPlan* plans, const void* job, const NsStep& st, hipStream_t s) {
    const NsPlan& p = plans[PHASE];
    if (p.cfg == NS_TILE32) {
        ns_few_kernel<PHASE><<<p.blocks, 64 * NSF_WAVES, 0, s>>>(job, st);
        PCX_LAUNCH_CHECK("ns_few_kernel");
        return PCX_OK;
    }
    if (p.cfg == NS_TILE64) return ns_product_as<PHASE, 1, 1, 3>(p, job, st, s);
    return ns_product_as<PHASE, 2, 2, 2>(p, job, st, s);
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

template <int T, int KIND> int ns_block_as(const NsTable& t, const NsFirst& un, const NsArgs& q, const NsCoef& c, unsigned n, int sm, hipStream_t s) {
    if (sm > 64 * 1024)
        (void)hipFuncSetAttribute((const void*)ns_block_kernel<T, KIND>, hipFuncAttributeMaxDynamicSharedMemorySize, sm);
    ns_block_kernel<T, KIND><<<n, 64 * NSB_WAVES, sm, s>>>(t, un, q, c);
    PCX_LAUNCH_CHECK("ns_block_kernel");
    return PCX_OK;
}
template <int T> int ns_block_of(int kind, const NsTable& t, const NsFirst& un, const NsArgs& q, const NsCoef& c, unsigned n, int sm, hipStream_t s) {
    if (kind == NSB_ONE) return ns_block_as<T, NSB_ONE>(t, un, q, c, n, sm, s);
    if (kind == NSB_MORE) return ns_block_as<T, NSB_MORE>(t, un, q, c, n, sm, s);
    return ns_block_as<T, NSB_BOTH>(t, un, q, c, n, sm, s);
}

int ns_run(const NsTable& t, const NsArgs& q, const float* coef, int steps, hipStream_t s) {
    int most, pairs;
    if (const int kind = ns_in_blocks(t, &most, &pairs)) {
        NsCoef c{};
        c.steps = steps;
        memcpy(c.c, coef, 3 * steps * sizeof(float));
        NsFirst un{};
        const unsigned n = ns_blocks(t, un, [](const NsMat&) { return (int64_t)1; });
        if (pairs <= NSB_WAVES) return ns_block_of<2>(kind, t, un, q, c, n, most, s);
        return ns_block_of<4>(kind, t, un, q, c, n, most, s);
    }
    NsJob job{t, q, {}, {}, {}};
    if (ns_all_short(t)) {
        const unsigned nn = ns_blocks(t, job.norm, [](const NsMat& e) { return (int64_t)e.parts; });
        const unsigned n = ns_blocks(t, job.split, [](const NsMat& e) { return (int64_t)long_slices(long_tiles(e)); });
        ns_norm_kernel<<<nn, 256, 0, s>>>(job);
        PCX_LAUNCH_CHECK("ns_norm_kernel");
        ns_long_kernel<NSL_FIRST><<<n, 64 * NSB_WAVES, 0, s>>>(q.ws, NsStep{});
        PCX_LAUNCH_CHECK("ns_long_kernel");
        for (int k = 0; k < steps; ++k) {
            const NsStep st{coef[3 * k], coef[3 * k + 1], coef[3 * k + 2], k & 1};
            if (k + 1 < steps) ns_long_kernel<NSL_STEP><<<n, 64 * NSB_WAVES, 0, s>>>(q.ws, st);
            else ns_long_kernel<NSL_LAST><<<n, 64 * NSB_WAVES, 0, s>>>(q.ws, st);
            PCX_LAUNCH_CHECK("ns_long_kernel");
        }
        return PCX_OK;
    }
    NsPlan plans[4];
    for (int ph = NS_GRAM; ph <= NS_LAST; ++ph) {
        plans[ph] = ns_plan(t, ph);
        job.product[ph] = plans[ph].un;
    }
    const unsigned nn = ns_blocks(t, job.norm, [](const NsMat& e) { return (int64_t)e.parts; });
    const unsigned ns = ns_blocks(t, job.split, [](const NsMat& e) { return (int64_t)(e.mp / 64) * (e.np / 64); });
    ns_norm_kernel<<<nn, 256, 0, s>>>(job);
    PCX_LAUNCH_CHECK("ns_norm_kernel");
    ns_split_kernel<<<ns, 256, 0, s>>>(q.ws);
    PCX_LAUNCH_CHECK("ns_split_kernel");
    for (int k = 0; k < steps; ++k) {
        const NsStep st{coef[3 * k], coef[3 * k + 1], coef[3 * k + 2], k & 1};
        int rc = ns_product<NS_GRAM>(plans, q.ws, st, s);
        if (!rc) rc = ns_product<NS_POLY>(plans, q.ws, st, s);
        if (!rc) rc = k + 1 < steps ? ns_product<NS_APPLY>(plans, q.ws, st, s) : ns_product<NS_LAST>(plans, q.ws, st, s);
        if (rc) return rc;
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
    return rows * cols <= (int64_t)1 << 31 && batch < (int64_t)1 << 24 && batch * tiles < (int64_t)1 << 26;
}

int ns_check(const char* what, int steps, const float* coef, float eps) {
    PCX_CHECK_ARG(steps >= 1 && steps <= NS_STEPS, "%s: 1 to %d steps (got %d)", what, NS_STEPS, steps);
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
        e.xr = a.cols;
        e.xc = 1;
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
    NsArgs q{};
    ns_single(t, batch, rows, cols);
    return (size_t)ns_place(t, q, nullptr);
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
    const int64_t need = ns_place(t, q, ws);
    if (!ws || ((uintptr_t)ws & 255) || (int64_t)ws_bytes < need) {
        set_error("orthogonalize: workspace of %zu bytes, %lld on a 256-byte boundary needed", ws_bytes, (long long)need);
        return PCX_EWORKSPACE;
    }
    NsMat& e = t.e[0];
    e.x = x;
    e.xb = batch_stride;
    e.xr = row_stride;
    e.xc = col_stride;
    e.out = out;
    q.dtype = dtype;
    q.eps = eps;
    return ns_run(t, q, coef, steps, stream);
}

extern "C" size_t pcx_muon_workspace_bytes(const pcx_muon_matrix* mats, int n) {
    if (n <= 0 || !mats) return 0;
    int64_t most = 0;
    for (int at = 0; at < n; at += NS_LIST) {
        NsTable t{};
        NsArgs q{};
        if (muon_part(mats, n, at, t) != PCX_OK) return 0;
        most = std::max(most, ns_place(t, q, nullptr));
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
        const int64_t need = ns_place(t, q, ws);
        if (!ws || ((uintptr_t)ws & 255) || (int64_t)ws_bytes < need) {
            set_error("muon_step: workspace of %zu bytes, %lld on a 256-byte boundary needed", ws_bytes, (long long)need);
            return PCX_EWORKSPACE;
        }
    }
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
        ns_place(t, q, ws);
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
