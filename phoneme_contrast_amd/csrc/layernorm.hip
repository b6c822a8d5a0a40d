// Layer norm over the last axis, forward and backward.
//
//   mean = sum_d x / D          var = sum_d (x - mean)^2 / D          rstd = 1 / sqrt(var + eps)
//   xhat = (x - mean) rstd      y = xhat w + b
//   g = dy w   c1 = sum_d g / D   c2 = sum_d g xhat / D   dx = rstd (g - c1 - xhat c2)
//   dw = sum_rows dy xhat       db = sum_rows dy
//
// Both passes are bound by HBM: 2 tensors move in the forward, 3 in the backward.  A row is read once and stays in
// registers between its reductions, and the backward sums dw / db over the rows of its block in registers, so x and dy
// are read once for dx, dw and db together.  Every sum is in 32 bits or more and in a fixed order: results repeat bit by bit.
// Rows far from zero: a mean off by one of its own steps would be the whole of a narrow row's xhat.  So the deviations
// d = x - m from the first mean m are summed next to their squares, e = sum d / D, var = sum d^2 / D - e^2 and
// xhat = (d - e) rstd; where e^2 makes up more than a quarter of sum d^2 / D (the subtraction would cancel), m moves to
// m + e first, which the row does at most twice.  A constant row gives the bias, whatever its value.  The statistics keep
// m + e rounded to float32: the backward's xhat is off by rstd times half a step of the mean.
// Measured: 8192 x 5120 in float16 forward 34 us a call, 4.9 TB/s (29.7 by the kernel's own clock, where a copy's 5.86 TB/s
// would take 28.6); 16384 x 4096 in bfloat16 with its gradients 140 us, 4.8 TB/s (forward 50, backward 85 and 6).  Rows of
// 4097 values, none of them aligned: bfloat16 forward 60 us, float32 92, with gradients 181 and 248.  12000 values: 8192
// rows of bfloat16 with gradients 226 us.  Behind 16384 values nothing is kept from one pass to the next: 4096 x 32768
// bfloat16 forward 122 us (92 at a copy's rate), with gradients 562 (229).
// Few rows are latency: 24 x 128 with its gradients 7 us in two kernels, 35 to 65 us of the host's way through autograd.
//
// A row belongs to 1 ... 64 lanes of a wave or to a block of just the waves it needs: sub-wave rows need no barrier, and
// wider ones one barrier per reduction.  Rows of up to 32 values are computed in 64 bits from x itself: at D = 2 the three
// terms of dx cancel to eps / (var + eps) of their size, which 32-bit statistics do not resolve, and such rows are short
// of bytes, not of arithmetic.
#include "kernels.h"

#include <type_traits>

namespace pcx {
namespace {

typedef __bf16 bf16;
typedef _Float16 f16;

constexpr int LN_MAX = 32768;    // 1024 threads x 32 values
constexpr int LN_NARROW = 32;    // rows up to here: 64-bit arithmetic, one value per lane
constexpr int LN_ALONE = 8192;   // rows up to here: a single block writes dw and db itself

struct LnArgs {
    int64_t rows;
    int D, tpr, wf32, cf32;      // tpr: lanes of a sub-wave row; wf32, cf32: w and b, dw and db are float32 (else x's type)
    float eps;
    const void* x;
    int64_t xs;                  // row strides in elements
    const void* w;               // readable rows of D values even without weights (hw, hb: 1 and 0 in their place)
    const void* b;
    bool hw, hb;
    void* y;
    float2* stat;                // [rows] {mean, rstd}; NULL: not kept
    const void* dy;
    int64_t dys;
    void* dx;                    // NULL: not wanted
    bool cols;                   // dw, db wanted
    void* part;                  // [blocks][2][D] partial dw, db, in 64 bits for narrow rows, else in 32; NULL: one block,
                                 // which writes them itself
    void* dw;
    void* db;
};

// V values that lie anywhere: rows of an odd length, slices, and strides that are no multiple of 16 bytes take the same
// 16-byte loads and stores as aligned ones.
template <typename T, int V> struct Pack {
    typedef T type __attribute__((ext_vector_type(V), aligned(alignof(T))));
};
template <typename T> struct Pack<T, 1> {
    typedef T type;
};

template <typename T, int V> using pack = typename Pack<T, V>::type;

template <int V, typename T> __device__ __forceinline__ pack<T, V> load_raw(const T* p) {
    return *reinterpret_cast<const pack<T, V>*>(p);
}
template <typename T, int V> __device__ __forceinline__ void widen(const pack<T, V>& t, float* v) {
    if constexpr (V == 1) {
        v[0] = (float)t;
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = (float)t[j];
    }
}
template <int V, typename T> __device__ __forceinline__ void load_v(const T* p, float* v) {
    constexpr int N = V * (int)sizeof(T) > 16 ? 16 / (int)sizeof(T) : V;  // (float weights of 16-bit rows: two loads)
#pragma unroll
    for (int k = 0; k < V / N; ++k) widen<T, N>(load_raw<N>(p + k * N), v + k * N);
}
template <int V, typename T> __device__ __forceinline__ void store_v(T* p, const float* v) {
    pack<T, V> t;
#pragma unroll
    for (int j = 0; j < V; ++j) t[j] = (T)v[j];
    *reinterpret_cast<pack<T, V>*>(p) = t;
}
// V weights; without any the pointer is some readable row of the same length, and the values are not used
template <int V, typename W> __device__ __forceinline__ void load_w(const void* w, bool has, int d, float* v, float none) {
    load_v<V>(static_cast<const W*>(w) + d, v);
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = has ? v[j] : none;
}

// A lane's V values of a row of D in chunk c.  Where the row ends inside them they are its last V instead: the first `skip`
// belong to the lane before, which does the same with them and stores the same, so only the row's sums leave them out.
template <int V> struct Place {
    int d, skip;   // first column, values that are another lane's (all of them behind the row's end)
    bool whole;    // nobody skips any: the same for all lanes
    __device__ __forceinline__ Place(int lane, int tpr, int c, int D) {
        const int at = (lane + c * tpr) * V;
        whole = (c + 1) * tpr * V <= D;
        d = whole ? at : min(at, D - V);
        skip = whole ? 0 : at - d;
    }
    __device__ __forceinline__ bool here() const { return whole || skip < V; }
};

// a block's sum of column d (pass 0: dw, 1: db)
template <typename T, typename P> __device__ __forceinline__ void put_column(const LnArgs& a, int pass, int d, P sum) {
    if (a.part) {
        static_cast<P*>(a.part)[((int64_t)blockIdx.x * 2 + pass) * a.D + d] = sum;
        return;
    }
    const float v = (float)sum;
    void* out = pass ? a.db : a.dw;
    if (!out) return;
    if (a.cf32) static_cast<float*>(out)[d] = v;
    else static_cast<T*>(out)[d] = (T)v;
}

// v of this lane and of the one at 2^LEVEL lanes' distance, in every lane; below LEVEL all lanes hold the same sums, so
// mirrored lanes serve for distances 4 and 8.  Within the registers: a sum over a wave through LDS (shuffles) waits for it
// six times, and a row has three of them on its way from its values to its result.
template <int LEVEL> __device__ __forceinline__ float pair_sum(float v) {
    if constexpr (LEVEL < 4) {
        constexpr int ctrl = LEVEL == 0 ? 0xb1 : LEVEL == 1 ? 0x4e : LEVEL == 2 ? 0x141 : 0x140;
        return v + __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), ctrl, 0xf, 0xf, true));
    } else {
        const unsigned u = __float_as_uint(v);
        const auto t = [&] {
            if constexpr (LEVEL == 4) return __builtin_amdgcn_permlane16_swap(u, u, false, false);
            else return __builtin_amdgcn_permlane32_swap(u, u, false, false);
        }();
        return __uint_as_float(t[0]) + __uint_as_float(t[1]);
    }
}
// sums over groups of n lanes, a power of two (ALL: 2^TOP)
template <bool ALL, int N, int TOP = 6, int LEVEL = 0> __device__ __forceinline__ void lane_sum(float (&v)[N], int n) {
    if constexpr (LEVEL < TOP) {
        if (ALL || n > 1 << LEVEL) {
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = pair_sum<LEVEL>(v[i]);
            lane_sum<ALL, N, TOP, LEVEL + 1>(v, n);
        }
    }
}

// sums over the lanes of a row: tpr lanes of a wave (WHOLE: all of them), or (BLOCK) all waves of the block through `red` with one barrier; the
// caller alternates between two `red` buffers, so a buffer is rewritten only behind the other's barrier
template <bool BLOCK, bool WHOLE, int N> __device__ __forceinline__ void row_sum(float (&v)[N], int tpr, float (*red)[16]) {
    lane_sum<WHOLE, N>(v, tpr);
    if constexpr (BLOCK) {
        if ((threadIdx.x & 63) == 0) {
#pragma unroll
            for (int i = 0; i < N; ++i) red[i][threadIdx.x >> 6] = v[i];
        }
        __syncthreads();
        // (a lane to a wave: a loop over the waves waits for LDS at each)
        const int w = threadIdx.x & 15;
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = w < tpr / 64 ? red[i][w] : 0.f;
        lane_sum<true, N, 4>(v, 16);
    }
}

// A block goes from row to row: the next row is on its way while this one is summed, and the weights stay in registers
// (read again per row they are as many bytes from L2 as the row itself).
template <typename T, int V, int E, bool BLOCK>
__global__ __launch_bounds__(BLOCK ? 1024 : 256) void ln_fwd_kernel(LnArgs a) {
    constexpr int NC = E / V;
    constexpr bool KEEP = E <= 16, AHEAD = KEEP;  // (what the registers of 1024 threads hold)
    constexpr bool WHOLE = BLOCK || E > V;        // (as ln_pick chooses)
    __shared__ float red[2][2][16];
    const int tpr = BLOCK ? (int)blockDim.x : a.tpr;
    const int lane = BLOCK ? (int)threadIdx.x : (int)(threadIdx.x & (unsigned)(tpr - 1));
    const int64_t rpb = BLOCK ? 1 : 256 / tpr, stride = gridDim.x * rpb;
    const float invd = 1.f / (float)a.D;
    float w[KEEP ? NC : 1][V], b[KEEP ? NC : 1][V];
    const auto weights = [&](int c, float* wv, float* bv) {
        const int d = Place<V>(lane, tpr, c, a.D).d;
        if (a.wf32) {
            load_w<V, float>(a.w, a.hw, d, wv, 1.f);
            load_w<V, float>(a.b, a.hb, d, bv, 0.f);
        } else {
            load_w<V, T>(a.w, a.hw, d, wv, 1.f);
            load_w<V, T>(a.b, a.hb, d, bv, 0.f);
        }
    };
    const auto fetch = [&](int64_t r, pack<T, V> (&raw)[NC]) {
        const T* x = static_cast<const T*>(a.x) + (r < a.rows ? r : 0) * a.xs;
#pragma unroll
        for (int c = 0; c < NC; ++c) raw[c] = load_raw<V>(x + Place<V>(lane, tpr, c, a.D).d);
    };
    int par = 0;
    int64_t r = (int64_t)blockIdx.x * rpb + (BLOCK ? 0 : (int)(threadIdx.x / (unsigned)tpr));
    pack<T, V> next[NC];
    if constexpr (AHEAD) fetch(r, next);
    if constexpr (KEEP) {
#pragma unroll
        for (int c = 0; c < NC; ++c) weights(c, w[c], b[c]);
    }
    for (int64_t r0 = (int64_t)blockIdx.x * rpb; r0 < a.rows; r0 += stride, r += stride) {
        float v[NC][V];
        float m[1] = {0.f};
        if constexpr (!AHEAD) fetch(r, next);
#pragma unroll
        for (int c = 0; c < NC; ++c) widen<T, V>(next[c], v[c]);
        if (AHEAD && r0 + stride < a.rows) fetch(r + stride, next);
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const Place<V> at(lane, tpr, c, a.D);
            if (at.whole) {
#pragma unroll
                for (int j = 0; j < V; ++j) m[0] = fmaf(v[c][j], invd, m[0]);  // (a sum of x could overflow)
            } else {
#pragma unroll
                for (int j = 0; j < V; ++j) m[0] = fmaf(j >= at.skip ? v[c][j] : 0.f, invd, m[0]);
            }
        }
        row_sum<BLOCK, WHOLE, 1>(m, tpr, red[par]);
        par ^= 1;
        float mean = m[0], e, var;
        // from deviations so far, those from a mean `shift` further -> whether that one is far from theirs
        const auto deviate = [&](float shift) {
            float s[2] = {0.f, 0.f};
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                const Place<V> at(lane, tpr, c, a.D);
#pragma unroll
                for (int j = 0; j < V; ++j) v[c][j] -= shift;
                if (at.whole) {
#pragma unroll
                    for (int j = 0; j < V; ++j) {
                        s[0] += v[c][j];
                        s[1] = fmaf(v[c][j], v[c][j], s[1]);
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < V; ++j) {
                        const float d = j >= at.skip ? v[c][j] : 0.f;
                        s[0] += d;
                        s[1] = fmaf(d, d, s[1]);
                    }
                }
            }
            row_sum<BLOCK, WHOLE, 2>(s, tpr, red[par]);
            par ^= 1;
            e = s[0] * invd;
            const float sq = s[1] * invd;
            var = sq < INFINITY ? fmaxf(sq - e * e, 0.f) : sq;  // (NaN stays NaN)
            return !(4.f * e * e <= sq && sq < INFINITY);
        };
        bool far = deviate(mean);
#pragma unroll 1
        for (int turn = 0; turn < 2 && (BLOCK ? far : __any(far)); ++turn) {  // (the same for a row's, and a wave's, lanes)
            const float to = far ? mean + e : mean, shift = to - mean;
            mean = to;
            far = deviate(shift);
        }
        const float rstd = 1.f / sqrtf(var + a.eps);
        if (r >= a.rows) continue;  // (a whole sub-wave row; the others of its wave go on)
        T* y = static_cast<T*>(a.y) + r * a.D;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const int k = KEEP ? c : 0;
            if constexpr (!KEEP) weights(c, w[0], b[0]);
#pragma unroll
            for (int j = 0; j < V; ++j) v[c][j] = fmaf((v[c][j] - e) * rstd, w[k][j], b[k][j]);
            const Place<V> at(lane, tpr, c, a.D);
            if (at.here()) store_v<V>(y + at.d, v[c]);
            if constexpr (!KEEP)  // (few weights in flight, or the registers spill)
                if (c % 4 == 3) asm volatile("" ::: "memory");
        }
        if (a.stat && lane == 0) a.stat[r] = make_float2(mean + e, rstd);
    }
}

template <typename T, int V, int E, bool BLOCK>
__global__ __launch_bounds__(BLOCK ? 1024 : 256) void ln_bwd_kernel(LnArgs a) {
    constexpr int NC = E / V;
    constexpr bool AHEAD = E <= 8 || sizeof(T) == 2;  // (16 float32 values a thread leave no registers for the next row,
    constexpr bool KEEP = E <= 8 || (AHEAD && !BLOCK);  // of 16 bits none for the weights in blocks of 1024 threads)
    constexpr bool WHOLE = BLOCK || E > V;
    __shared__ float red[2][2][16];
    extern __shared__ __attribute__((aligned(16))) float cols[];  // sub-wave rows: [4 waves][D] of dw, then of db
    const int tpr = BLOCK ? (int)blockDim.x : a.tpr;
    const int lane = BLOCK ? (int)threadIdx.x : (int)(threadIdx.x & (unsigned)(tpr - 1));
    const int64_t rpb = BLOCK ? 1 : 256 / tpr, stride = gridDim.x * rpb;
    const float invd = 1.f / (float)a.D;
    int64_t r = (int64_t)blockIdx.x * rpb + (BLOCK ? 0 : (int)(threadIdx.x / (unsigned)tpr));
    pack<T, V> nx[NC], ng[NC];
    float2 nst;
    const auto fetch = [&](int64_t row) {
        const int64_t q = row < a.rows ? row : 0;
        const T* x = static_cast<const T*>(a.x) + q * a.xs;
        const T* dy = static_cast<const T*>(a.dy) + q * a.dys;
        nst = a.stat[q];
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const int d = Place<V>(lane, tpr, c, a.D).d;
            nx[c] = load_raw<V>(x + d);
            ng[c] = load_raw<V>(dy + d);
        }
    };
    if constexpr (AHEAD) fetch(r);
    float sw[NC][V], sb[NC][V], w[KEEP ? NC : 1][V];
    const auto weight = [&](int c, float* wv) {
        const int d = Place<V>(lane, tpr, c, a.D).d;
        if (a.wf32) load_w<V, float>(a.w, a.hw, d, wv, 1.f);
        else load_w<V, T>(a.w, a.hw, d, wv, 1.f);
    };
#pragma unroll
    for (int c = 0; c < NC; ++c) {
#pragma unroll
        for (int j = 0; j < V; ++j) sw[c][j] = sb[c][j] = 0.f;
        if constexpr (KEEP) weight(c, w[c]);
    }
    int par = 0;
    for (int64_t r0 = (int64_t)blockIdx.x * rpb; r0 < a.rows; r0 += stride, r += stride) {
        const bool on = r < a.rows;
        if constexpr (!AHEAD) fetch(r);
        const float2 st = nst;
        float xh[NC][V], g[NC][V];
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            if (on) {
                widen<T, V>(nx[c], xh[c]);
                widen<T, V>(ng[c], g[c]);
            } else {
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    xh[c][j] = st.x;
                    g[c][j] = 0.f;
                }
            }
        }
        if (AHEAD && r0 + stride < a.rows) fetch(r + stride);
        float s[2] = {0.f, 0.f};
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const int k = KEEP ? c : 0;
            if constexpr (!KEEP) weight(c, w[0]);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                xh[c][j] = (xh[c][j] - st.x) * st.y;
                sb[c][j] += g[c][j];
                sw[c][j] = fmaf(g[c][j], xh[c][j], sw[c][j]);
                g[c][j] *= w[k][j];
            }
            const Place<V> at(lane, tpr, c, a.D);
            if (at.whole) {
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    s[0] += g[c][j];
                    s[1] = fmaf(g[c][j], xh[c][j], s[1]);
                }
            } else {
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    s[0] += j >= at.skip ? g[c][j] : 0.f;
                    s[1] += j >= at.skip ? g[c][j] * xh[c][j] : 0.f;
                }
            }
        }
        if (!a.dx) continue;  // (the same for the whole grid)
        row_sum<BLOCK, WHOLE, 2>(s, tpr, red[par]);
        par ^= 1;
        const float c1 = s[0] * invd, c2 = s[1] * invd;
        if (!on) continue;
        T* dx = static_cast<T*>(a.dx) + r * a.D;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
#pragma unroll
            for (int j = 0; j < V; ++j) g[c][j] = st.y * (g[c][j] - fmaf(xh[c][j], c2, c1));
            const Place<V> at(lane, tpr, c, a.D);
            if (at.here()) store_v<V>(dx + at.d, g[c]);
        }
    }
    if (!a.cols) return;
    if constexpr (BLOCK) {
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const Place<V> at(lane, tpr, c, a.D);
            if (at.here()) {
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    put_column<T>(a, 0, at.d + j, sw[c][j]);
                    put_column<T>(a, 1, at.d + j, sb[c][j]);
                }
            }
        }
    } else {
        // the wave's rows, then the block's four waves, in lane and wave order
        float* cw = cols + (threadIdx.x >> 6) * a.D;
#pragma unroll
        for (int pass = 0; pass < 2; ++pass) {
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                const Place<V> at(lane, tpr, c, a.D);
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    float t = pass ? sb[c][j] : sw[c][j];
                    for (int o = tpr; o < 64; o <<= 1) t += __shfl_xor(t, o, 64);
                    if ((threadIdx.x & 63) < (unsigned)tpr && at.here()) cw[at.d + j] = t;
                }
            }
            __syncthreads();
            for (int d = threadIdx.x; d < a.D; d += 256)
                put_column<T>(a, pass, d, (cols[d] + cols[a.D + d]) + (cols[2 * a.D + d] + cols[3 * a.D + d]));
            __syncthreads();
        }
    }
}

// Rows of up to 32 values in 64 bits, one value per lane (tpr = the power of two at or above D).
template <typename T, bool BWD> __global__ __launch_bounds__(256) void ln_narrow_kernel(LnArgs a) {
    __shared__ double cols[4][LN_NARROW];
    const int tpr = a.tpr, d = threadIdx.x & (tpr - 1), rpb = 256 / tpr;
    const bool in = d < a.D;
    float wf[1] = {0.f}, bf[1] = {0.f};
    if (in) {
        if (a.wf32) {
            load_w<1, float>(a.w, a.hw, d, wf, 1.f);
            load_w<1, float>(a.b, a.hb, d, bf, 0.f);
        } else {
            load_w<1, T>(a.w, a.hw, d, wf, 1.f);
            load_w<1, T>(a.b, a.hb, d, bf, 0.f);
        }
    }
    double sw = 0., sb = 0.;
    for (int64_t r0 = (int64_t)blockIdx.x * rpb; r0 < a.rows; r0 += (int64_t)gridDim.x * rpb) {
        const int64_t r = r0 + (int)(threadIdx.x / (unsigned)tpr);
        const bool on = in && r < a.rows;
        const double x = on ? (double)(float)static_cast<const T*>(a.x)[r * a.xs + d] : 0.;
        double s = x;
        for (int o = tpr >> 1; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
        const double u = on ? x - s / a.D : 0.;
        s = u * u;
        for (int o = tpr >> 1; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
        const double rstd = 1. / sqrt(s / a.D + (double)a.eps), xh = u * rstd;
        if constexpr (!BWD) {
            if (on) static_cast<T*>(a.y)[r * a.D + d] = (T)(float)(xh * wf[0] + bf[0]);
        } else {
            const double dy = on ? (double)(float)static_cast<const T*>(a.dy)[r * a.dys + d] : 0.;
            sb += dy;
            sw += dy * xh;
            const double g = dy * wf[0];
            double c1 = g, c2 = g * xh;
            for (int o = tpr >> 1; o > 0; o >>= 1) {
                c1 += __shfl_xor(c1, o, 64);
                c2 += __shfl_xor(c2, o, 64);
            }
            if (on && a.dx) static_cast<T*>(a.dx)[r * a.D + d] = (T)(float)(rstd * (g - c1 / a.D - xh * (c2 / a.D)));
        }
    }
    if constexpr (BWD) {
        if (!a.cols) return;
#pragma unroll
        for (int pass = 0; pass < 2; ++pass) {
            double t = pass ? sb : sw;
            for (int o = tpr; o < 64; o <<= 1) t += __shfl_xor(t, o, 64);
            if ((threadIdx.x & 63) < (unsigned)tpr && in) cols[threadIdx.x >> 6][d] = t;
            __syncthreads();
            if (threadIdx.x < (unsigned)a.D)
                put_column<T>(a, pass, threadIdx.x, (cols[0][threadIdx.x] + cols[1][threadIdx.x]) +
                                                        (cols[2][threadIdx.x] + cols[3][threadIdx.x]));
            __syncthreads();
        }
    }
}

// The backward of rows that no block holds in registers (behind 16384 values): read again for each sum, from L2, where a
// row stays meanwhile.
template <typename T> __global__ __launch_bounds__(1024) void ln_long_bwd_kernel(LnArgs a) {
    __shared__ float red[2][2][16];
    const float invd = 1.f / (float)a.D;
    int par = 0;
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const T* x = static_cast<const T*>(a.x) + r * a.xs;
        const T* dy = static_cast<const T*>(a.dy) + r * a.dys;
        const float2 st = a.stat[r];
        const auto go = [&](auto kind) {
            using W = decltype(kind);
            float s[2] = {0.f, 0.f};
#pragma unroll 4
            for (int d = threadIdx.x; d < a.D; d += 1024) {
                float w[1];
                load_w<1, W>(a.w, a.hw, d, w, 1.f);
                const float g = (float)dy[d] * w[0];
                s[0] += g;
                s[1] = fmaf(g, ((float)x[d] - st.x) * st.y, s[1]);
            }
            row_sum<true, true, 2>(s, 1024, red[par]);
            const float c1 = s[0] * invd, c2 = s[1] * invd;
            T* dx = static_cast<T*>(a.dx) + r * a.D;
#pragma unroll 4
            for (int d = threadIdx.x; d < a.D; d += 1024) {
                float w[1];
                load_w<1, W>(a.w, a.hw, d, w, 1.f);
                const float xh = ((float)x[d] - st.x) * st.y;
                dx[d] = (T)(st.y * ((float)dy[d] * w[0] - fmaf(xh, c2, c1)));
            }
        };
        if (a.wf32) go(float());
        else go(T());
        par ^= 1;
    }
}
// their partial dw, db: a thread owns a column, a block a slab of rows
template <typename T> __global__ __launch_bounds__(256) void ln_long_cols_kernel(LnArgs a, int64_t slab) {
    const int d = blockIdx.x * 256 + threadIdx.x;
    if (d >= a.D) return;
    const int64_t r0 = blockIdx.y * slab, r1 = r0 + slab < a.rows ? r0 + slab : a.rows;
    float sw = 0.f, sb = 0.f;
    for (int64_t r = r0; r < r1; ++r) {
        const float2 st = a.stat[r];
        const float g = (float)static_cast<const T*>(a.dy)[r * a.dys + d];
        sb += g;
        sw = fmaf(g, ((float)static_cast<const T*>(a.x)[r * a.xs + d] - st.x) * st.y, sw);
    }
    float* pw = static_cast<float*>(a.part) + (int64_t)blockIdx.y * 2 * a.D;
    pw[d] = sw;
    pw[a.D + d] = sb;
}

// dw, db from the blocks' partials: 32 columns x 32 slices of blocks per thread block, summed in slice order, in 64 bits (in
// 32 they were the larger part of the error: dw and db of 4096 x 128 1.2 times a cascaded sum's, up to 1.5)
template <typename T, typename P> __global__ __launch_bounds__(1024) void ln_cols_kernel(const P* __restrict__ part, int nblk, int D,
                                                                                         T* __restrict__ dw, T* __restrict__ db) {
    __shared__ double red[32][33];
    const int c = threadIdx.x & 31, sl = threadIdx.x >> 5;
    const int64_t col = (int64_t)blockIdx.x * 32 + c;  // of 2 D
    double s = 0.;
    if (col < 2 * (int64_t)D)
        for (int k = sl; k < nblk; k += 32) s += part[(int64_t)k * 2 * D + col];
    red[sl][c] = s;
    __syncthreads();
    if (sl == 0 && col < 2 * (int64_t)D) {
        s = 0.;
#pragma unroll
        for (int k = 0; k < 32; ++k) s += red[k][c];
        T* out = col < D ? dw : db;
        if (out) out[col < D ? col : col - D] = (T)(float)s;
    }
}

// ---------------------------------------------------------------- host
struct LnPick {
    int tpr, ept;   // lanes of a row, values of a lane
    bool block;     // a block per row (tpr threads), else rows within waves
};

// Rows within a wave up to 64 lanes of 16 values; behind that a block per row, of as many waves as leave 8 values to a
// thread while that is up to 1024 threads, 16 up to 1024, then 32.  The forward in 16 bits goes on with 16 values behind 512
// threads, fewer waves to meet: 16384 rows of 5120 bfloat16 values 63 us, 77 with 8 a thread; its backward has no registers
// to keep twice the sums and the next row: 114 us with 16, 98 with 8 (float32 alike: 4100 values 161 and 146).
LnPick ln_pick(int D, int V, bool bwd) {
    if (D <= 64 * V) {
        LnPick p{64, V, false};
        while (p.tpr > 1 && (p.tpr / 2) * V >= D) p.tpr /= 2;
        return p;
    }
    for (int e = 8; e <= 16; e *= 2)
        if (e >= V && D <= 64 * e) return {64, e, false};
    const auto threads = [&](int e) { return ((D + e - 1) / e + 63) / 64 * 64; };
    if (threads(8) <= (V > 4 && !bwd ? 512 : 1024)) return {threads(8), 8, true};
    if (threads(16) <= 1024) return {threads(16), 16, true};
    return {threads(32), 32, true};
}

int64_t ln_rows_per_block(int D, int V, bool bwd) {
    if (D <= LN_NARROW) {
        int tpr = 1;
        while (tpr < D) tpr *= 2;
        return 256 / tpr;
    }
    const LnPick p = ln_pick(D, V, bwd);
    return p.block ? 1 : 256 / p.tpr;
}

// as many blocks as give every block the same number of passes over rows, `most` or fewer
int ln_even(int64_t passes, int64_t most) {
    const int64_t each = (passes + most - 1) / most;
    return (int)((passes + each - 1) / each);
}

// The forward keeps 1536 threads of a CU busy.  The backward's partial sums are 8 D bytes per block, written and read
// once, next to the rows' own 3 tensors: two blocks a CU, one from 513 threads on, and no block with fewer than 4 passes
// (backward of 1003 x 1537 in bfloat16 with 8, 4 and 2: 12.8, 12.8 and 17.5 us; 4096 x 128 in float32 10.1, 9.0 and 9.3).
// us with 1 / 2 / 3 / 4 blocks a CU, 256 threads each: 65536 x 128 float32 33.3 / 27.8 / 28.0 / 30.0,
// 65536 x 512 80.6 / 82.6 / 86.0 / 89.6, 131072 x 256 112 / 81 / 83 / 87, 262144 x 128 bfloat16 59 / 46 / 45 / 47.
int ln_fwd_blocks(int64_t rows, int D, int V) {
    const int64_t rpb = ln_rows_per_block(D, V, false), passes = (rows + rpb - 1) / rpb;
    const int threads = D > LN_NARROW && ln_pick(D, V, false).block ? ln_pick(D, V, false).tpr : 256;
    return ln_even(passes, (int64_t)num_cus() * std::max(1, 1536 / threads));
}
int ln_bwd_blocks(int64_t rows, int D, int V) {
    const int64_t rpb = ln_rows_per_block(D, V, true), passes = (rows + rpb - 1) / rpb;
    const int threads = D > LN_NARROW && ln_pick(D, V, true).block ? ln_pick(D, V, true).tpr : 256;
    return ln_even(passes, std::max<int64_t>(1, std::min<int64_t>((int64_t)num_cus() * (threads > 512 ? 1 : 2), (passes + 3) / 4)));
}

template <typename T, int V, int E, bool BLOCK, bool BWD> int ln_go(const LnArgs& a, int blocks, hipStream_t s) {
    const int threads = BLOCK ? a.tpr : 256;
    if constexpr (BWD) {
        const size_t sm = !BLOCK && a.cols ? (size_t)4 * a.D * sizeof(float) : 0;
        ln_bwd_kernel<T, V, E, BLOCK><<<blocks, threads, sm, s>>>(a);
        PCX_LAUNCH_CHECK("ln_bwd_kernel");
    } else {
        ln_fwd_kernel<T, V, E, BLOCK><<<blocks, threads, 0, s>>>(a);
        PCX_LAUNCH_CHECK("ln_fwd_kernel");
    }
    return PCX_OK;
}

template <typename T> int ln_long_bwd(const LnArgs& a, int blocks, hipStream_t s) {
    if (a.cols) {
        const int64_t slab = (a.rows + blocks - 1) / blocks;
        ln_long_cols_kernel<T><<<dim3((unsigned)ceil_div(a.D, 256), (unsigned)blocks), 256, 0, s>>>(a, slab);
        PCX_LAUNCH_CHECK("ln_long_cols_kernel");
    }
    if (!a.dx) return PCX_OK;
    ln_long_bwd_kernel<T><<<(unsigned)std::min<int64_t>(a.rows, 1 << 20), 1024, 0, s>>>(a);
    PCX_LAUNCH_CHECK("ln_long_bwd_kernel");
    return PCX_OK;
}

template <typename T, bool BWD> int ln_run(LnArgs a, int blocks, hipStream_t s) {
    constexpr int V = 16 / (int)sizeof(T);
    if (a.D <= LN_NARROW) {
        a.tpr = 1;
        while (a.tpr < a.D) a.tpr *= 2;
        ln_narrow_kernel<T, BWD><<<blocks, 256, 0, s>>>(a);
        PCX_LAUNCH_CHECK("ln_narrow_kernel");
        return PCX_OK;
    }
    const LnPick p = ln_pick(a.D, V, BWD);
    a.tpr = p.tpr;
    if (!p.block) {
        if (p.ept == V) return ln_go<T, V, V, false, BWD>(a, blocks, s);
        if constexpr (V < 8)
            if (p.ept == 8) return ln_go<T, V, 8, false, BWD>(a, blocks, s);
        return ln_go<T, V, 16, false, BWD>(a, blocks, s);
    }
    if (p.ept == 8) return ln_go<T, V, 8, true, BWD>(a, blocks, s);
    if (p.ept == 16) return ln_go<T, V, 16, true, BWD>(a, blocks, s);
    if constexpr (BWD) return ln_long_bwd<T>(a, blocks, s);
    else return ln_go<T, V, 32, true, false>(a, blocks, s);
}
template <bool BWD> int ln_any(const LnArgs& a, int dtype, int blocks, hipStream_t s) {
    if (dtype == PCX_F32) return ln_run<float, BWD>(a, blocks, s);
    if (dtype == PCX_BF16) return ln_run<bf16, BWD>(a, blocks, s);
    return ln_run<f16, BWD>(a, blocks, s);
}

int ln_dtype_size(int dtype) { return dtype == PCX_F32 ? 4 : dtype == PCX_BF16 || dtype == PCX_F16 ? 2 : 0; }

}  // namespace

size_t layernorm_bwd_ws(int64_t rows, int D, int es) {
    if (rows <= 0 || D <= 0) return 0;
    const int n = ln_bwd_blocks(rows, D, 16 / es);
    return n > 1 || D > LN_ALONE ? (size_t)n * 2 * D * (D <= LN_NARROW ? sizeof(double) : sizeof(float)) : 0;
}

LnArgs ln_args(const LayerNormArgs& q) {
    LnArgs a{};
    a.rows = q.rows;
    a.D = q.D;
    a.eps = q.eps;
    a.x = q.x;
    a.xs = q.xs;
    a.hw = q.w != nullptr;
    a.hb = q.b != nullptr;
    a.wf32 = (a.hw || a.hb) && q.wdtype == PCX_F32;
    a.w = q.w ? q.w : q.b ? q.b : q.x;
    a.b = q.b ? q.b : a.w;
    a.y = q.y;
    a.stat = reinterpret_cast<float2*>(q.stat);
    a.dy = q.dy;
    a.dys = q.dys;
    a.dx = q.dx;
    return a;
}

int launch_layernorm_fwd(const LayerNormArgs& q, hipStream_t s) {
    const LnArgs a = ln_args(q);
    return ln_any<false>(a, q.dtype, ln_fwd_blocks(a.rows, a.D, 16 / ln_dtype_size(q.dtype)), s);
}

int launch_layernorm_bwd(const LayerNormArgs& q, hipStream_t s) {
    LnArgs a = ln_args(q);
    a.cols = q.dw || q.db;
    a.dw = q.dw;
    a.db = q.db;
    a.cf32 = q.wdtype == PCX_F32;
    const int blocks = ln_bwd_blocks(a.rows, a.D, 16 / ln_dtype_size(q.dtype));
    if (blocks > 1 || a.D > LN_ALONE) a.part = q.ws;
    const int rc = ln_any<true>(a, q.dtype, blocks, s);
    if (rc || !a.cols || !a.part) return rc;
    const int cb = ceil_div(2 * (int64_t)a.D, 32);
    const auto join = [&](auto kind) {
        using T = decltype(kind);
        T *dw = static_cast<T*>(q.dw), *db = static_cast<T*>(q.db);
        if (a.D <= LN_NARROW) ln_cols_kernel<T, double><<<cb, 1024, 0, s>>>(static_cast<const double*>(a.part), blocks, a.D, dw, db);
        else ln_cols_kernel<T, float><<<cb, 1024, 0, s>>>(static_cast<const float*>(a.part), blocks, a.D, dw, db);
    };
    if (q.wdtype == PCX_F32) join(float());
    else if (q.wdtype == PCX_BF16) join(bf16());
    else join(f16());
    PCX_LAUNCH_CHECK("ln_cols_kernel");
    return PCX_OK;
}

}  // namespace pcx

using namespace pcx;

static int ln_check(const char* what, int dtype, int wdtype, int64_t rows, int64_t D, int64_t xs, float eps) {
    PCX_CHECK_ARG(ln_dtype_size(dtype) != 0, "%s: unknown element type %d", what, dtype);
    PCX_CHECK_ARG(wdtype == dtype || wdtype == PCX_F32, "%s: weight and bias must have the input's type or be float32", what);
    PCX_CHECK_ARG(rows >= 0 && D >= 1 && D <= LN_MAX, "%s: rows of 1 to %d values supported (got %lld x %lld)", what, LN_MAX,
                  (long long)rows, (long long)D);
    PCX_CHECK_ARG(xs >= D || rows <= 1, "%s: row stride %lld below the row length %lld", what, (long long)xs, (long long)D);
    PCX_CHECK_ARG(eps > 0.f && eps < 1e30f, "%s: eps must be positive (got %g)", what, (double)eps);
    return PCX_OK;
}

extern "C" size_t pcx_layernorm_workspace_bytes(int dtype, int64_t rows, int64_t D) {
    const int es = ln_dtype_size(dtype);
    if (!es || rows < 0 || D < 1 || D > LN_MAX) return 0;
    return layernorm_bwd_ws(rows, (int)D, es);
}

extern "C" int pcx_layernorm_forward(int dtype, int wdtype, int64_t rows, int64_t D, const void* x, int64_t x_stride,
                                     const void* w, const void* b, float eps, void* y, float* stats, hipStream_t stream) {
    int rc = ln_check("layernorm_forward", dtype, wdtype, rows, D, x_stride, eps);
    if (rc) return rc;
    if (rows == 0) return PCX_OK;
    PCX_CHECK_ARG(x && y, "layernorm_forward: NULL buffer");
    LayerNormArgs q{};
    q.dtype = dtype; q.wdtype = wdtype; q.rows = rows; q.D = (int)D; q.eps = eps;
    q.x = x; q.xs = x_stride; q.w = w; q.b = b; q.y = y; q.stat = stats;
    return launch_layernorm_fwd(q, stream);
}

extern "C" int pcx_layernorm_backward(int dtype, int wdtype, int64_t rows, int64_t D, const void* x, int64_t x_stride,
                                      const void* w, float eps, const float* stats, const void* dy, int64_t dy_stride,
                                      void* dx, void* dw, void* db, void* ws, size_t ws_bytes, hipStream_t stream) {
    int rc = ln_check("layernorm_backward", dtype, wdtype, rows, D, x_stride, eps);
    if (rc) return rc;
    PCX_CHECK_ARG(dy_stride >= D || rows <= 1, "layernorm_backward: gradient row stride below the row length");
    PCX_CHECK_ARG(rows >= 1, "layernorm_backward: no rows");
    PCX_CHECK_ARG(x && dy && stats, "layernorm_backward: NULL buffer");
    if (!dx && !dw && !db) return PCX_OK;
    const size_t need = pcx_layernorm_workspace_bytes(dtype, rows, D);
    if ((dw || db) && need && (!ws || ws_bytes < need)) {
        set_error("layernorm_backward: workspace of %zu bytes, %zu needed", ws_bytes, need);
        return PCX_EWORKSPACE;
    }
    LayerNormArgs q{};
    q.dtype = dtype; q.wdtype = wdtype; q.rows = rows; q.D = (int)D; q.eps = eps;
    q.x = x; q.xs = x_stride; q.w = w; q.stat = const_cast<float*>(stats); q.dy = dy; q.dys = dy_stride;
    q.dx = dx; q.dw = dw; q.db = db; q.ws = ws;
    return launch_layernorm_bwd(q, stream);
}
