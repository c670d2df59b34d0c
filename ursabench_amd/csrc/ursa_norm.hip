// ursa_norm.hip — K16: layer norm (forward, backward with the weight's gradient, the residual sum in front of it) and K17: an
// activation in 8 bits and back.
//
//   z = x (+ r, rounded to the tensors' type: what the caller keeps is what is normalised)
//   mean = (sum_d z_d) / D ; var = (sum_d (z_d - mean)^2) / D ; rstd = 1 / sqrt(var + eps) ; xhat = (z - mean) rstd
//   the mean's own rounding (its sum's, and the division's) would move every xhat of the row the same way, in rows far from zero by more
//   than their deviation: with m the mean as it comes out, rest = (sum_d (z_d - m)) / D, mean = m + rest, xhat = ((z - m) - rest) rstd and
//   var = (sum_d (z_d - m)^2) / D - rest^2. The backward pass has that mean rounded once, to fp32.
//   y = xhat gamma + beta
//   t = dy gamma ; dx = rstd (t - (sum_d t) / D - xhat (sum_d t xhat) / D) (+ dz) ; dgamma = sum_rows dy xhat ; dbeta = sum_rows dy
//
// What bounds it: memory. Each row is read once into registers and both sums of the forward (the mean, then the squares around
// it: no cancellation) and of the backward run over the registers; statistics, sums and the accumulators of dgamma / dbeta are
// fp32. A row belongs to TPR threads (16 for the narrowest, so that a wave holds four rows; one wave; one workgroup), CV values
// per thread. dgamma / dbeta: a workgroup walks rows with a fixed stride and keeps its columns' sums in registers, stores them
// once, and a second launch adds the workgroups' sums in a fixed order - no atomics, the same bits every time.
// 16,384 x 4,096 bf16: the sum and its norm 108 us (537 MB, 5.0 TB/s), backward with a gradient past the norm 135 us (4.0 TB/s; a
// large copy moves 4.8). One row: the launch, 5 us up to 16,384 features. A longer one does not fit a workgroup's registers and is
// walked three times (twice) by one workgroup: 20,000 features 12 us forward and 21 backward, 2^20 417 and 707; 512 rows of 2^17
// bf16 121 and 290 us (dgamma / dbeta 82 of them).
#include "ursa_ops.h"

namespace {

using namespace ursa;

// sum over the TPR threads of a row; `red`: 2 x 16 floats of LDS for TPR > 64 (two slots: consecutive sums need one barrier each)
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float* red, int slot) {
#pragma unroll
    for (int o = (TPR < 64 ? TPR : 64) / 2; o > 0; o >>= 1) v += __shfl_xor(v, o);
    if constexpr (TPR > 64) {
        float* r = red + slot * 16;
        if ((threadIdx.x & 63) == 0) r[threadIdx.x >> 6] = v;
        __syncthreads();
        v = r[0];
#pragma unroll
        for (int w = 1; w < TPR / 64; ++w) v += r[w];
    }
    return v;
}

// two sums over a row at once, in the slots behind that of row_sum's slot 0: 3 x 16 floats of LDS
template <int TPR>
__device__ __forceinline__ float2 row_sums(float a, float b, float* red) {
#pragma unroll
    for (int o = (TPR < 64 ? TPR : 64) / 2; o > 0; o >>= 1) a += __shfl_xor(a, o), b += __shfl_xor(b, o);
    if constexpr (TPR > 64) {
        if ((threadIdx.x & 63) == 0) red[16 + (threadIdx.x >> 6)] = a, red[32 + (threadIdx.x >> 6)] = b;
        __syncthreads();
        a = red[16], b = red[32];
#pragma unroll
        for (int w = 1; w < TPR / 64; ++w) a += red[16 + w], b += red[32 + w];
    }
    return make_float2(a, b);
}

// 1 / sqrt of the variance around m + rest; rounding may leave a constant row's below zero. Past the range it is infinite (rest^2 may
// be, too), and a NaN stays one.
__device__ __forceinline__ float inverse_deviation(float mean_square, float rest, float eps) {
    const float var = mean_square < INFINITY ? mean_square - rest * rest : mean_square;
    return 1.f / sqrtf((var < 0.f ? 0.f : var) + eps);
}

// the exponent byte of this thread's block of 32 (V values here, the rest in the neighbouring 32 / V - 1 threads)
template <typename T, int V>
__device__ __forceinline__ int block_exponent(const float (&v)[V]) {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < V; ++i) { const uint32_t b = magnitude_bits(v[i]); top = b > top ? b : top; }
#pragma unroll
    for (int o = 1; o < kBlock8 / V; o <<= 1) { const uint32_t b = (uint32_t)__shfl_xor((int)top, o); top = b > top ? b : top; }
    return exponent8<T>(top);
}

template <int V>
__device__ __forceinline__ void store_q(int8_t* __restrict__ p, const float (&v)[V], int e) {
    int8_t t[V];
#pragma unroll
    for (int i = 0; i < V; ++i) t[i] = (int8_t)quantise8(v[i], e);
    __builtin_memcpy(p, t, sizeof t);                        // q rows are padded to whole blocks: always in range
}

template <int V>
__device__ __forceinline__ void load_q(const int8_t* __restrict__ p, int e, float (&v)[V]) {
    int8_t t[V];
    __builtin_memcpy(t, p, sizeof t);
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = value8(t[i], e);
}

template <typename T, typename P>
struct NormFwd {
    const T *x, *r;
    T *z, *y;
    const P *gamma, *beta;
    float *mean, *rstd;
    int8_t *q, *e;
    int64_t M, D;
    float eps, d;                        // d: D, to divide by (1 / D is rounded for most widths)
};

template <typename T, typename P, int TPR, int CV>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void k_norm_fwd(NormFwd<T, P> a) {
    constexpr int V = Piece<T>::kN, C = CV / V, R = TPR < 256 ? 256 / TPR : 1;
    __shared__ float red[48];
    const int64_t row = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * R + threadIdx.x / TPR;
    if (row >= a.M) return;                                  // TPR > 64: a workgroup is one row, so nobody waits for the leavers
    const int t = threadIdx.x % TPR;
    const int64_t base = row * a.D;
    const int64_t qpitch = (a.D + kBlock8 - 1) / kBlock8 * kBlock8;
    float v[C][V];
    float sum = 0.f;
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const int64_t d = (int64_t)(c * TPR + t) * V, left = a.D - d;
        load_piece<T, V>(a.x + base + d, left, v[c]);
        if (a.r) {
            float b[V];
            load_piece<T, V>(a.r + base + d, left, b);
#pragma unroll
            for (int i = 0; i < V; ++i) v[c][i] = (float)(T)(v[c][i] + b[i]);
            store_piece<T, V>(a.z + base + d, left, v[c]);
        }
#pragma unroll
        for (int i = 0; i < V; ++i) sum += v[c][i];
    }
    const float mean = row_sum<TPR>(sum, red, 0) / a.d;
    float off = 0.f, sq = 0.f;
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const int64_t d = (int64_t)(c * TPR + t) * V;
        if (a.q && d < qpitch) {
            const int e = block_exponent<T, V>(v[c]);
            store_q<V>(a.q + row * qpitch + d, v[c], e);
            if (d % kBlock8 == 0) a.e[row * (qpitch / kBlock8) + d / kBlock8] = (int8_t)e;
        }
#pragma unroll
        for (int i = 0; i < V; ++i) {
            v[c][i] -= mean;
            const float in = d + i < a.D ? v[c][i] : 0.f;
            off += in, sq += in * in;
        }
    }
    const float2 sums = row_sums<TPR>(off, sq, red);
    const float rest = sums.x / a.d, rstd = inverse_deviation(sums.y / a.d, rest, a.eps);
    if (a.mean && t == 0) a.mean[row] = mean + rest, a.rstd[row] = rstd;
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const int64_t d = (int64_t)(c * TPR + t) * V, left = a.D - d;
        float g[V], b[V];
        if (a.gamma) load_piece<P, V>(a.gamma + d, left, g);
        if (a.beta) load_piece<P, V>(a.beta + d, left, b);
#pragma unroll
        for (int i = 0; i < V; ++i) {
            float o = (v[c][i] - rest) * rstd;
            if (a.gamma) o *= g[i];
            if (a.beta) o += b[i];
            v[c][i] = o;
        }
        store_piece<T, V>(a.y + base + d, left, v[c]);
    }
}

template <typename T, typename P>
struct NormBwd {
    const T* x;                          // or q / e
    const int8_t *q, *e;
    const T *dy, *dz;
    const P* gamma;
    const float *mean, *rstd;
    T* dx;
    float* partial;                      // [gridDim.x][2][D], or NULL
    int64_t M, D;
    float d;
};

// a row's numbers of this thread as they are in memory
template <typename T, int C>
struct Raw {
    T v[C][Piece<T>::kN];
    template <int TPR>
    __device__ __forceinline__ void load(const T* __restrict__ row, int t, int64_t D) {
        constexpr int V = Piece<T>::kN;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int64_t d = (int64_t)(c * TPR + t) * V;
            if (d + V <= D) {
                __builtin_memcpy(v[c], row + d, 16);
            } else {
#pragma unroll
                for (int i = 0; i < V; ++i) v[c][i] = d + i < D ? row[d + i] : (T)0.f;
            }
        }
    }
};

template <int V, int C>
struct Raw8 {
    int8_t v[C][V], e[C];
    template <int TPR>
    __device__ __forceinline__ void load(const int8_t* __restrict__ q, const int8_t* __restrict__ ex, int t, int64_t pitch) {
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int64_t d = (int64_t)(c * TPR + t) * V;
            if (d < pitch) {
                __builtin_memcpy(v[c], q + d, V);
                e[c] = ex[d / kBlock8];
            } else {
#pragma unroll
                for (int i = 0; i < V; ++i) v[c][i] = 0;
                e[c] = 0;
            }
        }
    }
};

constexpr int bwd_threads(int tpr) { return tpr <= 64 ? 256 : tpr; }      // rows of a wave or less: several in a workgroup

// PACKED: x comes in its 8-bit form; DZ: a gradient reaches z by another way
template <typename T, typename P, int TPR, int CV, bool PACKED, bool DZ>
__global__ __launch_bounds__(bwd_threads(TPR)) void k_norm_bwd(NormBwd<T, P> a) {
    constexpr int V = Piece<T>::kN, C = CV / V, R = bwd_threads(TPR) / TPR;
    constexpr int kJoin = R > 1 ? R * TPR * CV : 32;
    constexpr bool kEarly = DZ && CV == 8;                       // dz with the rest of a row: 16 columns leave no registers for it
    __shared__ float red[kJoin];
    const int t = threadIdx.x % TPR, sub = threadIdx.x / TPR;
    const int64_t qpitch = (a.D + kBlock8 - 1) / kBlock8 * kBlock8, stride = (int64_t)gridDim.x * R;
    float dg[C][V] = {}, db[C][V] = {}, g[C][V];
    const auto load_gamma = [&](int c) {
        const int d = (c * TPR + t) * V;
        if (a.gamma) {
            load_piece<P, V>(a.gamma + d, (int)a.D - d, g[c]);
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) g[c][i] = 1.f;
        }
    };
    if constexpr (CV == 8)
#pragma unroll
        for (int c = 0; c < C; ++c) load_gamma(c);
    Raw<T, C> rx, rd, rz;
    Raw8<V, C> rq;
    float mean = 0.f, rstd = 0.f;
    auto fetch = [&](int64_t row) {
        if constexpr (PACKED) rq.template load<TPR>(a.q + row * qpitch, a.e + row * (qpitch / kBlock8), t, qpitch);
        else rx.template load<TPR>(a.x + row * a.D, t, a.D);
        rd.template load<TPR>(a.dy + row * a.D, t, a.D);
        if constexpr (kEarly) rz.template load<TPR>(a.dz + row * a.D, t, a.D);
        mean = a.mean[row], rstd = a.rstd[row];
    };
    for (int64_t row = (int64_t)blockIdx.x * R + sub; row < a.M; row += stride) {
        const int64_t base = row * a.D;
        fetch(row);                                              // all of it before the first sum waits for any
        const float rs = rstd;
        float xh[C][V], tt[C][V], z[C][V];
        float s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int left = (int)a.D - (c * TPR + t) * V;
            if constexpr (CV != 8) load_gamma(c);                // 16 columns: once for every row, for want of registers
#pragma unroll
            for (int i = 0; i < V; ++i) {
                float x;
                if constexpr (PACKED) x = value8(rq.v[c][i], rq.e[c]);
                else x = (float)rx.v[c][i];
                if constexpr (kEarly) z[c][i] = (float)rz.v[c][i];
                tt[c][i] = (float)rd.v[c][i];
                xh[c][i] = (x - mean) * rs;                      // behind the row's end dy is 0, so these never count
                dg[c][i] += i < left ? tt[c][i] * xh[c][i] : 0.f;
                db[c][i] += tt[c][i];
                tt[c][i] *= g[c][i];
                s1 += tt[c][i];
                s2 += i < left ? tt[c][i] * xh[c][i] : 0.f;
            }
        }
        if constexpr (TPR > 64) __syncthreads();                 // the previous row's sums have been read
        const float m1 = row_sum<TPR>(s1, red, 0) / a.d, m2 = row_sum<TPR>(s2, red, 1) / a.d;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int64_t d = (int64_t)(c * TPR + t) * V, left = a.D - d;
            if constexpr (CV != 8) asm volatile("" ::: "memory");
            if constexpr (DZ && !kEarly) load_piece<T, V>(a.dz + base + d, left, z[c]);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                tt[c][i] = rs * (tt[c][i] - m1 - xh[c][i] * m2);
                if constexpr (DZ) tt[c][i] += z[c][i];
            }
            if (a.dx) store_piece<T, V>(a.dx + base + d, left, tt[c]);
        }
    }
    if (!a.partial) return;
    float* out = a.partial + (int64_t)blockIdx.x * 2 * a.D;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        auto& acc = which ? db : dg;
        if constexpr (R > 1) {                                   // the R rows that this workgroup walks side by side
            __syncthreads();
#pragma unroll
            for (int c = 0; c < C; ++c)
#pragma unroll
                for (int i = 0; i < V; ++i) red[sub * (TPR * CV) + (c * TPR + t) * V + i] = acc[c][i];
            __syncthreads();
            for (int d = threadIdx.x; d < TPR * CV && d < a.D; d += 256) {
                float s = red[d];
#pragma unroll
                for (int r = 1; r < R; ++r) s += red[r * (TPR * CV) + d];
                out[which * a.D + d] = s;
            }
        } else {
#pragma unroll
            for (int c = 0; c < C; ++c) {
                const int64_t d = (int64_t)(c * TPR + t) * V;
                store_piece<float, V>(out + which * a.D + d, a.D - d, acc[c]);
            }
        }
    }
}

// Rows that do not fit the registers of a workgroup: the same sums in three (two) walks over the row, re-read from the cache.
template <typename T, typename P>
__global__ __launch_bounds__(1024) void k_norm_fwd_long(NormFwd<T, P> a) {
    constexpr int V = Piece<T>::kN, TPR = 1024;
    __shared__ float red[48];
    const int64_t row = (int64_t)blockIdx.y * gridDim.x + blockIdx.x, base = row * a.D, step = (int64_t)TPR * V;
    if (row >= a.M) return;                                  // the whole workgroup
    const int64_t qpitch = (a.D + kBlock8 - 1) / kBlock8 * kBlock8;
    const T* src = a.r ? a.z : a.x;
    float v[V], sum = 0.f;
    for (int64_t d = (int64_t)threadIdx.x * V; d < qpitch; d += step) {      // whole blocks of 32: neighbouring threads stay together
        load_piece<T, V>(a.x + base + d, a.D - d, v);
        if (a.r) {
            float b[V];
            load_piece<T, V>(a.r + base + d, a.D - d, b);
#pragma unroll
            for (int i = 0; i < V; ++i) v[i] = (float)(T)(v[i] + b[i]);
            store_piece<T, V>(a.z + base + d, a.D - d, v);               // read back by this thread only
        }
        if (a.q) {
            const int e = block_exponent<T, V>(v);
            store_q<V>(a.q + row * qpitch + d, v, e);
            if (d % kBlock8 == 0) a.e[row * (qpitch / kBlock8) + d / kBlock8] = (int8_t)e;
        }
#pragma unroll
        for (int i = 0; i < V; ++i) sum += v[i];
    }
    const float mean = row_sum<TPR>(sum, red, 0) / a.d;
    float off = 0.f, sq = 0.f;
    for (int64_t d = (int64_t)threadIdx.x * V; d < a.D; d += step) {
        load_piece<T, V>(src + base + d, a.D - d, v);
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float in = d + i < a.D ? v[i] - mean : 0.f;
            off += in, sq += in * in;
        }
    }
    const float2 sums = row_sums<TPR>(off, sq, red);
    const float rest = sums.x / a.d, rstd = inverse_deviation(sums.y / a.d, rest, a.eps);
    if (a.mean && threadIdx.x == 0) a.mean[row] = mean + rest, a.rstd[row] = rstd;
    for (int64_t d = (int64_t)threadIdx.x * V; d < a.D; d += step) {
        float g[V], b[V];
        load_piece<T, V>(src + base + d, a.D - d, v);
        if (a.gamma) load_piece<P, V>(a.gamma + d, a.D - d, g);
        if (a.beta) load_piece<P, V>(a.beta + d, a.D - d, b);
#pragma unroll
        for (int i = 0; i < V; ++i) {
            float o = (v[i] - mean - rest) * rstd;
            if (a.gamma) o *= g[i];
            if (a.beta) o += b[i];
            v[i] = o;
        }
        store_piece<T, V>(a.y + base + d, a.D - d, v);
    }
}

template <typename T, typename P>
__global__ __launch_bounds__(1024) void k_norm_bwd_long(NormBwd<T, P> a) {
    constexpr int V = Piece<T>::kN, TPR = 1024;
    __shared__ float red[32];
    const int64_t row = (int64_t)blockIdx.y * gridDim.x + blockIdx.x, base = row * a.D, step = (int64_t)TPR * V;
    if (row >= a.M) return;                                  // the whole workgroup
    const int64_t qpitch = (a.D + kBlock8 - 1) / kBlock8 * kBlock8;
    const float mean = a.mean[row], rstd = a.rstd[row];
    float m1 = 0.f, m2 = 0.f;
    for (int walk = 0; walk < 2; ++walk) {
        float s1 = 0.f, s2 = 0.f;
        for (int64_t d = (int64_t)threadIdx.x * V; d < a.D; d += step) {
            const int64_t left = a.D - d;
            float xh[V], t[V], g[V], z[V];
            if (a.q) load_q<V>(a.q + row * qpitch + d, a.e[row * (qpitch / kBlock8) + d / kBlock8], xh);
            else load_piece<T, V>(a.x + base + d, left, xh);
            load_piece<T, V>(a.dy + base + d, left, t);
            if (a.gamma) load_piece<P, V>(a.gamma + d, left, g);
            if (walk && a.dz) load_piece<T, V>(a.dz + base + d, left, z);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                xh[i] = (xh[i] - mean) * rstd;
                if (a.gamma) t[i] *= g[i];
                if (!walk) s1 += t[i], s2 += i < left ? t[i] * xh[i] : 0.f;
                else t[i] = rstd * (t[i] - m1 - xh[i] * m2) + (a.dz ? z[i] : 0.f);
            }
            if (walk && a.dx) store_piece<T, V>(a.dx + base + d, left, t);
        }
        if (!walk) m1 = row_sum<TPR>(s1, red, 0) / a.d, m2 = row_sum<TPR>(s2, red, 1) / a.d;
    }
}

// dgamma / dbeta of long rows: a thread owns V columns and walks the rows of its slice (gridDim.y of them; one: nothing to add up)
template <typename T, typename P>
__global__ __launch_bounds__(256) void k_norm_columns_long(NormBwd<T, P> a, P* __restrict__ dgamma, P* __restrict__ dbeta) {
    constexpr int V = Piece<T>::kN;
    const int64_t d = ((int64_t)blockIdx.x * 256 + threadIdx.x) * V;
    if (d >= a.D) return;
    const int64_t qpitch = (a.D + kBlock8 - 1) / kBlock8 * kBlock8, left = a.D - d;
    float dg[V] = {}, db[V] = {};
    for (int64_t row = blockIdx.y; row < a.M; row += gridDim.y) {
        float xh[V], t[V];
        if (a.q) load_q<V>(a.q + row * qpitch + d, a.e[row * (qpitch / kBlock8) + d / kBlock8], xh);
        else load_piece<T, V>(a.x + row * a.D + d, left, xh);
        load_piece<T, V>(a.dy + row * a.D + d, left, t);
        const float mean = a.mean[row], rstd = a.rstd[row];
#pragma unroll
        for (int i = 0; i < V; ++i) dg[i] += t[i] * ((xh[i] - mean) * rstd), db[i] += t[i];
    }
    if (gridDim.y == 1) {
        if (dgamma) store_piece<P, V>(dgamma + d, left, dg);
        if (dbeta) store_piece<P, V>(dbeta + d, left, db);
        return;
    }
    float* out = a.partial + (int64_t)blockIdx.y * 2 * a.D;
    store_piece<float, V>(out + d, left, dg);
    store_piece<float, V>(out + a.D + d, left, db);
}

// the workgroups' sums, added in ascending order in 8 strands and the strands in order: 32 columns x 8 strands a workgroup
template <typename P>
__global__ __launch_bounds__(256) void k_norm_join(const float* __restrict__ partial, int groups, int64_t D, P* __restrict__ dgamma, P* __restrict__ dbeta) {
    __shared__ float s[8][32];
    const int col = threadIdx.x & 31, strand = threadIdx.x >> 5;
    const int64_t j = (int64_t)blockIdx.x * 32 + col;          // 0 .. 2 D: dgamma, then dbeta
    float acc = 0.f;
    if (j < 2 * D)
#pragma unroll 8
        for (int g = strand; g < groups; g += 8) acc += partial[(int64_t)g * 2 * D + j];
    s[strand][col] = acc;
    __syncthreads();
    if (strand || j >= 2 * D) return;
#pragma unroll
    for (int k = 1; k < 8; ++k) acc += s[k][col];
    P* out = j < D ? dgamma : dbeta;
    if (out) out[j < D ? j : j - D] = (P)acc;
}

// one pass each way, 16 bytes of x a thread and turn: 8192 x 4096 bf16 (102 MB) 20 us to pack, 22 to unpack
template <typename T>
__global__ __launch_bounds__(256) void k_pack8(const T* __restrict__ x, int8_t* __restrict__ q, int8_t* __restrict__ e, int64_t M, int64_t D, int64_t qpitch) {
    constexpr int V = Piece<T>::kN;
    const int64_t per_row = qpitch / V, n = M * per_row;
    for (int64_t p = (int64_t)blockIdx.x * 256 + threadIdx.x; p < n; p += (int64_t)gridDim.x * 256) {   // 32 / V neighbours leave together
        const int64_t row = p / per_row, d = (p - row * per_row) * V;
        float v[V];
        load_piece<T, V>(x + row * D + d, D - d, v);
        const int ex = block_exponent<T, V>(v);
        store_q<V>(q + p * V, v, ex);
        if (d % kBlock8 == 0) e[p * V / kBlock8] = (int8_t)ex;
    }
}

template <typename T>
__global__ __launch_bounds__(256) void k_unpack8(const int8_t* __restrict__ q, const int8_t* __restrict__ e, T* __restrict__ x, int64_t M, int64_t D, int64_t qpitch) {
    constexpr int V = Piece<T>::kN;
    const int64_t per_row = qpitch / V, n = M * per_row;
    for (int64_t p = (int64_t)blockIdx.x * 256 + threadIdx.x; p < n; p += (int64_t)gridDim.x * 256) {
        const int64_t row = p / per_row, d = (p - row * per_row) * V;
        float v[V];
        load_q<V>(q + p * V, e[p * V / kBlock8], v);
        store_piece<T, V>(x + row * D + d, D - d, v);
    }
}

constexpr int64_t kLong = 16384;         // features that the register forms hold

// rows side by side in one workgroup of the forward, by width (the dispatch below)
int rows_per_group(int64_t D) { return D <= 128 ? 16 : D <= 2048 ? 4 : 1; }

// a launch has less than 2^32 threads in a dimension: many rows go over two
dim3 grid_of(int64_t blocks) {
    const int64_t x = blocks < (1 << 20) ? blocks : 1 << 20;
    return dim3((unsigned)x, (unsigned)((blocks + x - 1) / x));
}

// Threads of a row in the backward's walk: 8 columns each, so that their sums leave registers for many waves (with 16 or 32 a CU holds
// few, and 16,384 x 4,096 bf16 with a gradient past the norm took 1.6 times as long). Above 8,192: 16 columns.
int bwd_row_threads(int64_t D) { return D <= 128 ? 16 : D <= 512 ? 64 : D <= 1024 ? 128 : D <= 2048 ? 256 : D <= 4096 ? 512 : 1024; }

// Workgroups of the walk: 1,024 threads a CU, and no more than leave each row slot four rows, so that the partial sums (2 D floats
// a workgroup: 16 MiB at most up to 8,192 features, 32 MiB above) stay small beside the rows. Long rows: slices of the columns' walk,
// which has a workgroup for every 4 KiB of a row already: 64 at most, four rows each, and within the same 32 MiB - one above 2^21 features.
int64_t bwd_groups(int64_t M, int64_t D) {
    if (D > kLong) {
        const int64_t rows = (M + 3) / 4, room = (32 << 20) / (8 * D), n = rows < room ? rows : room;
        return n < 1 ? 1 : n < 64 ? n : 64;
    }
    const int64_t tpr = bwd_row_threads(D), threads = bwd_threads((int)tpr), R = threads / tpr, most = 256 * 1024 / threads, need = (M + 4 * R - 1) / (4 * R);
    return need < most ? need : most;
}

template <typename T, typename P>
int norm_fwd(const NormFwd<T, P>& a, hipStream_t s) {
    const int64_t D = a.D, R = rows_per_group(D), blocks = (a.M + R - 1) / R;
    void (*fn)(NormFwd<T, P>) = D <= 128 ? k_norm_fwd<T, P, 16, 8> : D <= 512 ? k_norm_fwd<T, P, 64, 8> : D <= 1024 ? k_norm_fwd<T, P, 64, 16>
                              : D <= 2048 ? k_norm_fwd<T, P, 64, 32> : D <= 4096 ? k_norm_fwd<T, P, 256, 16> : D <= 8192 ? k_norm_fwd<T, P, 256, 32>
                              : D <= kLong ? k_norm_fwd<T, P, 1024, 16> : k_norm_fwd_long<T, P>;
    hipLaunchKernelGGL(fn, grid_of(blocks), dim3(D <= 8192 ? 256 : 1024), 0, s, a);
    return launch_status();
}

template <typename T, typename P, bool PACKED, bool DZ>
auto norm_bwd_for(int64_t D) {
    return D <= 128 ? k_norm_bwd<T, P, 16, 8, PACKED, DZ> : D <= 512 ? k_norm_bwd<T, P, 64, 8, PACKED, DZ> : D <= 1024 ? k_norm_bwd<T, P, 128, 8, PACKED, DZ>
         : D <= 2048 ? k_norm_bwd<T, P, 256, 8, PACKED, DZ> : D <= 4096 ? k_norm_bwd<T, P, 512, 8, PACKED, DZ>
         : D <= 8192 ? k_norm_bwd<T, P, 1024, 8, PACKED, DZ> : k_norm_bwd<T, P, 1024, 16, PACKED, DZ>;
}

template <typename T, typename P>
int norm_bwd(const NormBwd<T, P>& a, P* dgamma, P* dbeta, hipStream_t s) {
    const int64_t D = a.D;
    const int groups = (int)bwd_groups(a.M, D);
    int rc = URSA_OK;
    if (D > kLong) {
        if (a.dx) hipLaunchKernelGGL((k_norm_bwd_long<T, P>), grid_of(a.M), dim3(1024), 0, s, a);
        if ((rc = launch_status())) return rc;
        if (!dgamma && !dbeta) return rc;
        hipLaunchKernelGGL((k_norm_columns_long<T, P>), dim3((unsigned)((D + 256 * Piece<T>::kN - 1) / (256 * Piece<T>::kN)), groups), dim3(256), 0, s, a, dgamma, dbeta);
        if (groups == 1) return launch_status();
    } else {
        void (*fn)(NormBwd<T, P>) = a.q ? (a.dz ? norm_bwd_for<T, P, true, true>(D) : norm_bwd_for<T, P, true, false>(D))
                                        : (a.dz ? norm_bwd_for<T, P, false, true>(D) : norm_bwd_for<T, P, false, false>(D));
        hipLaunchKernelGGL(fn, dim3(groups), dim3(bwd_threads(bwd_row_threads(D))), 0, s, a);
    }
    if ((rc = launch_status()) || !a.partial) return rc;
    hipLaunchKernelGGL(k_norm_join<P>, dim3((unsigned)((2 * D + 31) / 32)), dim3(256), 0, s, (const float*)a.partial, groups, D, dgamma, dbeta);
    return launch_status();
}

bool bad_dtype(int32_t d) { return d < URSA_F32 || d > URSA_F16; }

int sizes_ok(int64_t M, int64_t D) {
    if (M < 0 || D < 0) return URSA_ESIZE;
    if (M > INT32_MAX || D > 1 << 27 || (M && D > (INT64_MAX >> 4) / M)) return URSA_ESIZE;
    return URSA_OK;
}

// f(T, P) for a pair of types; parameters are of the tensors' type or fp32
#define URSA_NORM_TYPES(dtype, pdtype, call)                                                                  \
    (dtype == URSA_F32 ? call(float, float) : dtype == URSA_BF16 ? (pdtype == URSA_F32 ? call(bf16, float) : call(bf16, bf16)) \
                                                                 : (pdtype == URSA_F32 ? call(f16, float) : call(f16, f16)))

}  // namespace

extern "C" int64_t ursa_layer_norm_ws_floats(int64_t M, int64_t D) {
    if (sizes_ok(M, D) || M == 0) return 0;
    const int64_t n = bwd_groups(M, D);
    return D > kLong && n == 1 ? 0 : n * 2 * D;
}

extern "C" int ursa_layer_norm_fwd(const void* x, const void* addend, void* z_out, void* y, const void* gamma, const void* beta, float* mean,
                                   float* rstd, int8_t* q, int8_t* e, int64_t M, int64_t D, float eps, int32_t dtype, int32_t pdtype,
                                   ursa_stream_t stream) {
    if (bad_dtype(dtype) || (pdtype != dtype && pdtype != URSA_F32)) return URSA_EFLAGS;
    if (int rc = sizes_ok(M, D)) return rc;
    if (!(eps >= 0.f)) return URSA_EVALUE;
    if (M == 0 || D == 0) return URSA_OK;
    if (!x || !y || (addend != nullptr) != (z_out != nullptr) || (mean != nullptr) != (rstd != nullptr) || (q != nullptr) != (e != nullptr)) return URSA_ENULL;
    const uintptr_t es = (uintptr_t)element_size(dtype) - 1, ps = (uintptr_t)element_size(pdtype) - 1;
    if (((uintptr_t)x | (uintptr_t)addend | (uintptr_t)z_out | (uintptr_t)y) & es || ((uintptr_t)gamma | (uintptr_t)beta) & ps ||
        ((uintptr_t)mean | (uintptr_t)rstd) & 3 || (uintptr_t)q & 15) return URSA_EALIGN;
#define URSA_CALL(T, P) norm_fwd<T, P>({(const T*)x, (const T*)addend, (T*)z_out, (T*)y, (const P*)gamma, (const P*)beta, mean, rstd, q, e, M, D, eps, (float)D}, (hipStream_t)stream)
    return URSA_NORM_TYPES(dtype, pdtype, URSA_CALL);
#undef URSA_CALL
}

extern "C" int ursa_layer_norm_bwd(const void* x, const int8_t* q, const int8_t* e, const void* dy, const void* dz, const void* gamma,
                                   const float* mean, const float* rstd, void* dx, void* dgamma, void* dbeta, float* ws, int64_t M, int64_t D,
                                   int32_t dtype, int32_t pdtype, ursa_stream_t stream) {
    if (bad_dtype(dtype) || (pdtype != dtype && pdtype != URSA_F32)) return URSA_EFLAGS;
    if (int rc = sizes_ok(M, D)) return rc;
    if (M == 0 || D == 0) return M == 0 && D && (dgamma || dbeta) ? URSA_EVALUE : URSA_OK;     // no rows: the caller's zeros
    if ((x != nullptr) == (q != nullptr) || (q != nullptr) != (e != nullptr) || !dy || !mean || !rstd || ((dgamma || dbeta) && ursa_layer_norm_ws_floats(M, D) && !ws)) return URSA_ENULL;
    const uintptr_t es = (uintptr_t)element_size(dtype) - 1, ps = (uintptr_t)element_size(pdtype) - 1;
    if (((uintptr_t)x | (uintptr_t)dy | (uintptr_t)dz | (uintptr_t)dx) & es || ((uintptr_t)gamma | (uintptr_t)dgamma | (uintptr_t)dbeta) & ps ||
        ((uintptr_t)mean | (uintptr_t)rstd | (uintptr_t)ws) & 3 || (uintptr_t)q & 15) return URSA_EALIGN;
    float* part = dgamma || dbeta ? ws : nullptr;
#define URSA_CALL(T, P) norm_bwd<T, P>({(const T*)x, q, e, (const T*)dy, (const T*)dz, (const P*)gamma, mean, rstd, (T*)dx, part, M, D, (float)D}, (P*)dgamma, (P*)dbeta, (hipStream_t)stream)
    return URSA_NORM_TYPES(dtype, pdtype, URSA_CALL);
#undef URSA_CALL
}

static int act8_sizes(const void* x, const int8_t* q, const int8_t* e, int64_t M, int64_t D, int32_t dtype) {
    if (bad_dtype(dtype)) return URSA_EFLAGS;
    if (int rc = sizes_ok(M, D)) return rc;
    if (M == 0 || D == 0) return 1;
    if (!x || !q || !e) return URSA_ENULL;
    if ((uintptr_t)x & (uintptr_t)(element_size(dtype) - 1) || (uintptr_t)q & 15) return URSA_EALIGN;
    return URSA_OK;
}

extern "C" int ursa_act8_pack(const void* x, int8_t* q, int8_t* e, int64_t M, int64_t D, int32_t dtype, ursa_stream_t stream) {
    const int rc = act8_sizes(x, q, e, M, D, dtype);
    if (rc) return rc > 0 ? URSA_OK : rc;
    const int64_t pitch = (D + kBlock8 - 1) / kBlock8 * kBlock8, n = M * pitch / (dtype == URSA_F32 ? 4 : 8), blocks = (n + 255) / 256;
    const dim3 grid((unsigned)(blocks < 16384 ? blocks : 16384));
    if (dtype == URSA_F32) hipLaunchKernelGGL(k_pack8<float>, grid, dim3(256), 0, (hipStream_t)stream, (const float*)x, q, e, M, D, pitch);
    else if (dtype == URSA_BF16) hipLaunchKernelGGL(k_pack8<bf16>, grid, dim3(256), 0, (hipStream_t)stream, (const bf16*)x, q, e, M, D, pitch);
    else hipLaunchKernelGGL(k_pack8<f16>, grid, dim3(256), 0, (hipStream_t)stream, (const f16*)x, q, e, M, D, pitch);
    return launch_status();
}

extern "C" int ursa_act8_unpack(const int8_t* q, const int8_t* e, void* x, int64_t M, int64_t D, int32_t dtype, ursa_stream_t stream) {
    const int rc = act8_sizes(x, q, e, M, D, dtype);
    if (rc) return rc > 0 ? URSA_OK : rc;
    const int64_t pitch = (D + kBlock8 - 1) / kBlock8 * kBlock8, n = M * pitch / (dtype == URSA_F32 ? 4 : 8), blocks = (n + 255) / 256;
    const dim3 grid((unsigned)(blocks < 16384 ? blocks : 16384));
    if (dtype == URSA_F32) hipLaunchKernelGGL(k_unpack8<float>, grid, dim3(256), 0, (hipStream_t)stream, q, e, (float*)x, M, D, pitch);
    else if (dtype == URSA_BF16) hipLaunchKernelGGL(k_unpack8<bf16>, grid, dim3(256), 0, (hipStream_t)stream, q, e, (bf16*)x, M, D, pitch);
    else hipLaunchKernelGGL(k_unpack8<f16>, grid, dim3(256), 0, (hipStream_t)stream, q, e, (f16*)x, M, D, pitch);
    return launch_status();
}
