// ursa_linear.hip — K15: the linear layer with its epilogue, y = act(x W' + b) + r, and its gradients.
//
//   z = x W' + b ; y = act(z) + r            act: none, relu, gelu (z Phi(z)), silu (z sigmoid(z))
//   dz = dy act'(z) ; dr = dy ; dx = dz W ; dW = dz' x ; db = sum_rows dz
//
// All three products are one kernel, C[m][n] = sum_k X(m, k) Y(n, k), whose operands are stored either along the contraction (k
// contiguous: x and W forward) or across it (W in dx; dz and x in dW). Both go to LDS as rows of 16-bit numbers; the first kind is
// read as eight consecutive k of a row (ds_read_b128), the second by the transposing LDS read (ds_read_b64_tr_b16), which hands
// each lane four k of its column. fp32 operands are split while they are staged, v = hi + mid + lo with three bf16 numbers
// (8 + 8 + 8 bits: exact from 2^-110 up; below, lo ends at 2^-133 and half of that is lost), and six of the nine partial products are
// summed in fp32: what is left out (mid lo twice, lo lo) is below 2^-21.9 of |x w| and 2^-25 on average, of either sign, and the bf16
// matrix instruction does 16 times the work of the fp32 one. Sums that come out not finite are taken once more without the split.
//
// Sums are fp32; a contraction is cut over workgroups where there are few tiles, and a second launch adds the pieces in order.
#include "ursa_ops.h"

namespace {

using namespace ursa;

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

constexpr int kFlat = 0, kAcross = 1, kAcross8 = 2;      // how an operand is stored: k contiguous; across k; across k in 8 bits

template <int K> struct Kind { static constexpr int value = K; };

template <typename T> struct Arith { typedef T type; };  // what the matrix instruction multiplies
template <> struct Arith<float> { typedef bf16 type; };

template <typename A>
__device__ __forceinline__ f32x4 mfma(s16x8 a, s16x8 b, f32x4 c) {
    if constexpr (__is_same(A, bf16)) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// Phi(z), the standard normal distribution, and e = exp(-z^2 / 2): Phi(-u) = e g(u) for u >= 0 with g(u) = erfcx(u / sqrt 2) / 2, and
// g as a polynomial in t = 1 / (1 + 0.3 u) without a constant term (g falls like 1 / u), fitted to the least largest relative error:
// 1.5e-7 in exact arithmetic, so the tails keep their relative accuracy. About 22 vector operations where erff takes three times that:
// an epilogue's activations would cost as much as its matrix instructions.
__device__ __forceinline__ float normal_cdf(float z, float& e) {
    const float u = fabsf(z), t = __builtin_amdgcn_rcpf(fmaf(0.3f, u, 1.f));
    e = __builtin_amdgcn_exp2f(z * z * -0.72134752044448170f);          // log2(e) / 2
    float g = 0.03567589074373245f;
    g = fmaf(g, t, -0.15720807015895844f);
    g = fmaf(g, t, 0.20636247098445892f);
    g = fmaf(g, t, -0.05369199067354202f);
    g = fmaf(g, t, 0.1285659670829773f);
    g = fmaf(g, t, 0.09991223365068436f);
    g = fmaf(g, t, 0.12075414508581161f);
    g = fmaf(g, t, 0.11962928622961044f);
    const float tail = g * t * e;
    return z > 0.f ? 1.f - tail : tail;
}

__device__ __forceinline__ float sigmoid(float z) { return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(z * -1.4426950408889634f)); }

// act over N values at once: one uniform branch for all of them
template <int N>
__device__ __forceinline__ void act_values(float (&v)[N], int act) {
    float e;
    if (act == URSA_ACT_GELU) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] *= normal_cdf(v[i], e);
    } else if (act == URSA_ACT_SILU) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] *= sigmoid(v[i]);
    } else if (act == URSA_ACT_RELU) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = v[i] < 0.f ? 0.f : v[i];      // a NaN stays one
    }
}

// g *= act'(z)
template <int N>
__device__ __forceinline__ void act_slopes(float (&g)[N], const float (&z)[N], int act) {
    if (act == URSA_ACT_GELU) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            float e;
            const float phi = normal_cdf(z[i], e);
            g[i] *= e > 0.f ? fmaf(z[i] * 0.39894228040143268f, e, phi) : phi;       // z that was rounded to an infinity: 0 or 1
        }
    } else if (act == URSA_ACT_SILU) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float s = sigmoid(z[i]), p = s * (1.f - s);
            g[i] *= p > 0.f ? fmaf(p, z[i], s) : s;                                   // likewise; a NaN stays one
        }
    } else if (act == URSA_ACT_RELU) {
#pragma unroll
        for (int i = 0; i < N; ++i) g[i] = z[i] <= 0.f ? 0.f : g[i];             // shut where z <= 0: open for a NaN, as the stock op's
    }
}

struct Operand {
    const void* p;               // [rows][k] (kFlat) or [k][rows] (kAcross); kAcross8: int8 [k][pitch]
    const int8_t* e;             // kAcross8: [k][pitch / 32]
    int64_t pitch;               // elements from one stored row to the next
    int rows;
};

struct Epilogue {
    void *out, *z;               // [M][N]; z (or NULL): x W' + b before the activation
    const void *bias, *residual; // [N], [M][N], or NULL
    float* partial;              // [slices][M][N] when the contraction is cut
    int act;
};

struct Shape {
    int M, N, K;
    int tiles_m, tiles_n, slices, k_slice;   // k_slice: a multiple of the k step
};

// one 8-element chunk on its way from memory to LDS
template <typename T, int KIND> struct Chunk { T v[8]; };
template <typename T> struct Chunk<T, kAcross8> { int8_t v[8]; int8_t e; };

template <typename T, int KIND>
__device__ __forceinline__ void load_chunk(Chunk<T, KIND>& c, const Operand& o, int64_t outer, int inner, bool whole, bool in, int inner_end) {
    // stored row `outer`, elements inner .. inner + 7: all of them (`whole`), or those below inner_end if `in`, and zeros
    if constexpr (KIND == kAcross8) {
        if (whole || (in && inner < inner_end)) {             // rows are padded to whole blocks of 32 with zeros
            __builtin_memcpy(c.v, (const int8_t*)o.p + outer * o.pitch + inner, 8);
            c.e = o.e[outer * (o.pitch / kBlock8) + inner / kBlock8];
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) c.v[i] = 0;
            c.e = 0;
        }
    } else {
        const T* p = (const T*)o.p + outer * o.pitch + inner;
        if (whole) {
            __builtin_memcpy(c.v, p, sizeof c.v);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) c.v[i] = in && inner + i < inner_end ? p[i] : (T)0.f;
        }
    }
}

template <typename T, int KIND> constexpr int planes() { return __is_same(T, float) && KIND != kAcross8 ? 3 : 1; }

// the chunk as `planes` vectors of eight 16-bit numbers
template <typename T, int KIND>
__device__ __forceinline__ void split_chunk(const Chunk<T, KIND>& c, s16x8 (&out)[3]) {
    typedef typename Arith<T>::type A;
    if constexpr (KIND == kAcross8) {
        // bytes + 128 convert in one instruction each; everything behind that is exact, the rounding to A too
        const float s = c.e == kNonFinite8 ? __builtin_nanf("") : pow2_bits(c.e);
        uint32_t b[2];
        __builtin_memcpy(b, c.v, 8);
        b[0] ^= 0x80808080u, b[1] ^= 0x80808080u;
#pragma unroll
        for (int i = 0; i < 8; ++i) out[0][i] = __builtin_bit_cast(short, (A)(((float)(b[i >> 2] >> (8 * (i & 3)) & 0xff) - 128.f) * s));
    } else if constexpr (__is_same(T, float)) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint32_t b = __builtin_bit_cast(uint32_t, (float)c.v[i]);
            const float r = c.v[i] - __builtin_bit_cast(float, b & 0xffff0000u);    // exact: the low 16 bits
            const bf16 mid = (bf16)r;
            const bf16 lo = (bf16)(r - (float)mid);
            out[0][i] = (short)(b >> 16);
            out[1][i] = __builtin_bit_cast(short, mid);
            out[2][i] = __builtin_bit_cast(short, lo);
        }
    } else {
        __builtin_memcpy(&out[0], c.v, 16);
    }
}

// LDS places of a 16-byte piece. kFlat: [rows][BK], the pieces of a row permuted so that eight rows' reads of one k fall into
// different banks; kAcross: [BK][R], 32-byte slots permuted by k so that the rows k .. k + 3 and k + 8 .. k + 11, which half a wave's
// transposing read takes, do (256 bytes: with the first four alone apart, half of the LDS's active cycles were conflicts).
template <int BK> __device__ __forceinline__ int flat_at(int row, int piece) {
    return BK == 64 ? row * 64 + ((piece ^ (row & 7)) << 3) : row * 32 + ((piece ^ ((row >> 1) & 3)) << 3);
}
template <int R> __device__ __forceinline__ int across_at(int k, int slot) {
    return k * R + ((slot ^ (R >= 128 ? (k & 3) | ((k >> 1) & 4) : (k & 3) ^ ((k >> 3) & 1))) << 4);
}

// the fragment of 16 rows from row0, k .. k + 31: lane l holds row l % 16, k + 8 (l / 16) .. + 7
template <int KIND, int BK, int R>
__device__ __forceinline__ s16x8 fragment(const short* plane, int row0, int k, int lane) {
    if constexpr (KIND == kFlat) {
        return *(const s16x8*)(plane + flat_at<BK>(row0 + (lane & 15), (k >> 3) + (lane >> 4)));
    } else {
        const int kr = k + 8 * (lane >> 4) + ((lane & 15) >> 2), in = (lane & 3) << 2;
        const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(plane + across_at<R>(kr, row0 >> 4) + in));
        const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(plane + across_at<R>(kr + 4, row0 >> 4) + in));
        return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
    }
}

// numbers (row, k) .. (row, k + U - 1) of an fp32 operand; zeros from k_end on
template <int KIND, int U>
__device__ __forceinline__ void numbers_at(const Operand& o, int row, int k, int k_end, float (&v)[U]) {
    if constexpr (KIND == kFlat) {
        load_piece<float, U>((const float*)o.p + row * o.pitch + k, k_end - k, v);
    } else {
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const int64_t at = k + i < k_end ? k + i : k_end - 1;
            if constexpr (KIND == kAcross8) v[i] = value8(((const int8_t*)o.p)[at * o.pitch + row], o.e[at * (o.pitch / kBlock8) + row / kBlock8]);
            else v[i] = ((const float*)o.p)[at * o.pitch + row];
            if (k + i >= k_end) v[i] = 0.f;
        }
    }
}

// The split's sums that are not finite, again. The parts of a number may differ in sign, so where hi hi is past the range and hi lo past
// the other end of it they make a NaN of an infinite sum; and the remainder of an infinite operand is one. Either way the sum is not
// finite and stays so. A wave that holds such a sum takes the 16 columns around it once more by the fp32 instruction, straight from
// memory (k as in k_rows), and keeps what that has in the place of it: infinities and NaNs as fp32 has them. 4096^3 (715 us): a row of
// them 1.9 ms, nothing else 2.7 ms; none of them: within 1 % of the kernels without this.
template <int XK, int YK, int FY, int FX>
__device__ __forceinline__ void sums_again(f32x4 (&acc)[FY][FX], const Operand& X, const Operand& Y, int m0, int n0, int k_begin, int k_end, int lane) {
    constexpr int U = FX > 2 ? 8 : 4;                     // k a lane and turn; the smaller tile keeps its registers
    float top[FY], most = 0.f;                            // the largest magnitude; a NaN is larger than all (two sums an instruction)
#pragma unroll
    for (int j = 0; j < FY; ++j) {
        top[j] = 0.f;
#pragma unroll
        for (int i = 0; i < FX; ++i)
#pragma unroll
            for (int v = 0; v < 4; ++v) top[j] = __builtin_elementwise_maximum(top[j], fabsf(acc[j][i][v]));
        most = __builtin_elementwise_maximum(most, top[j]);
    }
    if (!__any(!(most < INFINITY))) return;
#pragma unroll
    for (int j = 0; j < FY; ++j) {
        if (!__any(!(top[j] < INFINITY))) continue;               // the whole wave goes on: the instruction takes every lane's numbers
        const int n = n0 + 16 * j + (lane & 15), ry = n < Y.rows ? n : Y.rows - 1;      // behind the last row: not stored
        f32x4 c[FX] = {};
        for (int k0 = k_begin; k0 < k_end; k0 += 4 * U) {
            const int k = k0 + U * (lane >> 4);
            float y[U], x[FX][U];
            numbers_at<YK>(Y, ry, k, k_end, y);
#pragma unroll
            for (int i = 0; i < FX; ++i) {
                const int m = m0 + 16 * i + (lane & 15);
                numbers_at<XK>(X, m < X.rows ? m : X.rows - 1, k, k_end, x[i]);
            }
#pragma unroll
            for (int i = 0; i < FX; ++i)
#pragma unroll
                for (int u = 0; u < U; ++u) c[i] = __builtin_amdgcn_mfma_f32_16x16x4f32(y[u], x[i][u], c[i], 0, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < FX; ++i)
#pragma unroll
            for (int v = 0; v < 4; ++v) acc[j][i][v] = fabsf(acc[j][i][v]) < INFINITY ? acc[j][i][v] : c[i][v];
    }
}

// C consecutive n of one m through the epilogue; `bias`: those of the bias, or zeros. z is kept in the tensors' type: half the bytes of
// fp32 to write, hold and read again, for a slope that is off by that rounding of z (gradients 1.66e-3 -> 1.77e-3, bf16 gelu).
template <typename T, int C>
__device__ __forceinline__ void finish(const Epilogue& ep, int64_t m, int n, int N, float (&v)[C], const float (&bias)[C]) {
    const int valid = N - n;
    const int64_t at = m * N + n;
#pragma unroll
    for (int i = 0; i < C; ++i) v[i] += bias[i];
    if (ep.z) store_piece<T, C>((T*)ep.z + at, valid, v);
    act_values(v, ep.act);
    if (ep.residual) {
        float t[C];
        load_piece<T, C>((const T*)ep.residual + at, valid, t);
#pragma unroll
        for (int i = 0; i < C; ++i) v[i] += t[i];
    }
    store_piece<T, C>((T*)ep.out + at, valid, v);
}

template <typename T, int C>
__device__ __forceinline__ void load_bias(const Epilogue& ep, int n, int N, float (&b)[C]) {
    if (ep.bias) {
        load_piece<T, C>((const T*)ep.bias + n, N - n, b);
    } else {
#pragma unroll
        for (int i = 0; i < C; ++i) b[i] = 0.f;
    }
}

// tile of this workgroup: workgroups go round the 8 XCDs, so every eighth is a neighbour in one L2; those take consecutive tiles, and
// consecutive tiles run down 8 rows of tiles before they step right, so that both operands of a group of tiles stay in that L2
__device__ __forceinline__ void tile_of(int id, const Shape& s, int& tm, int& tn) {
    const int n = s.tiles_m * s.tiles_n, per = n >> 3, rem = n & 7, x = id & 7, i = id >> 3;
    const int t = x < rem ? x * (per + 1) + i : rem * (per + 1) + (x - rem) * per + i;
    const int band = 8 * s.tiles_n, b = t / band, rows = s.tiles_m - 8 * b < 8 ? s.tiles_m - 8 * b : 8, j = t - b * band;
    tm = 8 * b + j % rows;
    tn = j / rows;
}

// TILE x TILE outputs by four waves (2 x 2), operands through registers (types that are converted, rows at any alignment). What lies
// behind an operand's rows only enters outputs that are not stored, so whole chunks are read there too: the last row again (kFlat),
// the next k's numbers (kAcross; there are TILE of them). Element by element, every step of a tile on the edge waited for each of its
// chunks in turn (1000 x 777 outputs, K 1111, fp16: forward 19.1 -> 16.2 us, dx 19.6 -> 14.4, dW 19.1 -> 16.3).
template <typename T, int XK, int YK, int TILE>
__global__ __launch_bounds__(256) void k_product(Operand X, Operand Y, Shape s, Epilogue ep) {
    typedef typename Arith<T>::type A;
    constexpr int BK = __is_same(T, float) ? 32 : 64, PX = planes<T, XK>(), PY = planes<T, YK>();
    constexpr int CH = TILE * BK / 8 / 256, F = TILE / 32;          // chunks a thread stages per operand; 16-row fragments a wave has
    __shared__ __attribute__((aligned(16))) short xs[PX][TILE * BK], ys[PY][TILE * BK];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int tm, tn;
    tile_of(blockIdx.x, s, tm, tn);
    const int m0 = tm * TILE, n0 = tn * TILE;
    const int k_begin = blockIdx.y * s.k_slice, k_end = s.K - k_begin < s.k_slice ? s.K : k_begin + s.k_slice;
    const int wm = (wave & 1) * (TILE / 2), wn = (wave >> 1) * (TILE / 2);
    Chunk<T, XK> cx[CH];
    Chunk<T, YK> cy[CH];
    auto fetch = [&](auto& c, const Operand& o, auto kind, int r0, int k0) {
        constexpr int KIND = decltype(kind)::value;
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            const int id = i * 256 + tid;
            if constexpr (KIND == kFlat) {
                const int row = r0 + id / (BK / 8), k = k0 + id % (BK / 8) * 8;
                load_chunk<T, KIND>(c[i], o, row < o.rows ? row : o.rows - 1, k, k + 8 <= k_end, true, k_end);
            } else {
                const int k = k0 + id / (TILE / 8), row = r0 + id % (TILE / 8) * 8;
                const bool in = k < k_end;
                load_chunk<T, KIND>(c[i], o, k, row, in && (row + 8 <= o.rows || (k < s.K - 1 && o.pitch >= TILE)), in, o.rows);
            }
        }
    };
    auto stage = [&](auto& c, auto& lds, auto kind) {
        constexpr int KIND = decltype(kind)::value, P = planes<T, KIND>();
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            const int id = i * 256 + tid;
            s16x8 out[3];
            split_chunk<T, KIND>(c[i], out);
            int at;
            if constexpr (KIND == kFlat) at = flat_at<BK>(id / (BK / 8), id % (BK / 8));
            else at = across_at<TILE>(id / (TILE / 8), id % (TILE / 8) >> 1) + (id % (TILE / 8) & 1) * 8;
#pragma unroll
            for (int p = 0; p < P; ++p) *(s16x8*)(&lds[p][at]) = out[p];
        }
    };
    f32x4 acc[F][F] = {};
    if (k_begin < k_end) {
        fetch(cx, X, Kind<XK>{}, m0, k_begin);
        fetch(cy, Y, Kind<YK>{}, n0, k_begin);
    }
    for (int k = k_begin; k < k_end; k += BK) {
        __syncthreads();
        stage(cx, xs, Kind<XK>{});
        stage(cy, ys, Kind<YK>{});
        __syncthreads();
        if (k + BK < k_end) {
            fetch(cx, X, Kind<XK>{}, m0, k + BK);
            fetch(cy, Y, Kind<YK>{}, n0, k + BK);
        }
#pragma unroll
        for (int kk = 0; kk < BK; kk += 32) {
            s16x8 fx[PX][F];
#pragma unroll
            for (int p = 0; p < PX; ++p)
#pragma unroll
                for (int i = 0; i < F; ++i) fx[p][i] = fragment<XK, BK, TILE>(xs[p], wm + 16 * i, kk, lane);
#pragma unroll
            for (int j = 0; j < F; ++j) {
                s16x8 fy[PY];
#pragma unroll
                for (int p = 0; p < PY; ++p) fy[p] = fragment<YK, BK, TILE>(ys[p], wn + 16 * j, kk, lane);
#pragma unroll
                for (int px = PX - 1; px >= 0; --px)                 // small products first
#pragma unroll
                    for (int py = PY - 1; py >= 0; --py)
                        if (px + py <= 2)
#pragma unroll
                            for (int i = 0; i < F; ++i) acc[j][i] = mfma<A>(fy[py], fx[px][i], acc[j][i]);
            }
        }
    }
    if constexpr (PX > 1) sums_again<XK, YK>(acc, X, Y, m0 + wm, n0 + wn, k_begin, k_end, lane);
    // accumulator of (fy, fx): lane l holds m = l % 16 and n = 4 (l / 16) .. + 3
#pragma unroll
    for (int i = 0; i < F; ++i) {
        const int m = m0 + wm + 16 * i + (lane & 15);
        if (m >= s.M) continue;
#pragma unroll
        for (int j = 0; j < F; ++j) {
            const int n = n0 + wn + 16 * j + 4 * (lane >> 4);
            if (n >= s.N) continue;
            float v[4] = {acc[j][i][0], acc[j][i][1], acc[j][i][2], acc[j][i][3]}, b[4];
            if (ep.partial) {
                store_piece<float, 4>(ep.partial + ((int64_t)blockIdx.y * s.M + m) * s.N + n, s.N - n, v);
            } else {
                load_bias<T, 4>(ep, n, s.N, b);
                finish<T, 4>(ep, m, n, s.N, v, b);
            }
        }
    }
}

// ---- 256 x 256 outputs by eight waves, 16-bit operands straight from memory to LDS ------------------------------------------
// A wave owns 128 x 64 outputs (32 accumulators of 16 x 16, two waves on each SIMD): 12 fragment reads feed 32 matrix instructions
// (bf16 8192^3: 1330 TFLOP/s each way, matrix pipe busy 0.69 of the cycles at the 1.77 GHz that the power allows, LDS 0.27). The
// fragments of the next 32 k are read while the present ones are multiplied. Two stages of 64 k in LDS: as soon as every wave has its
// last fragments of a stage, the pieces of the stage after the next start from memory to LDS, past the registers, and have a whole
// stage's time to arrive. A wave's 64 pieces land side by side, so what spreads the banks is a permutation of the addresses that they
// come from (and gaps between the rows of a kAcross stage). Buffer loads: what lies behind an operand's last element reads as 0. For
// operands whose rows and start are multiples of 16 bytes and whose rows are at most 2^22 long (32-bit offsets within a tile).
typedef __attribute__((address_space(3))) const void* lptr;
typedef int i32x4 __attribute__((ext_vector_type(4)));

// 16 bytes from each lane's `offset` in the buffer to LDS at `dst` + 16 lane (dst the same in the whole wave). Not the compiler's
// builtin: that one makes it wait for every such load before the next LDS read of any address. Whoever reads the LDS waits
// (vmcnt(0), then a barrier). m0 has no other use here. The compiler does not look into the block for hazards: the wait states
// cover a scalar register that a vector instruction wrote just before (five) and m0 (one).
__device__ __forceinline__ void memory_to_lds(i32x4 buffer, uint32_t offset, const short* dst) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
                 ::"s"((uint32_t)(uintptr_t)(lptr)dst), "v"(offset), "s"(buffer) : "memory");
}

constexpr int kWideK = 64;
constexpr int64_t kWideMaxPitch = 1 << 22;

// A stage of R rows: kFlat [R][64], kAcross [64][R] with 64 bytes after every 1,024 where R = 256 (two k rows) and 128 after every 8 k
template <int R> constexpr int pair_pitch() { return R == 256 ? 2 * R + 32 : 2 * R; }     // shorts from k to k + 2 (within 8 k)
template <int R> constexpr int stage_shorts() { return kWideK / 2 * pair_pitch<R>() + kWideK / 8 * 64; }
template <int R> __device__ __forceinline__ constexpr int row_at(int k) { return (k >> 1) * pair_pitch<R>() + (k & 1) * R + (k >> 3) * 64; }

// where the 32-byte slot of 16 rows lies within a k row: k .. k + 3 and k + 8 .. k + 11 have to fall into different banks
template <int R> __device__ __forceinline__ int slot_of(int slot, int k) { return R == 256 ? slot ^ (k & 1) : slot ^ (k & 3); }

// an operand's tile on its way: the buffer starts at (r0, k) and ends with the operand, so that rows and k behind it are out of range
template <typename T, int KIND, int R, int THREADS>
struct WideTile {
    static constexpr int kPieces = R * kWideK / 8 / THREADS;
    uint64_t at, end;            // addresses
    uint32_t offset, step;       // of this lane's piece 0; from one piece to the next
    int k0, advance;             // k of piece 0 within the stage (kFlat: of every piece); bytes from stage to stage
    __device__ __forceinline__ WideTile(const Operand& o, int r0, int k_begin, int K, int wave, int lane) {
        const uint64_t p = (uint64_t)o.p;
        if constexpr (KIND == kFlat) {
            const int row = wave * 8 + (lane >> 3), piece = (lane & 7) ^ (row & 7);        // piece i: THREADS / 8 rows further
            k0 = piece * 8;
            offset = (uint32_t)(row * o.pitch + k0) * 2, step = (uint32_t)(THREADS / 8 * o.pitch * 2), advance = kWideK * 2;
            at = p + ((uint64_t)r0 * o.pitch + k_begin) * 2, end = p + (uint64_t)o.rows * o.pitch * 2;
        } else {
            constexpr int PER = R / 8;                                                     // pieces of a k row
            const int id = wave * 64 + lane, k = id / PER, slot = slot_of<R>((id % PER) >> 1, k);   // piece i: THREADS / PER k further
            k0 = k;
            offset = (uint32_t)(k * o.pitch + slot * 16 + (lane & 1) * 8) * 2, step = (uint32_t)(THREADS / PER * o.pitch * 2);
            advance = (int)(kWideK * o.pitch * 2);
            at = p + ((uint64_t)k_begin * o.pitch + r0) * 2, end = p + (uint64_t)K * o.pitch * 2;
        }
    }
    // piece i of the stage from k, which is left to the next stage with the last piece
    __device__ __forceinline__ void fetch(short* stage, int wave, int i, int k, int K) {
        const int64_t left = (int64_t)(end - at);
        const uint32_t records = left <= 0 ? 0 : left < 0x7fffffff ? (uint32_t)left : 0x7fffffffu;
        const i32x4 buffer = {(int)(uint32_t)at, (int)((at >> 32) & 0xffff), (int)records, 0x00027000};
        uint32_t from = offset + i * step;
        if constexpr (KIND == kFlat)
            if (k + kWideK > K) from = k + k0 < K ? from : 0x80000000u;                    // the row goes on with other numbers
        const int load = i * (THREADS / 64) + wave;                                        // 512 shorts: 512 / R k rows of kAcross
        short* dst = stage + (KIND == kFlat ? load * 512 : row_at<R>(load * (512 / R)));
        memory_to_lds(buffer, from, dst);
        if (i == kPieces - 1) at += advance;
    }
};

// memory from `at` to `end`: reads behind it give 0
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer_of(uint64_t at, uint64_t end) {
    const int64_t left = (int64_t)(end - at);
    return __builtin_amdgcn_make_buffer_rsrc((void*)at, 0, left <= 0 ? 0 : left < 0x7fffffff ? (int)left : 0x7fffffff, 0x00027000);
}

// a kAcross8 operand: 8 bytes and their exponent a piece through registers, one stage ahead of the others; LDS holds what a kAcross
// stage would
template <typename T, int R, int THREADS>
struct WideTile<T, kAcross8, R, THREADS> {
    static constexpr int kPieces = R * kWideK / 8 / THREADS, kRows = THREADS / (R / 8);      // k from piece to piece
    Chunk<T, kAcross8> c[kPieces];
    uint64_t at, end, at_e, end_e;
    uint32_t offset, offset_e, step, step_e;
    int to;                       // of piece 0 within a stage
    __device__ __forceinline__ WideTile(const Operand& o, int r0, int k_begin, int K, int wave, int lane) {
        const int id = wave * 64 + lane, kr = id / (R / 8), piece = id % (R / 8);
        const int64_t pe = o.pitch / kBlock8;
        offset = (uint32_t)(kr * o.pitch + piece * 8), offset_e = (uint32_t)(kr * pe + piece / 4);
        step = (uint32_t)(kRows * o.pitch), step_e = (uint32_t)(kRows * pe);
        at = (uint64_t)o.p + (uint64_t)k_begin * o.pitch + r0, end = (uint64_t)o.p + (uint64_t)K * o.pitch;
        at_e = (uint64_t)o.e + (uint64_t)k_begin * pe + r0 / kBlock8, end_e = (uint64_t)o.e + (uint64_t)K * pe;
        to = row_at<R>(kr) + (slot_of<R>(piece >> 1, kr) << 4) + (piece & 1) * 8;
    }
    // piece i of the next stage; behind the last k: zeros
    __device__ __forceinline__ void load(int i) {
        const uint2 b = __builtin_bit_cast(uint2, __builtin_amdgcn_raw_buffer_load_b64(buffer_of(at, end), offset + i * step, 0, 0));
        __builtin_memcpy(c[i].v, &b, 8);
        c[i].e = (int8_t)__builtin_amdgcn_raw_buffer_load_b8(buffer_of(at_e, end_e), offset_e + i * step_e, 0, 0);
        if (i == kPieces - 1) at += (uint64_t)step * kPieces, at_e += (uint64_t)step_e * kPieces;
    }
    __device__ __forceinline__ void put(short* stage, int i) {
        s16x8 out[3];
        split_chunk<T, kAcross8>(c[i], out);
        static_assert(kRows % 8 == 0, "the permutation of the slots repeats every 4 k, the gaps every 8");
        *(s16x8*)(stage + to + row_at<R>(i * kRows)) = out[0];
    }
};

template <int KIND, int R>
__device__ __forceinline__ s16x8 wide_fragment(const short* stage, int row0, int k, int lane) {
    if constexpr (KIND == kFlat) {
        return *(const s16x8*)(stage + flat_at<kWideK>(row0 + (lane & 15), (k >> 3) + (lane >> 4)));
    } else {
        const int kr = 8 * (lane >> 4) + ((lane & 15) >> 2);
        const short* p = stage + row_at<R>(k) + row_at<R>(kr) + (slot_of<R>(row0 >> 4, kr) << 4) + ((lane & 3) << 2);
        const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)p);
        const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + 2 * pair_pitch<R>()));
        return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
    }
}

// A wave's 16 FX x 64 outputs through LDS, 16 rows of fp32 sums at a time, so that a lane stores 8 neighbours and a row is stored whole:
// a lane of an accumulator holds m = l % 16, n = 4 (l / 16) .. + 3. Each wave has its own 16 x 68 floats (the pitch spreads the banks).
template <typename T, int FX>
__device__ __forceinline__ void store_tile(const f32x4 (&acc)[4][FX], float* lds, int wave, int lane, int m0, int n0, const Shape& s, const Epilogue& ep) {
    constexpr int P = 68;
    float* tile = lds + wave * (16 * P);
    const int n = n0 + 8 * (lane & 7);
    float bias[8];
    load_bias<T, 8>(ep, n, s.N, bias);
#pragma unroll
    for (int i = 0; i < FX; ++i) {
#pragma unroll
        for (int j = 0; j < 4; ++j) *(f32x4*)(tile + (lane & 15) * P + 16 * j + 4 * (lane >> 4)) = acc[j][i];
#pragma unroll 1
        for (int r = 0; r < 2; ++r) {
            const int row = 8 * r + (lane >> 3), m = m0 + 16 * i + row;
            const float* from = tile + row * P + 8 * (lane & 7);
            const f32x4 a = *(const f32x4*)from, b = *(const f32x4*)(from + 4);
            float v[8] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
            if (m >= s.M || n >= s.N) continue;
            if (ep.partial) store_piece<float, 8>(ep.partial + ((int64_t)blockIdx.y * s.M + m) * s.N + n, s.N - n, v);
            else finish<T, 8>(ep, m, n, s.N, v, bias);
        }
    }
}

// R x R outputs by WAVES waves, two across m; a wave: 16 FX x 16 FY of them
template <typename T, int XK, int YK, int R>
__global__ __launch_bounds__(R == 256 ? 512 : 256, 2) void k_product_wide(Operand X, Operand Y, Shape s, Epilogue ep) {
    constexpr int BK = kWideK, THREADS = R == 256 ? 512 : 256, WAVES = THREADS / 64, FX = R / 32, FY = R / (8 * WAVES);
    typedef WideTile<T, XK, R, THREADS> TileX;
    typedef WideTile<T, YK, R, THREADS> TileY;
    constexpr int kPieces = TileX::kPieces;
    __shared__ __attribute__((aligned(16))) short lds[2][2][stage_shorts<R>()];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    int tm, tn;
    tile_of(blockIdx.x, s, tm, tn);
    const int m0 = tm * R, n0 = tn * R;
    const int k_begin = blockIdx.y * s.k_slice, k_end = s.K - k_begin < s.k_slice ? s.K : k_begin + s.k_slice;
    const int steps = (k_end - k_begin + BK - 1) / BK;
    const int wm = (wave & 1) * (16 * FX), wn = (wave >> 1) * (16 * FY);
    TileX tx(X, m0, k_begin, s.K, wave, lane);
    TileY ty(Y, n0, k_begin, s.K, wave, lane);
    f32x4 acc[FY][FX] = {};                               // [n][m]
    // two sets of fragments; beside a kAcross8 operand's pieces there are registers for one of X's, refilled behind its last use
    constexpr int A1 = YK == kAcross8 ? 0 : 1;
    s16x8 fx[A1 + 1][FX], fy[2][FY];
    // fetches and fragment reads run past the last step without a branch: nobody uses what they bring
#pragma unroll
    for (int st = 0; st < 2; ++st) {
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            tx.fetch(lds[st][0], wave, i, k_begin + st * BK, s.K);
            if constexpr (YK != kAcross8) ty.fetch(lds[st][1], wave, i, k_begin + st * BK, s.K);
            else ty.load(i);
        }
        if constexpr (YK == kAcross8)
#pragma unroll
            for (int i = 0; i < kPieces; ++i) ty.put(lds[st][1], i);
    }
    if constexpr (YK != kAcross8) {
        static_assert(2 * kPieces == 8, "the second stage's loads");
        asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
    } else {
#pragma unroll
        for (int i = 0; i < kPieces; ++i) ty.load(i);
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    }
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
#pragma unroll
    for (int j = 0; j < FY; ++j) fy[0][j] = wide_fragment<YK, R>(lds[0][1], wn + 16 * j, 0, lane);
#pragma unroll
    for (int g = 0; g < FX; ++g) fx[0][g] = wide_fragment<XK, R>(lds[0][0], wm + 16 * g, 0, lane);
    for (int t = 0; t < steps; ++t) {
        short *xs = lds[t & 1][0], *ys = lds[t & 1][1];
        const short *xn = lds[(t + 1) & 1][0], *yn = lds[(t + 1) & 1][1];
#pragma unroll
        for (int g = 0; g < FX; ++g) {                    // first 32 k; the second's fragments on their way
            if (g < FY) fy[1][g] = wide_fragment<YK, R>(ys, wn + 16 * g, 32, lane);
            if (A1) fx[A1][g] = wide_fragment<XK, R>(xs, wm + 16 * g, 32, lane);
#pragma unroll
            for (int j = 0; j < FY; ++j) acc[j][g] = mfma<T>(fy[0][j], fx[0][g], acc[j][g]);
            if (!A1) fx[0][g] = wide_fragment<XK, R>(xs, wm + 16 * g, 32, lane);
        }
        // the order to issue them in: a group of reads, the instructions that cover it (+2 - 4 % with transposing reads)
        constexpr int RX = XK == kFlat ? 1 : 2, RB = RX + (YK == kFlat ? 1 : 2);
#pragma unroll
        for (int g = 0; A1 && g < FY; ++g) {
            __builtin_amdgcn_sched_group_barrier(0x100, RB, 0);
            __builtin_amdgcn_sched_group_barrier(0x8, FY, 0);
        }
#pragma unroll
        for (int g = FY; A1 && g < FX; ++g) {
            __builtin_amdgcn_sched_group_barrier(0x100, RX, 0);
            __builtin_amdgcn_sched_group_barrier(0x8, FY, 0);
        }
        // every wave has read all of this stage, and this wave's pieces of the next one have arrived
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        const int k = k_begin + (t + 2) * BK;
#pragma unroll
        for (int g = 0; g < FX; ++g) {
            if (g < kPieces) {
                tx.fetch(xs, wave, g, k, s.K);
                if constexpr (YK != kAcross8) ty.fetch(ys, wave, g, k, s.K);
                else ty.put(ys, g), ty.load(g);
            }
            if (g < FY) fy[0][g] = wide_fragment<YK, R>(yn, wn + 16 * g, 0, lane);
            if (A1) fx[0][g] = wide_fragment<XK, R>(xn, wm + 16 * g, 0, lane);
#pragma unroll
            for (int j = 0; j < FY; ++j) acc[j][g] = mfma<T>(fy[1][j], fx[A1][g], acc[j][g]);
            if (!A1) fx[0][g] = wide_fragment<XK, R>(xn, wm + 16 * g, 0, lane);
        }
    }
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");      // nothing is on its way to LDS any more, and nobody reads it
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    static_assert(FY == 4, "64 columns a wave");
    store_tile<T, FX>(acc, (float*)&lds[0][0][0], wave, lane, m0 + wm, n0 + wn, s, ep);
}

// ---- fp32: 256 x 128 outputs by eight waves, the operands split while they are staged ---------------------------------------
// A wave owns 64 x 64 outputs; 24 fragment reads (three planes of each operand) feed 96 matrix instructions. Two stages of 32 k: while
// one is multiplied, the numbers of the next, which are in registers already, are split and stored to the other, and those of the
// one after it are fetched; one barrier a stage. 24 numbers a thread and stage take about 220 vector instructions, beside the matrix
// instructions of both waves of the SIMD (4096^3: 217 TFLOP/s, matrix pipe busy 0.59 of the cycles at 1.9 GHz; the two waves in
// opposite phases, one staging while the other multiplies, measured the same). Buffer loads, as above; rows of at most 2^21 numbers,
// kFlat ones a multiple of 8.
constexpr int kSplitM = 256, kSplitN = 128, kSplitK = 32, kSplitThreads = 512;
constexpr int64_t kSplitMaxPitch = 1 << 21;

template <int KIND, int R>
struct SplitTile {
    static constexpr int kPieces = R * kSplitK / 8 / kSplitThreads, P = KIND == kAcross8 ? 1 : 3, kShorts = P * R * kSplitK;
    static constexpr int kSize = KIND == kAcross8 ? 1 : 4;
    Chunk<float, KIND> c[kPieces];
    uint64_t at, end, at_e, end_e;
    uint32_t offset, step, offset_e, step_e;
    int k0, to;                   // k of the pieces (kFlat) within the stage; where piece 0 goes
    int64_t advance, advance_e;
    __device__ __forceinline__ SplitTile(const Operand& o, int r0, int k_begin, int K, int tid) {
        const uint64_t p = (uint64_t)o.p;
        at_e = end_e = 0, offset_e = step_e = 0, advance_e = 0, k0 = 0;
        if constexpr (KIND == kFlat) {
            const int row = tid / (kSplitK / 8), piece = tid % (kSplitK / 8);               // piece i: 128 rows further
            k0 = piece * 8, to = flat_at<kSplitK>(row, piece);
            offset = (uint32_t)(row * o.pitch + k0) * 4, step = (uint32_t)(kSplitThreads / (kSplitK / 8) * o.pitch * 4), advance = kSplitK * 4;
            at = p + ((uint64_t)r0 * o.pitch + k_begin) * 4, end = p + (uint64_t)o.rows * o.pitch * 4;
        } else {
            const int k = tid / (R / 8), piece = tid % (R / 8);                             // piece i: kSplitThreads / (R / 8) k further
            to = across_at<R>(k, piece >> 1) + (piece & 1) * 8;
            offset = (uint32_t)(k * o.pitch + piece * 8) * kSize, step = (uint32_t)(kSplitThreads / (R / 8) * o.pitch) * kSize;
            advance = (int64_t)kSplitK * o.pitch * kSize;
            at = p + ((uint64_t)k_begin * o.pitch + r0) * kSize, end = p + (uint64_t)K * o.pitch * kSize;
            if constexpr (KIND == kAcross8) {
                const int64_t pe = o.pitch / kBlock8;
                offset_e = (uint32_t)(k * pe + piece / 4), step_e = (uint32_t)(kSplitThreads / (R / 8) * pe), advance_e = kSplitK * pe;
                at_e = (uint64_t)o.e + (uint64_t)k_begin * pe + r0 / kBlock8, end_e = (uint64_t)o.e + (uint64_t)K * pe;
            }
        }
    }
    // piece i of the stage from k
    __device__ __forceinline__ void load(int i, int k, int K) {
        const __amdgpu_buffer_rsrc_t b = buffer_of(at, end);
        uint32_t from = offset + i * step;
        if constexpr (KIND == kFlat)
            if (k + kSplitK > K) from = k + k0 < K ? from : 0x80000000u;                    // the row goes on with other numbers
        if constexpr (KIND == kAcross8) {
            const auto v = __builtin_amdgcn_raw_buffer_load_b64(b, from, 0, 0);
            __builtin_memcpy(c[i].v, &v, 8);
            c[i].e = (int8_t)__builtin_amdgcn_raw_buffer_load_b8(buffer_of(at_e, end_e), offset_e + i * step_e, 0, 0);
        } else {
            const auto lo = __builtin_amdgcn_raw_buffer_load_b128(b, from, 0, 0), hi = __builtin_amdgcn_raw_buffer_load_b128(b, from + 16, 0, 0);
            __builtin_memcpy(c[i].v, &lo, 16);
            __builtin_memcpy(c[i].v + 4, &hi, 16);
        }
        if (i == kPieces - 1) at += advance, at_e += advance_e;
    }
    __device__ __forceinline__ void put(short* stage, int i) {
        constexpr int kMore = KIND == kFlat ? kSplitThreads / (kSplitK / 8) * kSplitK : kSplitThreads / (R / 8) * R;   // shorts from piece to piece
        static_assert(KIND == kFlat || kPieces == 1 || kSplitThreads / (R / 8) % 8 == 0, "the permutation repeats");
        s16x8 out[3];
        split_chunk<float, KIND>(c[i], out);
#pragma unroll
        for (int p = 0; p < P; ++p) *(s16x8*)(stage + p * (R * kSplitK) + to + i * kMore) = out[p];
    }
};

template <int XK, int YK>
__global__ __launch_bounds__(kSplitThreads, 2) void k_product_split(Operand X, Operand Y, Shape s, Epilogue ep) {
    typedef SplitTile<XK, kSplitM> TileX;
    typedef SplitTile<YK, kSplitN> TileY;
    constexpr int BK = kSplitK, PX = TileX::P, PY = TileY::P;
    static_assert(TileX::kPieces == 2 && TileY::kPieces == 1, "three pieces a thread");
    __shared__ __attribute__((aligned(16))) short lds[2][TileX::kShorts + TileY::kShorts];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    int tm, tn;
    tile_of(blockIdx.x, s, tm, tn);
    const int m0 = tm * kSplitM, n0 = tn * kSplitN;
    const int k_begin = blockIdx.y * s.k_slice, k_end = s.K - k_begin < s.k_slice ? s.K : k_begin + s.k_slice;
    const int steps = (k_end - k_begin + BK - 1) / BK;
    const int wm = (wave & 3) * 64, wn = (wave >> 2) * 64;
    TileX tx(X, m0, k_begin, s.K, tid);
    TileY ty(Y, n0, k_begin, s.K, tid);
    f32x4 acc[4][4] = {};                                 // [n][m]
    tx.load(0, k_begin, s.K), tx.load(1, k_begin, s.K), ty.load(0, k_begin, s.K);
    tx.put(lds[0], 0), tx.put(lds[0], 1), ty.put(lds[0] + TileX::kShorts, 0);
    tx.load(0, k_begin + BK, s.K), tx.load(1, k_begin + BK, s.K), ty.load(0, k_begin + BK, s.K);
    for (int t = 0; t < steps; ++t) {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();                     // this stage is stored, and nobody reads the other one
        asm volatile("" ::: "memory");
        const short *xs = lds[t & 1], *ys = xs + TileX::kShorts;
        short* next = lds[(t + 1) & 1];
        const int k = k_begin + (t + 2) * BK;
        s16x8 fx[PX][4], fy[2][PY];
#pragma unroll
        for (int p = 0; p < PY; ++p) fy[0][p] = fragment<YK, BK, kSplitN>(ys + p * (kSplitN * BK), wn, 0, lane);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int p = 0; p < PX; ++p) fx[p][i] = fragment<XK, BK, kSplitM>(xs + p * (kSplitM * BK), wm + 16 * i, 0, lane);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (j < 3) {
#pragma unroll
                for (int p = 0; p < PY; ++p) fy[(j + 1) & 1][p] = fragment<YK, BK, kSplitN>(ys + p * (kSplitN * BK), wn + 16 * (j + 1), 0, lane);
            }
            // past the last step nobody uses what these bring
            if (j < 2) tx.put(next, j), tx.load(j, k, s.K);
            if (j == 2) ty.put(next + TileX::kShorts, 0), ty.load(0, k, s.K);
#pragma unroll
            for (int px = PX - 1; px >= 0; --px)          // small products first
#pragma unroll
                for (int py = PY - 1; py >= 0; --py)
                    if (px + py <= 2)
#pragma unroll
                        for (int i = 0; i < 4; ++i) acc[j][i] = mfma<bf16>(fy[j & 1][py], fx[px][i], acc[j][i]);
        }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    sums_again<XK, YK>(acc, X, Y, m0 + wm, n0 + wn, k_begin, k_end, lane);
    store_tile<float, 4>(acc, (float*)&lds[0][0], wave, lane, m0 + wm, n0 + wn, s, ep);
}

// ---- few rows: y for M <= 16 MT, the weights read once ----------------------------------------------------------------------
// Bound by the weights' bytes. A workgroup owns 16 features; its waves take turns at 32 kAhead k, whose pieces of 16 rows of W it
// fetches together, straight into the registers of the matrix instruction - no LDS on the way, no barrier until the waves' sums
// are added up, in their order, by LDS (one row, 4096 x 4096 bf16: 8.5 us, 3.9 TB/s). fp32: the fp32 instruction, eight times for
// 32 k (lane l has k = 8 (l / 16) + i for the i-th, in both operands); there is time for it beside the loads, and the split would cost
// more vector work than that.
template <typename T, int MT, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void k_rows(Operand X, Operand Y, Shape s, Epilogue ep) {
    constexpr int kAhead = __is_same(T, float) ? (MT == 1 ? 4 : 2) : (MT == 1 ? 8 : MT == 2 ? 4 : 2);
    __shared__ __attribute__((aligned(16))) float sums[WAVES][MT][16][16];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r = lane & 15, kl = 8 * (lane >> 4);
    const int n0 = blockIdx.x * 16;
    const int k_begin = blockIdx.y * s.k_slice, k_end = s.K - k_begin < s.k_slice ? s.K : k_begin + s.k_slice;
    // rows past the end: the last one again, its sums are not stored
    const T* w = (const T*)Y.p + (int64_t)(n0 + r < s.N ? n0 + r : s.N - 1) * Y.pitch + kl;
    const T* x[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) x[i] = (const T*)X.p + (int64_t)(16 * i + r < s.M ? 16 * i + r : s.M - 1) * X.pitch + kl;
    f32x4 acc[MT] = {};
    struct Piece8 { T v[8]; };
    const auto multiply = [&](const Piece8& a, const Piece8& b, f32x4& c) {
        if constexpr (__is_same(T, float)) {
#pragma unroll
            for (int i = 0; i < 8; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.v[i], b.v[i], c, 0, 0, 0);
        } else {
            c = mfma<T>(__builtin_bit_cast(s16x8, a), __builtin_bit_cast(s16x8, b), c);
        }
    };
    int k = k_begin + wave * 32 * kAhead;
    for (; k + 32 * kAhead <= k_end; k += WAVES * 32 * kAhead) {
        Piece8 pw[kAhead], px[kAhead][MT];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) __builtin_memcpy(&pw[u], w + k + 32 * u, sizeof(Piece8));
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
#pragma unroll
            for (int i = 0; i < MT; ++i) __builtin_memcpy(&px[u][i], x[i] + k + 32 * u, sizeof(Piece8));
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
#pragma unroll
            for (int i = 0; i < MT; ++i) multiply(pw[u], px[u][i], acc[i]);
    }
    for (const int turn = k + 32 * kAhead; k < k_end && k < turn; k += 32) {      // the slice's end, by the wave whose turn it is
        Piece8 pw, px;
        const auto part = [&](const T* from, Piece8& p) {
            if (k + kl + 8 <= k_end) {
                __builtin_memcpy(&p, from + k, sizeof p);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) p.v[i] = k + kl + i < k_end ? from[k + i] : (T)0.f;
            }
        };
        part(w, pw);
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            part(x[i], px);
            multiply(pw, px, acc[i]);
        }
    }
#pragma unroll
    for (int i = 0; i < MT; ++i) *(f32x4*)&sums[wave][i][r][4 * (lane >> 4)] = acc[i];      // [m][n]
    __syncthreads();
    for (int id = tid; id < 64 * MT; id += 64 * WAVES) {
        const int m = id >> 2, n = n0 + 4 * (id & 3);
        if (m >= s.M || n >= s.N) continue;
        float v[4] = {}, b[4];
#pragma unroll
        for (int u = 0; u < WAVES; ++u) {
            const f32x4 t = *(const f32x4*)&sums[u][m >> 4][m & 15][4 * (id & 3)];
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] += t[i];
        }
        if (ep.partial) {
            store_piece<float, 4>(ep.partial + ((int64_t)blockIdx.y * s.M + m) * s.N + n, s.N - n, v);
        } else {
            load_bias<T, 4>(ep, n, s.N, b);
            finish<T, 4>(ep, m, n, s.N, v, b);
        }
    }
}

// the slices of a cut contraction, added in ascending order, and the epilogue
template <typename T>
__global__ __launch_bounds__(256) void k_join(Shape s, Epilogue ep) {
    const int quads = (s.N + 3) / 4;
    const int64_t n_q = (int64_t)s.M * quads;
    for (int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x; id < n_q; id += (int64_t)gridDim.x * 256) {
        const int64_t m = id / quads;
        const int n = (int)(id - m * quads) * 4;
        float v[4] = {}, t[4];
        for (int z = 0; z < s.slices; ++z) {
            load_piece<float, 4>(ep.partial + (z * (int64_t)s.M + m) * s.N + n, s.N - n, t);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] += t[i];
        }
        load_bias<T, 4>(ep, n, s.N, t);
        finish<T, 4>(ep, m, n, s.N, v, t);
    }
}

// dz = dy act'(z) and the slices' sums of its columns: one pass, bound by its bytes. A workgroup: PIECES column pieces x 256 / PIECES
// rows at a time, the loads of kRows of those together. 32 pieces; 8 where one slice has all rows, so that the activation's
// arithmetic is spread over more workgroups (gelu, 128 x 200 fp16: 14.9 -> 7.8 us, 256 x 4096 bf16: 28.7 -> 9.0). 8192 x 8192 bf16,
// gelu, from memory: 102 us for 402 MB, 3.9 TB/s.
// dz is rounded to the tensors' type: it is the matrix instruction's operand, and a second part of it would double both products (8192 x
// 2048 -> 8192 bf16: 470 us more of 795). dx and dW are then off by two roundings, dz's and their own, where the sums alone would leave
// one: relative L2 2.42e-3 against 1.66e-3 in bf16, 3.0e-4 against 2.1e-4 in fp16 - as the stock ops of the type are. db has dz in fp32.
constexpr int kRows = 4;

// V elements from p as they are in memory, of which `room` are the tensor's: past a row's end those of the next one, whose sums are
// not stored. No conversion in here: it would wait for this load before the next one starts.
template <typename T, int V>
__device__ __forceinline__ void load_raw(const T* __restrict__ p, int64_t room, T (&v)[V]) {
    if (room >= V) {
        __builtin_memcpy(v, p, sizeof v);
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = i < room ? p[i] : (T)0.f;
    }
}

template <typename T, int PIECES>
__global__ __launch_bounds__(256) void k_act_grad(const T* __restrict__ dy, const T* __restrict__ z, T* __restrict__ dz, float* __restrict__ partial,
                                                  T* __restrict__ db, int64_t M, int N, int act, int rows) {
    constexpr int V = Piece<T>::kN, STRANDS = 256 / PIECES;
    __shared__ float red[STRANDS][PIECES * V];
    const int piece = threadIdx.x % PIECES, strand = threadIdx.x / PIECES;
    const int64_t n = ((int64_t)blockIdx.x * PIECES + piece) * V, left = N - n;
    const int64_t begin = (int64_t)blockIdx.y * rows, end = begin + rows < M ? begin + rows : M;
    float s[V] = {};
    if (left > 0)
        for (int64_t m0 = begin + strand; m0 < end; m0 += STRANDS * kRows) {
            T raw[2][kRows][V];
#pragma unroll
            for (int r = 0; r < kRows; ++r) {
                const int64_t m = m0 + STRANDS * r, at = m * N + n, room = m < end ? M * N - at : 0;
                load_raw<T, V>(dy + at, room, raw[0][r]);
                if (z) load_raw<T, V>(z + at, room, raw[1][r]);
            }
#pragma unroll
            for (int r = 0; r < kRows; ++r) {
                const int64_t m = m0 + STRANDS * r;
                if (m >= end) break;
                float g[V], a[V];
#pragma unroll
                for (int i = 0; i < V; ++i) g[i] = (float)raw[0][r][i], a[i] = z ? (float)raw[1][r][i] : 0.f;
                if (z) act_slopes(g, a, act);
                if (dz) store_piece<T, V>(dz + m * N + n, left, g);         // dz NULL: the column sums alone are wanted
#pragma unroll
                for (int i = 0; i < V; ++i) s[i] += g[i];                   // before dz is rounded to its type
            }
        }
    if (!partial && !db) return;
#pragma unroll
    for (int i = 0; i < V; ++i) red[strand][piece * V + i] = s[i];
    __syncthreads();
    for (int c = threadIdx.x; c < PIECES * V; c += 256) {
        float t = red[0][c];
#pragma unroll
        for (int w = 1; w < STRANDS; ++w) t += red[w][c];
        const int64_t col = (int64_t)blockIdx.x * PIECES * V + c;
        if (col >= N) continue;
        if (db) db[col] = (T)t;                                             // one slice: nothing to add up
        else partial[(int64_t)blockIdx.y * N + col] = t;
    }
}

template <typename T>
__global__ __launch_bounds__(256) void k_columns_join(const float* __restrict__ partial, int slices, int N, T* __restrict__ out) {
    __shared__ float s[8][32];
    const int col = threadIdx.x & 31, strand = threadIdx.x >> 5, n = blockIdx.x * 32 + col;
    float acc = 0.f;
    if (n < N)
#pragma unroll 8
        for (int g = strand; g < slices; g += 8) acc += partial[(int64_t)g * N + n];
    s[strand][col] = acc;
    __syncthreads();
    if (strand || n >= N) return;
#pragma unroll
    for (int k = 1; k < 8; ++k) acc += s[k][col];
    out[n] = (T)acc;
}

// ---- plans ----------------------------------------------------------------------------------
struct Plan {
    int tm, tn;                  // outputs of a workgroup
    bool wide;                   // the large forms: k_product_wide, k_product_split
    Shape s;
    int64_t ws() const { return s.slices > 1 ? (int64_t)s.slices * s.M * s.N * 4 : 0; }
};

// The form, by the number of workgroups that it gives the 256 CUs, and the cut of the contraction where there are fewer than one
// (two of the smaller forms) for each: at most 16 slices of at least eight k steps. `wide`: the operands suit the large forms (see
// there); `packed`: one of them comes in 8 bits. Measured, both sides of each border (us; more points in profiles/dense_borders.txt):
//   16 bits, 256 x 256 from 192 tiles on: 8192 x 1024 outputs, K 4096 (128 tiles): 92, cut in two 82, in 128 x 128 67; x 1280 (160
//            tiles, the one point where the other form is ahead): 89 against 104; x 1536 (192): 93 against 107; 8192 x 8192, K 2048:
//            224 against 277. With an operand in 8 bits, whose conversion the larger tile halves, also cut: 1024 x 4096, K 8192: 93
//            against 104; 2048 x 2048, K 4096: 63 against 64
//   16 bits, 128 x 128 where they reach 256 workgroups, cut in four at most: 2048^3: 28 against 34 in 64 x 64; 2048 x 1536, K 1024
//            (192, too few): 14.9 against 16.7; 1024^3 (64): 13.5 against 10.3. A cut form costs its join: 2048 x 1024, K 2048 in two 25
//            against 21 in 64 x 64. Two workgroups a CU where each has 48 steps left: 1024 x 4096, K 8192: 79 against 90, K 6144: 64
//            against 68; K 4096 (32 steps): 50 against 47
//   fp32, 256 x 128 where they reach 192 workgroups, cut from 96 tiles or K 2048 on: 1024 x 1024 outputs, K 4096: 65 against 75 in
//            64 x 64; 4096 x 1024, K 1024 (128 tiles): 63 - 66 against 63; 2048 x 1536 (96): 55 against 49; 2048 x 1024 (64): 42 against
//            37; 1024^3: 34 against 28; uncut 4096 x 2048, K 512 (256): 53 against 62, x 1536 (192): 46 against 49
Plan plan_of(int64_t M, int64_t N, int64_t K, int32_t dtype, bool wide, bool packed) {
    Plan p;
    const int bk = dtype == URSA_F32 ? 32 : 64;
    const int64_t steps = (K + bk - 1) / bk, most = steps / 8 < 1 ? 1 : steps / 8 < 16 ? steps / 8 : 16;
    const auto tiles_of = [&](int tm, int tn) { return ((M + tm - 1) / tm) * ((N + tn - 1) / tn); };
    const int64_t big = tiles_of(128, 128);
    p.tm = p.tn = big >= 256 ? 128 : 64;
    p.wide = false;
    if (wide && dtype == URSA_F32) {
        const int64_t n = tiles_of(kSplitM, kSplitN);
        if (n >= 192 || (n * most >= 192 && (n >= 96 || steps >= 64))) p.tm = kSplitM, p.tn = kSplitN, p.wide = true;
    } else if (wide) {
        const int64_t n = tiles_of(256, 256);
        if (n >= 192 || (packed && n * most >= 192)) p.tm = p.tn = 256;
        else if (big * (most < 4 ? most : 4) >= 256) p.tm = p.tn = 128;
        p.wide = p.tm >= 128;
    }
    p.s.M = (int)M, p.s.N = (int)N, p.s.K = (int)K;
    p.s.tiles_m = (int)((M + p.tm - 1) / p.tm), p.s.tiles_n = (int)((N + p.tn - 1) / p.tn);
    const int64_t tiles = (int64_t)p.s.tiles_m * p.s.tiles_n, want = p.wide && (p.tm == 256 || tiles < 256 || steps < 96) ? 256 : 512;
    int64_t cut = tiles < want && tiles ? want / tiles : 1;
    if (cut > most) cut = most;
    const int64_t per = (steps + cut - 1) / cut;
    p.s.k_slice = (int)((per > 0 ? per : 1) * bk);
    p.s.slices = per > 0 ? (int)((steps + per - 1) / per) : 1;
    return p;
}

template <typename T>
int join(const Shape& s, const Epilogue& ep, hipStream_t st) {
    const int64_t quads = (int64_t)s.M * ((s.N + 3) / 4), blocks = (quads + 255) / 256;
    hipLaunchKernelGGL(k_join<T>, dim3((unsigned)(blocks < 8192 ? blocks : 8192)), dim3(256), 0, st, s, ep);
    return launch_status();
}

// whether an operand (rows of `pitch` elements) suits the large forms
bool suits(int32_t dtype, int kind, const void* p, int64_t pitch) {
    return dtype == URSA_F32 ? pitch <= kSplitMaxPitch && (kind != kFlat || pitch % 8 == 0) : pitch % 8 == 0 && pitch <= kWideMaxPitch && ((uintptr_t)p & 15) == 0;
}

// Few rows: 16, 32 or 64 of them. Four waves a workgroup of 16 features where those give two workgroups a CU, up to sixteen where
// there are fewer, and the contraction cut (at least 2,048 k a slice) where sixteen waves do not fill the CUs either.
int rows_form(int64_t M) { return M <= 16 ? 1 : M <= 32 ? 2 : M <= 64 ? 4 : 0; }

Shape rows_shape(int64_t M, int64_t N, int64_t K) {
    Shape s = {};
    s.M = (int)M, s.N = (int)N, s.K = (int)K;
    const int64_t groups = (N + 15) / 16;
    int64_t cut = groups < 128 ? 256 / groups : 1;
    if (cut > K / 2048) cut = K / 2048;
    if (cut > 16) cut = 16;
    if (cut < 1) cut = 1;
    s.k_slice = (int)(((K + cut - 1) / cut + 31) / 32 * 32);
    if (s.k_slice < 32) s.k_slice = 32;
    s.slices = (int)((K + s.k_slice - 1) / s.k_slice);
    if (s.slices < 1) s.slices = 1;
    return s;
}

template <typename T, int MT>
int rows_product(const Operand& x, const Operand& y, const Shape& s, Epilogue ep, hipStream_t st) {
    if (s.slices == 1) ep.partial = nullptr;
    const unsigned groups = (unsigned)((s.N + 15) / 16);
    const dim3 grid(groups, (unsigned)s.slices);
    if (groups >= 512) hipLaunchKernelGGL((k_rows<T, MT, 4>), grid, dim3(256), 0, st, x, y, s, ep);
    else if (groups >= 128) hipLaunchKernelGGL((k_rows<T, MT, 8>), grid, dim3(512), 0, st, x, y, s, ep);
    else hipLaunchKernelGGL((k_rows<T, MT, 16>), grid, dim3(1024), 0, st, x, y, s, ep);
    const int rc = launch_status();
    return rc || s.slices == 1 ? rc : join<T>(s, ep, st);
}

template <typename T, int XK, int YK>
int product(const Operand& x, const Operand& y, const Plan& p, Epilogue ep, hipStream_t st) {
    if (p.s.slices == 1) ep.partial = nullptr;
    const dim3 grid((unsigned)(p.s.tiles_m * p.s.tiles_n), (unsigned)p.s.slices);
    if (p.wide) {
        if constexpr (__is_same(T, float)) hipLaunchKernelGGL((k_product_split<XK, YK>), grid, dim3(kSplitThreads), 0, st, x, y, p.s, ep);
        else if (p.tm == 256) hipLaunchKernelGGL((k_product_wide<T, XK, YK, 256>), grid, dim3(512), 0, st, x, y, p.s, ep);
        else hipLaunchKernelGGL((k_product_wide<T, XK, YK, 128>), grid, dim3(256), 0, st, x, y, p.s, ep);
    } else if (p.tm == 128) {
        hipLaunchKernelGGL((k_product<T, XK, YK, 128>), grid, dim3(256), 0, st, x, y, p.s, ep);
    } else {
        hipLaunchKernelGGL((k_product<T, XK, YK, 64>), grid, dim3(256), 0, st, x, y, p.s, ep);
    }
    const int rc = launch_status();
    return rc || p.s.slices == 1 ? rc : join<T>(p.s, ep, st);
}

#define URSA_LINEAR_TYPES(dtype, call) (dtype == URSA_F32 ? call(float) : dtype == URSA_BF16 ? call(bf16) : call(f16))

// The kernels count rows and k in 32 bits, a few steps past the end; a launch has less than 2^32 threads in a dimension.
constexpr int64_t kMaxRows = INT32_MAX - 8192, kMaxFeatures = 1 << 27;
bool tiles_fit(int64_t M, int64_t N) { return ((M + 127) / 128) * ((N + 127) / 128) < 1 << 24; }      // (64 x 64 is for few tiles)

// 0: go on; 1: nothing to write; < 0: an error
int check(int64_t M, int64_t N, int64_t K, int32_t dtype) {
    if (dtype < URSA_F32 || dtype > URSA_F16) return URSA_EFLAGS;
    if (M < 0 || N < 0 || K < 0 || M > kMaxRows || N > kMaxFeatures || K > kMaxFeatures || !tiles_fit(M, N)) return URSA_ESIZE;
    return M == 0 || N == 0 ? 1 : 0;
}

bool misaligned(int32_t dtype, uintptr_t pointers) { return pointers & (uintptr_t)(element_size(dtype) - 1); }

int act_rows(int64_t M, int64_t N, int32_t dtype) {       // rows of a slice of k_act_grad: about 2,048 workgroups, 32 rows at least
    const int64_t cols = (N + 32 * 16 / element_size(dtype) - 1) / (32 * 16 / element_size(dtype));
    int64_t slices = 2048 / (cols ? cols : 1);
    if (slices < 1) slices = 1;
    if (slices > 256) slices = 256;
    const int64_t rows = ((M + slices - 1) / slices + 7) / 8 * 8;
    return (int)(M <= 256 ? 256 : rows < 32 ? 32 : rows);         // few rows: one slice, which spares the second launch
}

template <typename T>
int backward(const T* dy, const T* x, const int8_t* q, const int8_t* e, const T* w, const T* z, T* dx, T* dw, T* db, char* ws, int64_t dz_bytes,
             int64_t M, int64_t N, int64_t K, int32_t dtype, int32_t act, hipStream_t st) {
    int rc = URSA_OK;
    T* dz = dz_bytes ? (T*)ws : nullptr;
    float* scratch = (float*)(ws + dz_bytes);
    if (dz || db) {
        const int rows = act_rows(M, N, dtype), slices = (int)((M + rows - 1) / rows), per = (slices == 1 ? 8 : 32) * Piece<T>::kN;
        if (M) {
            hipLaunchKernelGGL((slices == 1 ? k_act_grad<T, 8> : k_act_grad<T, 32>), dim3((unsigned)((N + per - 1) / per), (unsigned)slices), dim3(256), 0, st, dy, act ? z : nullptr, dz,
                               db && slices > 1 ? scratch : nullptr, slices == 1 ? db : nullptr, M, (int)N, act, rows);
            if ((rc = launch_status())) return rc;
        }
        if (db && slices != 1) {
            hipLaunchKernelGGL(k_columns_join<T>, dim3((unsigned)((N + 31) / 32)), dim3(256), 0, st, (const float*)scratch, slices, (int)N, db);
            if ((rc = launch_status())) return rc;
        }
    }
    const T* g = dz ? dz : dy;
    if (dx && M && K) {
        const Operand X{g, nullptr, N, (int)M}, Y{w, nullptr, K, (int)K};
        if ((rc = product<T, kFlat, kAcross>(X, Y, plan_of(M, K, N, dtype, suits(dtype, kFlat, g, N) && suits(dtype, kAcross, w, K), false), {dx, nullptr, nullptr, nullptr, scratch, URSA_ACT_NONE}, st))) return rc;
    }
    if (dw && K) {
        const Epilogue ep{dw, nullptr, nullptr, nullptr, scratch, URSA_ACT_NONE};
        const Operand X{g, nullptr, N, (int)N}, Y{q ? (const void*)q : x, e, q ? (K + kBlock8 - 1) / kBlock8 * kBlock8 : K, (int)K};
        const Plan p = plan_of(N, K, M, dtype, suits(dtype, kAcross, g, N) && (q ? K <= kSplitMaxPitch : suits(dtype, kAcross, x, K)), q != nullptr);
        rc = q ? product<T, kAcross, kAcross8>(X, Y, p, ep, st) : product<T, kAcross, kAcross>(X, Y, p, ep, st);
    }
    return rc;
}

// scratch of a product: what any of its forms takes (the operands' alignment decides)
int64_t most_ws(int64_t M, int64_t N, int64_t K, int32_t dtype) {
    const int64_t a = plan_of(M, N, K, dtype, false, false).ws(), b = plan_of(M, N, K, dtype, true, false).ws(), c = plan_of(M, N, K, dtype, true, true).ws();
    return a > b ? (a > c ? a : c) : (b > c ? b : c);
}

// of a backward call: dz (with an activation), then what one of its launches needs at a time - they run one after another
struct BwdScratch {
    int64_t dz, rest;
    BwdScratch(int64_t M, int64_t N, int64_t K, int32_t dtype, int32_t act, bool dx, bool dw, bool db) : dz(0), rest(0) {
        if (act && (dx || dw)) dz = (M * N * element_size(dtype) + 255) / 256 * 256;
        if (dx && M && K) rest = most_ws(M, K, N, dtype);
        if (dw && N && K) { const int64_t n = most_ws(N, K, M, dtype); rest = n > rest ? n : rest; }
        if (db) { const int64_t r = act_rows(M, N, dtype), n = (M + r - 1) / r * N * 4; rest = n > rest ? n : rest; }
    }
};

}  // namespace

extern "C" int64_t ursa_linear_ws_bytes(int64_t M, int64_t N, int64_t K, int32_t dtype) {
    if (check(M, N, K, dtype)) return 0;
    if (!rows_form(M)) return most_ws(M, N, K, dtype);
    const Shape s = rows_shape(M, N, K);
    return s.slices > 1 ? (int64_t)s.slices * M * N * 4 : 0;
}

extern "C" int64_t ursa_linear_bwd_ws_bytes(int64_t M, int64_t N, int64_t K, int32_t dtype, int32_t act, int32_t dx, int32_t dw, int32_t db) {
    if (check(M, N, K, dtype) < 0) return 0;
    const BwdScratch s(M, N, K, dtype, act, dx, dw, db);
    return s.dz + s.rest;
}

extern "C" int ursa_linear_act(const void* x, const void* w, const void* bias, const void* residual, void* y, void* z, void* ws, int64_t M,
                               int64_t N, int64_t K, int32_t dtype, int32_t act, ursa_stream_t stream) {
    if (act < URSA_ACT_NONE || act > URSA_ACT_SILU) return URSA_EFLAGS;
    if (int rc = check(M, N, K, dtype)) return rc > 0 ? URSA_OK : rc;
    const Plan p = plan_of(M, N, K, dtype, suits(dtype, kFlat, x, K) && suits(dtype, kFlat, w, K), false);
    const int form = rows_form(M);
    const Shape few = rows_shape(M, N, K);
    if ((K && (!x || !w)) || !y || ((form ? few.slices > 1 : p.s.slices > 1) && !ws)) return URSA_ENULL;
    if (misaligned(dtype, (uintptr_t)x | (uintptr_t)w | (uintptr_t)bias | (uintptr_t)residual | (uintptr_t)y | (uintptr_t)z) || (uintptr_t)ws & 3) return URSA_EALIGN;
    const Operand X{x, nullptr, K, (int)M}, Y{w, nullptr, K, (int)N};
    const Epilogue ep{y, z, bias, residual, (float*)ws, act};
    if (form) {
#define URSA_CALL(T) (form == 1 ? rows_product<T, 1>(X, Y, few, ep, (hipStream_t)stream) : form == 2 ? rows_product<T, 2>(X, Y, few, ep, (hipStream_t)stream) \
                                                                                         : rows_product<T, 4>(X, Y, few, ep, (hipStream_t)stream))
        return URSA_LINEAR_TYPES(dtype, URSA_CALL);
#undef URSA_CALL
    }
#define URSA_CALL(T) product<T, kFlat, kFlat>(X, Y, p, ep, (hipStream_t)stream)
    return URSA_LINEAR_TYPES(dtype, URSA_CALL);
#undef URSA_CALL
}

extern "C" int ursa_linear_bwd(const void* dy, const void* x, const int8_t* q, const int8_t* e, const void* w, const void* z, void* dx, void* dw,
                               void* db, void* ws, int64_t M, int64_t N, int64_t K, int32_t dtype, int32_t act, ursa_stream_t stream) {
    if (act < URSA_ACT_NONE || act > URSA_ACT_SILU) return URSA_EFLAGS;
    if (int rc = check(M, N, K, dtype); rc < 0) return rc;
    if ((dx && !tiles_fit(M, K)) || (dw && !tiles_fit(N, K))) return URSA_ESIZE;
    if (N == 0 || !(dx || dw || db)) return URSA_OK;
    const BwdScratch size(M, N, K, dtype, act, dx, dw, db);
    if (M && (!dy || (act && !z) || (dx && K && !w) || (dw && K && ((x != nullptr) == (q != nullptr) || (q != nullptr) != (e != nullptr))) ||
              (size.dz + size.rest && !ws))) return URSA_ENULL;
    if (misaligned(dtype, (uintptr_t)dy | (uintptr_t)x | (uintptr_t)w | (uintptr_t)z | (uintptr_t)dx | (uintptr_t)dw | (uintptr_t)db) ||
        (uintptr_t)q & 15 || (uintptr_t)ws & 15) return URSA_EALIGN;
#define URSA_CALL(T) backward<T>((const T*)dy, (const T*)x, q, e, (const T*)w, (const T*)z, (T*)dx, (T*)dw, (T*)db, (char*)ws, size.dz, M, N, K, dtype, act, (hipStream_t)stream)
    return URSA_LINEAR_TYPES(dtype, URSA_CALL);
#undef URSA_CALL
}
