// Root-mean-square norm of rows with the residual's addition, on gfx950, forward and backward, and
// with the result in e4m3 and one scale per row for the 8-bit product (linear_8bit.hip):
//
//   r = x + residual,  s = (mean r^2 + eps)^(-1/2),  y = r s w
//   dr = s (w dy - n mean(w dy n)) + g_r with n = r s,  dw = sum over rows of dy n
//
// Bound by memory: every input is read once and every output written once.  A row stays in the
// registers of LPR lanes (4, 8, 16, 64, 256, 512 or 1024: a quarter wavefront for the rows of the weight
// network, up to a whole workgroup of 16 wavefronts), N vectors of 16 bytes per lane, so that the
// second use of a row (after its sum of squares is known) costs no second read.
//
// Sums are taken in float over a lane's elements, then over the lanes by DPP exchanges and, for rows
// wider than a wavefront, through LDS, always in the same order.  dw is summed in registers by
// workgroups that walk over rows, one partial row per workgroup, added up by a second kernel in a
// fixed order: no atomics, the same bits on every run.
//
// Measured, where a large copy moves 5.1 TB/s: with a residual, 81920 x 128 float 30.5 us forward (5.5 TB/s),
// 28 + 4 us backward; 8192 x 4096 bfloat16 43 us and 71 + 4 us; to e4m3, 262144 x 256 bfloat16 88 us
// (5.3).  Few rows are bound by their launches: 2.5 to 4 us for each of the three.
#include "narrow_types.h"

#include <type_traits>

#include "device_info.h"

namespace kvae {

template <int CTRL>
__device__ __forceinline__ float row_exchange(float x) {
    return __builtin_bit_cast(
        float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ float lane_value(float x, int lane) {
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), lane));
}

struct Add {
    __device__ static float of(float a, float b) { return a + b; }
};
struct Max {   // a NaN is passed over
    __device__ static float of(float a, float b) { return fmaxf(a, b); }
};

// OP over the LPR lanes of a row, in every one of them.  slot: LDS of one float per wavefront and
// call site (a row wider than a wavefront only).
template <typename OP, int LPR>
__device__ __forceinline__ float over_row(float v, float* slot) {
    v = OP::of(v, row_exchange<0xB1>(v));            // neighbours, pairs, halves of a row of 16, its mirror
    v = OP::of(v, row_exchange<0x4E>(v));
    if constexpr (LPR > 4) v = OP::of(v, row_exchange<0x141>(v));
    if constexpr (LPR > 8) v = OP::of(v, row_exchange<0x140>(v));
    if constexpr (LPR > 16)
        v = OP::of(OP::of(lane_value(v, 0), lane_value(v, 16)),
                   OP::of(lane_value(v, 32), lane_value(v, 48)));
    if constexpr (LPR > 64) {
        constexpr int WAVES = LPR / 64;
        if ((threadIdx.x & 63) == 0) slot[threadIdx.x >> 6] = v;
        __syncthreads();
        v = slot[0];
#pragma unroll
        for (int i = 1; i < WAVES; ++i) v = OP::of(v, slot[i]);
    }
    return v;
}

struct NormArgs {
    long rows;
    int D;
    const void* x;
    const void* residual;
    long x_row, residual_row;
    const void* weight;
    int weight_f32;
    float eps;
    void* y;             // T, or e4m3 bytes
    float* scale;        // e4m3 only
    void* sum;           // r, or NULL
    float* rstd;         // or NULL
    // backward: r = x (+ residual)
    const void* dy;
    const void* dsum;    // or NULL
    long dy_row, dsum_row;
    void* dx;
    float* partial;      // (gridDim.x, D): dw of each workgroup's rows
};

// Element `at` of the weight, which is float or has the rows' type.
template <typename T>
__device__ __forceinline__ float weight_at(const NormArgs& g, int at) {
    return g.weight_f32 ? static_cast<const float*>(g.weight)[at]
                        : widen(static_cast<const T*>(g.weight)[at]);
}

// V elements of a row from column `at`; columns past D read as zero.
template <typename T, int V>
__device__ __forceinline__ void row_load(const T* row, int at, int D, float (&out)[V]) {
    if (at + V <= D) {
        const Pack<T, V> p = load_pack<T, V>(row + at);
#pragma unroll
        for (int v = 0; v < V; ++v) out[v] = widen(p.v[v]);
    } else {
#pragma unroll
        for (int v = 0; v < V; ++v) out[v] = at + v < D ? widen(row[at + v]) : 0.f;
    }
}
template <typename T, int V>
__device__ __forceinline__ void row_store(T* row, int at, int D, const float (&x)[V]) {
    if (at + V <= D) {
        Pack<T, V> p;
#pragma unroll
        for (int v = 0; v < V; ++v) p.v[v] = narrow<T>(x[v]);
        store_pack<T, V>(row + at, p);
    } else {
#pragma unroll
        for (int v = 0; v < V; ++v)
            if (at + v < D) row[at + v] = narrow<T>(x[v]);
    }
}

// Four floats, at most 448 in size, to four e4m3 bytes (nearest, ties to even).
__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
    int p = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, p, true);
}
constexpr float E4M3_MAX = 448.f;
// the smallest scale is the smallest normal float: its reciprocal is finite, and an all-zero row has
// one too
constexpr float SMALLEST_SCALE = 1.17549435e-38f;
__device__ __forceinline__ float clamp_e4m3(float x) {   // keeps a NaN
    return x > E4M3_MAX ? E4M3_MAX : (x < -E4M3_MAX ? -E4M3_MAX : x);
}
// What a row is multiplied by on its way to codes, to twice float's digits: hi + lo.
struct Factor {
    float hi, lo;
};
// (p + rest) k, rounded once: where a quotient lies next to the middle of two codes, the roundings of a
// chain of float products would decide between them.
__device__ __forceinline__ float times(float p, float rest, Factor k) {
#pragma clang fp contract(off)
    // (contracted, the last sum would hold what t leaves of the product twice)
    const float t = p * k.hi;
    return t + (__builtin_fmaf(p, k.hi, -t) + __builtin_fmaf(p, k.lo, rest * k.hi));
}
template <int V>
__device__ __forceinline__ void row_store_e4m3(uint8_t* row, int at, int D, const float (&x)[V], const float (&rest)[V],
                                               Factor k) {
    uint32_t w[V / 4];
#pragma unroll
    for (int v = 0; v < V; v += 4) {
        float t[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) t[i] = clamp_e4m3(times(x[v + i], rest[v + i], k));
        w[v / 4] = e4m3x4(t[0], t[1], t[2], t[3]);
    }
    if (at + V <= D) {
        Pack<uint8_t, V> p;
        __builtin_memcpy(&p, w, V);
        using R = typename RawVec<V>::type;
        struct __attribute__((packed)) Any { R r; };
        reinterpret_cast<Any*>(row + at)->r = __builtin_bit_cast(R, p);
    } else {
#pragma unroll
        for (int v = 0; v < V; ++v)
            if (at + v < D) row[at + v] = (uint8_t)(w[v / 4] >> (8 * (v % 4)));
    }
}

template <int LPR>
constexpr int norm_block() { return LPR > 256 ? LPR : 256; }

// NORM: the norm above; otherwise rows are only quantised (y = x).
template <typename T, int LPR, int N, bool QUANT, bool NORM>
__global__ void __launch_bounds__(norm_block<LPR>()) norm_forward_kernel(NormArgs g) {
    constexpr int V = 16 / sizeof(T);
    constexpr int RPB = norm_block<LPR>() / LPR;   // rows a workgroup works on together
    __shared__ float slots[3][16];
    const int lane = threadIdx.x % LPR;
    const long row = (long)blockIdx.x * RPB + threadIdx.x / LPR;
    if (LPR <= 64 && row >= g.rows) return;        // (LPR > 64: one row per workgroup, all there)
    float r[N][V], rest[QUANT ? N : 1][V];
    float spread = 1.f;                            // QUANT: y = (r + rest) spread
    const T* x = static_cast<const T*>(g.x) + row * g.x_row;
    const T* res = static_cast<const T*>(g.residual);
    if (NORM && res) res += row * g.residual_row;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int at = (i * LPR + lane) * V;
        row_load<T, V>(x, at, g.D, r[i]);
        if constexpr (NORM) {
            if (res) {
                float b[V];
                row_load<T, V>(res, at, g.D, b);
#pragma unroll
                for (int v = 0; v < V; ++v) r[i][v] += b[v];
            }
        }
    }
    if constexpr (NORM) {
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int v = 0; v < V; ++v) ss += r[i][v] * r[i][v];
        ss = over_row<Add, LPR>(ss, slots[0]);
        const float s = 1.f / sqrtf(ss / (float)g.D + g.eps);
        if (g.rstd && lane == 0) g.rstd[row] = s;
        // QUANT: s = power spread, a power of two (by which a product is exact) and a number in [1, 2)
        float power = s;
        if (QUANT && s >= SMALLEST_SCALE && s < __builtin_inff()) {
            power = __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, s) & 0x7F800000u);
            spread = __builtin_bit_cast(float, (__builtin_bit_cast(uint32_t, s) & 0x007FFFFFu) | 0x3F800000u);
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int at = (i * LPR + lane) * V;
            if (g.sum) row_store<T, V>(static_cast<T*>(g.sum) + row * g.D, at, g.D, r[i]);
            float w[V];
            if (g.weight_f32) {
                row_load<float, V>(static_cast<const float*>(g.weight), at, g.D, w);
            } else {
                row_load<T, V>(static_cast<const T*>(g.weight), at, g.D, w);
            }
#pragma unroll
            for (int v = 0; v < V; ++v) {
                if constexpr (QUANT) {
                    const float n = r[i][v] * power;
                    r[i][v] = n * w[v];
                    rest[i][v] = __builtin_fmaf(n, w[v], -r[i][v]);
                } else {
                    r[i][v] = r[i][v] * s * w[v];
                }
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int v = 0; v < V; ++v) rest[i][v] = 0.f;
    }
    if constexpr (QUANT) {
        float big = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int v = 0; v < V; ++v) big = fmaxf(big, fabsf(r[i][v]));
        big = over_row<Max, LPR>(big, slots[1]);
        const float scale = fmaxf(big * spread * (1.f / E4M3_MAX), SMALLEST_SCALE);
        float more = 0.f;                          // the largest product is big + more
        if constexpr (NORM) {
            more = -__builtin_inff();
#pragma unroll
            for (int i = 0; i < N; ++i)
#pragma unroll
                for (int v = 0; v < V; ++v)
                    if (fabsf(r[i][v]) == big) more = fmaxf(more, r[i][v] < 0.f ? -rest[i][v] : rest[i][v]);
            more = over_row<Max, LPR>(more, slots[2]);
        }
        Factor k = {spread / SMALLEST_SCALE, 0.f};
        if (scale > SMALLEST_SCALE) {
            k.hi = E4M3_MAX / big;                 // spread / scale, in which spread cancels
            if (big < __builtin_inff()) k.lo = (__builtin_fmaf(-k.hi, big, E4M3_MAX) - k.hi * more) / big;
        }
        if (lane == 0) g.scale[row] = scale;
#pragma unroll
        for (int i = 0; i < N; ++i)
            row_store_e4m3<V>(static_cast<uint8_t*>(g.y) + row * g.D, (i * LPR + lane) * V, g.D,
                              r[i], rest[i], k);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            row_store<T, V>(static_cast<T*>(g.y) + row * g.D, (i * LPR + lane) * V, g.D, r[i]);
    }
}

template <typename T, int LPR, int N>
__global__ void __launch_bounds__(norm_block<LPR>()) norm_backward_kernel(NormArgs g) {
    constexpr int V = 16 / sizeof(T);
    constexpr int RPB = norm_block<LPR>() / LPR;
    __shared__ float slots[2][16];
    const int lane = threadIdx.x % LPR;
    float dw[N][V], w[N][V];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int at = (i * LPR + lane) * V;
        if (g.weight_f32) {
            row_load<float, V>(static_cast<const float*>(g.weight), at, g.D, w[i]);
        } else {
            row_load<T, V>(static_cast<const T*>(g.weight), at, g.D, w[i]);
        }
#pragma unroll
        for (int v = 0; v < V; ++v) dw[i][v] = 0.f;
    }
    int turn = 0;   // two LDS slots in turn: a wavefront that is a row ahead writes the other one
    for (long first = (long)blockIdx.x * RPB; first < g.rows; first += (long)gridDim.x * RPB, turn ^= 1) {
        const long row = first + threadIdx.x / LPR;
        if (LPR <= 64 && row >= g.rows) continue;
        const T* x = static_cast<const T*>(g.x) + row * g.x_row;
        const T* dy = static_cast<const T*>(g.dy) + row * g.dy_row;
        const float s = g.rstd[row];
        float r[N][V], d[N][V];
        float along = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int at = (i * LPR + lane) * V;
            row_load<T, V>(x, at, g.D, r[i]);
            row_load<T, V>(dy, at, g.D, d[i]);
            if (g.residual) {
                float b[V];
                row_load<T, V>(static_cast<const T*>(g.residual) + row * g.residual_row, at, g.D, b);
#pragma unroll
                for (int v = 0; v < V; ++v) r[i][v] += b[v];
            }
        }
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int v = 0; v < V; ++v) {
                r[i][v] *= s;                          // n
                dw[i][v] += d[i][v] * r[i][v];
                d[i][v] *= w[i][v];
                along += d[i][v] * r[i][v];
            }
        along = over_row<Add, LPR>(along, slots[turn]) / (float)g.D;
        const T* gr = static_cast<const T*>(g.dsum);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int at = (i * LPR + lane) * V;
            float out[V];
            if (gr) {
                row_load<T, V>(gr + row * g.dsum_row, at, g.D, out);
            } else {
#pragma unroll
                for (int v = 0; v < V; ++v) out[v] = 0.f;
            }
#pragma unroll
            for (int v = 0; v < V; ++v) out[v] += s * (d[i][v] - r[i][v] * along);
            row_store<T, V>(static_cast<T*>(g.dx) + row * g.D, at, g.D, out);
        }
    }
    // a wavefront's rows of lanes are added by exchanges, then the wavefronts in LDS, always in the same order
    if constexpr (RPB > 1) {
        __shared__ float total[4][LPR * N * V];
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int v = 0; v < V; ++v) {
                float t = dw[i][v];
#pragma unroll
                for (int apart = LPR; apart < 64; apart *= 2) t += __shfl_xor(t, apart);
                if ((threadIdx.x & 63) < LPR) total[threadIdx.x >> 6][(i * LPR + lane) * V + v] = t;
            }
        __syncthreads();
        for (int at = threadIdx.x; at < g.D; at += norm_block<LPR>())
            g.partial[(long)blockIdx.x * g.D + at] = total[0][at] + total[1][at] + total[2][at] + total[3][at];
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            row_store<float, V>(g.partial + (long)blockIdx.x * g.D, (i * LPR + lane) * V, g.D, dw[i]);
    }
}

// dw (D) from the workgroups' partial rows, rounded to the weight's type.  64 columns per
// workgroup; its 16 wavefronts take every 16th row and are added in order.
template <typename T>
__global__ void __launch_bounds__(1024) norm_weight_grad_kernel(long parts, int D,
                                                                const float* __restrict__ partial,
                                                                T* __restrict__ dw) {
    __shared__ float sums[16][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int at = blockIdx.x * 64 + lane;
    float s = 0.f;
    if (at < D) {
#pragma unroll 16
        for (long i = wave; i < parts; i += 16) s += partial[i * D + at];
    }
    sums[wave][lane] = s;
    __syncthreads();
    if (wave == 0 && at < D) {
#pragma unroll
        for (int i = 1; i < 16; ++i) s += sums[i][lane];
        dw[at] = narrow<T>(s);
    }
}

// Lanes per row and vectors per lane: the fewest lanes that hold the row in one or two vectors each (beyond
// 1024 lanes more), so that a narrow row does not leave lanes idle and the backward kernel's four rows of
// floats leave room for four to six wavefronts to a SIMD.  (Up to four vectors of eight 16-bit elements took
// 221 registers; backward, bfloat16: 16384 x 2048 101 us against 71, 4096 x 8192 102 against 68, 65536 x 512
// 105 against 69; forward 45 to 51 against 43 to 45.  2500000 x 16 with 16 lanes to a row 249 us forward and
// 425 backward, with four 79 and 132.)
template <typename T, typename F>
static int with_shape(int D, F&& f) {
    constexpr int V = 16 / sizeof(T);
    const int vecs = (D + V - 1) / V;
    const auto call = [&](auto lpr, auto n) { return f(lpr, n); };
#define KVAE_NORM_SHAPE(LPR, N)                                                                   \
    if (vecs <= LPR * N)                                                                          \
        return call(std::integral_constant<int, LPR>{}, std::integral_constant<int, N>{});
    KVAE_NORM_SHAPE(4, 1)
    KVAE_NORM_SHAPE(8, 1)
    KVAE_NORM_SHAPE(16, 1)
    KVAE_NORM_SHAPE(16, 2)
    KVAE_NORM_SHAPE(64, 1)
    KVAE_NORM_SHAPE(64, 2)
    KVAE_NORM_SHAPE(256, 1)
    KVAE_NORM_SHAPE(512, 1)
    KVAE_NORM_SHAPE(1024, 1)
    KVAE_NORM_SHAPE(1024, 2)
    if constexpr (sizeof(T) == 4) { KVAE_NORM_SHAPE(1024, 4) }   // 16-bit rows end at 1024 x 2
#undef KVAE_NORM_SHAPE
    return KVAE_E_UNSUPPORTED;
}

static int check_norm(const kvae_rms_norm* d) {
    if (!d || d->rows < 1 || d->D < 1 || !d->x || !d->weight) return KVAE_E_BADARG;
    if (d->D > KVAE_NORM_MAX_WIDTH) return KVAE_E_UNSUPPORTED;
    if (d->dtype != KVAE_F32 && d->dtype != KVAE_BF16 && d->dtype != KVAE_F16)
        return KVAE_E_UNSUPPORTED;
    if (d->weight_dtype != KVAE_F32 && d->weight_dtype != d->dtype) return KVAE_E_UNSUPPORTED;
    if (d->rows > 0x7fffffffL) return KVAE_E_TOOLARGE;
    return KVAE_OK;
}

static NormArgs norm_args(const kvae_rms_norm* d) {
    NormArgs g{};
    g.rows = d->rows, g.D = (int)d->D;
    g.x = d->x, g.x_row = d->x_stride;
    g.residual = d->residual, g.residual_row = d->residual_stride;
    g.weight = d->weight, g.weight_f32 = d->weight_dtype == KVAE_F32;
    g.eps = d->eps;
    g.y = d->y;
    g.scale = static_cast<float*>(d->scale);
    g.sum = d->sum, g.rstd = static_cast<float*>(d->rstd);
    g.dy = d->dy, g.dsum = d->dsum, g.dy_row = d->dy_stride, g.dsum_row = d->dsum_stride;
    g.dx = d->dx, g.partial = static_cast<float*>(d->partial);
    return g;
}

template <bool QUANT, bool NORM>
static int run_forward(int dtype, const NormArgs& all, hipStream_t stream) {
    return for_element_type(dtype, [&](auto e) {
        using T = decltype(e);
        return with_shape<T>(all.D, [&](auto lpr, auto n) {
            constexpr int LPR = decltype(lpr)::value, N = decltype(n)::value;
            constexpr int BLOCK = norm_block<LPR>(), RPB = BLOCK / LPR;
            // (a launch has fewer than 2^32 threads: rows beyond go in further launches)
            constexpr long MOST = (1L << 31) / LPR;
            for (long first = 0; first < all.rows; first += MOST) {
                NormArgs g = all;
                g.rows = all.rows - first < MOST ? all.rows - first : MOST;
                g.x = static_cast<const T*>(all.x) + first * all.x_row;
                if (all.residual) g.residual = static_cast<const T*>(all.residual) + first * all.residual_row;
                g.y = static_cast<char*>(all.y) + first * all.D * (QUANT ? 1 : (long)sizeof(T));
                if (all.scale) g.scale = all.scale + first;
                if (all.sum) g.sum = static_cast<T*>(all.sum) + first * all.D;
                if (all.rstd) g.rstd = all.rstd + first;
                norm_forward_kernel<T, LPR, N, QUANT, NORM>
                    <<<dim3((unsigned)((g.rows + RPB - 1) / RPB)), BLOCK, 0, stream>>>(g);
            }
            return hipGetLastError() == hipSuccess ? KVAE_OK : KVAE_E_LAUNCH;
        });
    });
}

// Workgroups of the backward kernel = partial rows of dw, at most (the buffer's): four per compute unit fill
// the card, fewer when there are not four rows for each.
static long norm_parts(long rows) {
    const long most = 4L * device_compute_units();
    const long want = (rows + 3) / 4;
    return want < most ? want : most;
}

}  // namespace kvae

using namespace kvae;

extern "C" int64_t kvae_rms_norm_backward_parts(int64_t rows) { return rows < 1 ? 0 : norm_parts(rows); }

extern "C" int kvae_rms_norm_forward(const kvae_rms_norm* d, void* stream) {
    const int rc = check_norm(d);
    if (rc != KVAE_OK) return rc;
    if (!d->y) return KVAE_E_BADARG;
    return run_forward<false, true>(d->dtype, norm_args(d), static_cast<hipStream_t>(stream));
}

extern "C" int kvae_rms_norm_quantized(const kvae_rms_norm* d, void* stream) {
    const int rc = check_norm(d);
    if (rc != KVAE_OK) return rc;
    if (!d->y || !d->scale) return KVAE_E_BADARG;
    return run_forward<true, true>(d->dtype, norm_args(d), static_cast<hipStream_t>(stream));
}

extern "C" int kvae_quantize_rows(int64_t rows, int64_t D, int dtype, const void* x, int64_t x_stride,
                                  void* q, void* scale, void* stream) {
    if (rows < 1 || D < 1 || !x || !q || !scale) return KVAE_E_BADARG;
    if (D > KVAE_NORM_MAX_WIDTH) return KVAE_E_UNSUPPORTED;
    if (rows > 0x7fffffffL) return KVAE_E_TOOLARGE;
    NormArgs g{};
    g.rows = rows, g.D = (int)D, g.x = x, g.x_row = x_stride, g.y = q;
    g.scale = static_cast<float*>(scale);
    return run_forward<true, false>(dtype, g, static_cast<hipStream_t>(stream));
}

extern "C" int kvae_rms_norm_backward(const kvae_rms_norm* d, void* stream) {
    const int rc = check_norm(d);
    if (rc != KVAE_OK) return rc;
    if (!d->dy || !d->dx || !d->partial || !d->dweight || !d->rstd) return KVAE_E_BADARG;
    const NormArgs g = norm_args(d);
    const hipStream_t s = static_cast<hipStream_t>(stream);
    return for_element_type(d->dtype, [&](auto e) {
        using T = decltype(e);
        return with_shape<T>(g.D, [&](auto lpr, auto n) {
            constexpr int LPR = decltype(lpr)::value, N = decltype(n)::value;
            // as many as there are rows for, and as fit on the card at once (wide rows take 512 and 1024 threads:
            // 8192 x 3000 bfloat16 48 us with three of 512 to a unit, 64 with four)
            constexpr int RPB = norm_block<LPR>() / LPR, FIT = LPR <= 256 ? 4 : LPR <= 512 ? 3 : 2;
            long parts = norm_parts(g.rows);
            if (parts > (g.rows + RPB - 1) / RPB) parts = (g.rows + RPB - 1) / RPB;
            if (parts > (long)FIT * device_compute_units()) parts = (long)FIT * device_compute_units();
            norm_backward_kernel<T, LPR, N><<<dim3((unsigned)parts), norm_block<LPR>(), 0, s>>>(g);
            const dim3 grid((unsigned)((g.D + 63) / 64));
            if (g.weight_f32) {
                norm_weight_grad_kernel<float>
                    <<<grid, 1024, 0, s>>>(parts, g.D, g.partial, static_cast<float*>(d->dweight));
            } else {
                norm_weight_grad_kernel<T>
                    <<<grid, 1024, 0, s>>>(parts, g.D, g.partial, static_cast<T*>(d->dweight));
            }
            return hipGetLastError() == hipSuccess ? KVAE_OK : KVAE_E_LAUNCH;
        });
    });
}
