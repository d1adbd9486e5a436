// Product of 8-bit rows on gfx950: y[m][n] = sx[m] sw[n] sum_k x[m][k] w[n][k] + bias[n], x and w in
// e4m3 with one float scale per row (what rms_norm_quantized and quantize_rows write), summed in
// float on the matrix instructions.
//
// 16-bit results of more than 32 rows take the instructions for 8-bit operands.  These add eight neighbouring
// products aligned to the largest of them and drop what lies 2^-14 or more below it (seen by feeding them one
// large and one small product, at every distance): each of the other seven loses less than 2^-13 of the largest.
// That is 1.6e-5 of a sum of Gaussian terms, a hundredth of a bfloat16 result's rounding and a fifteenth of a
// half's, but more than float sums lose, and all of a small result where large products cancel.  Otherwise the
// bytes are widened to half, which holds every e4m3 value, and multiplied by the instructions for half operands,
// at half the rate, whose sums are float throughout (1e-8 on the same terms): for float results, which would show
// the difference, and for up to 32 rows, where reading w is most of the work (bfloat16, 8-bit operands against
// widened ones, weights not used just before: 1 x 6144 x 2048 4.84 us both, 32 x 4096 x 4096 6.82 both, 64 rows 7.9
// against 8.8; the same weights call after call: 3.85 against 4.3 and 6.0 against 6.2; 16384 x 4096 x 4096 220
// against 475).
//
// Both operands lie along k, so a lane's 32 operand bytes are contiguous in memory.  w takes the
// first operand's place: then a lane's results are four neighbouring n of one row m, which go out
// as one wide store, and the matrix instruction's k order does not matter as both sides share it.
//
// Three forms.  Few rows: reading w once is the work; a workgroup takes 16 rows of w (64 when there are enough
// of them) and up to 64 of x, its wavefronts share out k and add up through LDS.  Tiles of 128 x 128 staged
// through registers and LDS, the next slice of k on its way while the present one is multiplied, three
// workgroups to a unit.  Large tiles of 256 x 256, fed from memory straight into LDS, for large products.
//
// Measured (bfloat16 results, kernel times).  The same operands call after call: 1 x 6144 x 2048 4.3 us (2.9 TB/s),
// 64 x 4096 x 4096 7 to 8.4 us, 256 x 4096 x 4096 12 us, 1024^3 6.5 us, 262144 x 384 x 128 48 us (4.9 TB/s, memory's
// rate), 4096^3 58 us, 16384 x 4096 x 4096 222 us = 2.5 PFLOP/s, 8192^3 432 us = 2.5.  Operands that were not used just
// before: 1 x 6144 x 2048 4.8 us, 262144 x 384 x 128 54, 16384 x 4096 x 4096 240 to 265, where the library's
// product of 8-bit operands takes 224 us.  A loop of nothing but these instructions reaches 3.4 to 4 PFLOP/s on random
// bytes (the clock comes down).  k = 4097 goes to tiles of 128: 450 us (495).  Float results: 16384 x 4096 x 4096
// 475 us (on new rows 565, where the library's product of half operands takes 510 to 550), 262144 x 384 x 128 89 us,
// 262144 x 128 x 128 29.
// Each round of large tiles spends some 12 us outside its loop (first requests, results); workgroups that stay and
// ask for the next tile's start before they write the last one's results were no faster (227 to 248 us).
#include "narrow_types.h"

#include "device_info.h"

namespace kvae {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v8i __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v16f __attribute__((ext_vector_type(16)));

struct LinearArgs {
    long M;
    int N, K;
    const uint8_t* x;
    const uint8_t* w;
    const float* sx;
    const float* sw;
    const float* bias;
    void* y;
};

struct __attribute__((packed)) AnyPiece { v4i v; };

// r without its first `bytes` (0 .. 16 and more), zero behind what is left
__device__ __forceinline__ v4i shift_down(const v4i& r, int bytes) {
    unsigned long lo = (unsigned)r.x | (unsigned long)(unsigned)r.y << 32;
    unsigned long hi = (unsigned)r.z | (unsigned long)(unsigned)r.w << 32;
    const int n = 8 * (bytes & 7);
    if (bytes >= 8) lo = hi, hi = 0;
    if (n) lo = lo >> n | hi << (64 - n), hi >>= n;
    if (bytes >= 16) lo = 0;
    return v4i{(int)lo, (int)(lo >> 32), (int)hi, (int)(hi >> 32)};
}

// 16 bytes of a row of K < 16 from byte k on; bytes at K and beyond are zero
__device__ __forceinline__ v4i first_bytes(const uint8_t* row, int k, int K) {
    unsigned long lo = 0, hi = 0;
#pragma unroll 1
    for (int i = 0; k + i < K; ++i) (i < 8 ? lo : hi) |= (unsigned long)row[k + i] << (8 * (i & 7));
    return v4i{(int)lo, (int)(lo >> 32), (int)hi, (int)(hi >> 32)};
}

typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));

// bytes 8 i .. 8 i + 7 of a lane's 32 as halves (exact)
__device__ __forceinline__ v8h widen8(const v8i& a, int i) {
    const v2h p = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a[2 * i], 1.f, false);
    const v2h q = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a[2 * i], 1.f, true);
    const v2h r = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a[2 * i + 1], 1.f, false);
    const v2h t = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a[2 * i + 1], 1.f, true);
    return v8h{p.x, p.y, q.x, q.y, r.x, r.y, t.x, t.y};
}

// whether results of this type, from blocks of 16 MT rows of x, take the products of widened operands
template <typename T, int MT = 4>
constexpr bool WIDENED = sizeof(T) == 4 || MT <= 2;

// four neighbouring results of one row
template <typename T>
__device__ __forceinline__ void store4(const LinearArgs& g, long m, int n, const float (&acc)[4]) {
    if (m >= g.M || n >= g.N) return;
    const float sx = g.sx[m];
    T* out = static_cast<T*>(g.y) + m * g.N + n;
    if (n + 4 <= g.N) {
        const Pack<float, 4> sw = load_pack<float, 4>(g.sw + n);
        Pack<float, 4> b{};
        if (g.bias) b = load_pack<float, 4>(g.bias + n);
        Pack<T, 4> p;
#pragma unroll
        for (int i = 0; i < 4; ++i) p.v[i] = narrow<T>(acc[i] * sx * sw.v[i] + b.v[i]);
        store_pack<T, 4>(out, p);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (n + i < g.N) out[i] = narrow<T>(acc[i] * sx * g.sw[n + i] + (g.bias ? g.bias[n + i] : 0.f));
    }
}

// A tile's scales and biases in LDS, asked for at the start and there when the results go out.
template <int ROWS>
struct Factors {
    float sx[ROWS], sw[ROWS], bias[ROWS];
};
template <int ROWS>
__device__ __forceinline__ void load_factors(const LinearArgs& g, long m0, int n0, Factors<ROWS>& f) {
    const int i = threadIdx.x;
    if (i < ROWS) {                                  // (those of rows that are not there are not used)
        const long m = m0 + i < g.M ? m0 + i : g.M - 1;
        const int n = n0 + i < g.N ? n0 + i : g.N - 1;
        const float sx = g.sx[m], sw = g.sw[n], bias = g.bias ? g.bias[n] : 0.f;
        f.sx[i] = sx, f.sw[i] = sw, f.bias[i] = bias;
    }
}

// Results of 32 JN rows by WN columns that a wavefront holds as JN x WN / 32 sums of a 32 x 32 instruction:
// a lane has row 32 j + lane % 32, columns 32 i + 8 q + 4 (lane / 32) .. + 3.  Written from there, an
// instruction would touch 32 rows with 16 bytes each; they go through LDS (`region`: the wavefront's own)
// and out in runs of a whole row of WN.  rm, rn: first row and column inside the tile that starts at
// (m0, n0); value(i, j, e): element e of sum (i, j).
template <typename T, int WN, int JN, int ROWS, typename F>
__device__ __forceinline__ void write_rows(const LinearArgs& g, const Factors<ROWS>& f, char* region, long m0, int n0,
                                           int rm, int rn, int lane, F&& value) {
    constexpr int ROW = WN * (int)sizeof(T), CHUNKS = ROW / 16, PER = 16 / (int)sizeof(T);
    const int row = lane & 31, half = lane >> 5;
    float sx[JN];
#pragma unroll
    for (int j = 0; j < JN; ++j) sx[j] = f.sx[rm + 32 * j + row];
#pragma unroll
    for (int i = 0; i < WN / 32; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int in = 32 * i + 8 * q + 4 * half;
            const v4f sw = *reinterpret_cast<const v4f*>(f.sw + rn + in);
            const v4f b = *reinterpret_cast<const v4f*>(f.bias + rn + in);
            // (the exclusive-or spreads the rows over the banks)
            const int chunk = in / PER ^ (row & (CHUNKS - 1));
            char* at = region + row * ROW + chunk * 16 + in % PER * (int)sizeof(T);
#pragma unroll
            for (int j = 0; j < JN; ++j) {
                Pack<T, 4> p;
#pragma unroll
                for (int e = 0; e < 4; ++e) p.v[e] = narrow<T>(value(i, j, 4 * q + e) * sx[j] * sw[e] + b[e]);
                *reinterpret_cast<Pack<T, 4>*>(at + 32 * j * ROW) = p;
            }
        }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    constexpr int STEP = 64 / CHUNKS;                // rows of one instruction
    const int r0 = lane / CHUNKS, c = lane % CHUNKS;
    const long m = m0 + rm;
    const int n = n0 + rn + c * PER;
    T* out = static_cast<T*>(g.y) + (m + r0) * g.N + n;
    const auto piece = [&](int k) {
        const int r = k * STEP + r0;
        return *reinterpret_cast<const Pack<T, PER>*>(region + r * ROW + (c ^ (r & (CHUNKS - 1))) * 16);
    };
    if (m + 32 * JN <= g.M && n0 + rn + WN <= g.N) {
#pragma unroll
        for (int k = 0; k < 32 * JN / STEP; ++k) store_pack<T, PER>(out + (long)k * STEP * g.N, piece(k));
    } else {
#pragma unroll 1
        for (int k = 0; k < 32 * JN / STEP; ++k) {
            const Pack<T, PER> p = piece(k);
            T* at = out + (long)k * STEP * g.N;
            if (m + k * STEP + r0 >= g.M) continue;
            if (n + PER <= g.N) {
                store_pack<T, PER>(at, p);
            } else {
#pragma unroll
                for (int e = 0; e < PER; ++e)
                    if (n + e < g.N) at[e] = p.v[e];
            }
        }
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

constexpr int TILE = 128, SLICE = 128;
// LDS place of 16-byte piece c of row r.  A wavefront reads piece c of 32 rows with its lower lanes and
// piece c + 1 with its upper lanes (which pieces a lane holds is free, as both operands share it); with
// this exclusive-or such a read meets no bank twice.  (With r % 8, and pieces c and c + 2, a read took
// 12 cycles of the LDS for 8: 16384 x 4096 x 1024 91 us against 82.)
__device__ __forceinline__ int row_key(int r) { return (r >> 1) & 7; }
__device__ __forceinline__ int piece_at(int r, int c) { return r * (SLICE / 16) + (c ^ row_key(r)); }

constexpr int FEW_WAVES = 8;
// Rows of x: blockIdx.y * 16 MT ..., rows of w: blockIdx.x * 16 NT ...  The wavefronts share out k in slices of
// 128 bytes.  The matrix instruction wants 16 rows side by side in 16 neighbouring lanes; loaded like that,
// every lane would be in another cache line (57 cycles of the address unit for an instruction of 1 KB).
// So eight lanes load a line, and the rows change lanes in LDS of the wavefront's own.
template <typename T, int MT, int NT>
__global__ void __launch_bounds__(64 * FEW_WAVES) linear_few_rows_kernel(LinearArgs g) {
    constexpr int ROWS16 = 16 * SLICE / 16;          // pieces of 16 rows
    __shared__ v4i lds[FEW_WAVES][(MT + NT) * ROWS16];
    static_assert(sizeof(lds) >= FEW_WAVES * MT * NT * 64 * sizeof(v4f), "holds the sums afterwards");
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const long m0 = (long)blockIdx.y * 16 * MT;
    const int n0 = blockIdx.x * 16 * NT;
    v4i* own = lds[wave];
    // a lane loads piece lane % 8 of rows lane / 8 and lane / 8 + 8 of NT blocks of w and of MT blocks of x
    // (rows that are not there repeat the last one: their results are not stored)
    const int piece = lane & 7;
    const uint8_t *xb = g.x + m0 * g.K, *wb = g.w + (long)n0 * g.K;
    const unsigned row0 = (unsigned)(lane >> 3) * (unsigned)g.K;     // byte offsets from the first rows
    const unsigned x_end = (unsigned)(g.M - m0 < 16 * MT ? g.M - m0 - 1 : 16 * MT - 1) * (unsigned)g.K;
    const unsigned w_end = (unsigned)(g.N - n0 < 16 * NT ? g.N - n0 - 1 : 16 * NT - 1) * (unsigned)g.K;
    const auto from = [&](int t, int i) {
        const unsigned row = row0 + (unsigned)(16 * (t < NT ? t : t - NT) + 8 * i) * (unsigned)g.K;
        return t < NT ? wb + (row < w_end ? row : w_end) : xb + (row < x_end ? row : x_end);
    };
    v4f acc[MT][NT];
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int u = 0; u < NT; ++u) acc[t][u] = v4f{0.f, 0.f, 0.f, 0.f};
    v4i in[NT + MT][2];
    const auto load = [&](int k0) {
        if (k0 + SLICE <= g.K) {
#pragma unroll
            for (int t = 0; t < NT + MT; ++t)
#pragma unroll
                for (int i = 0; i < 2; ++i) in[t][i] = reinterpret_cast<const AnyPiece*>(from(t, i) + (k0 + 16 * piece))->v;
        } else if (NT > 1 || g.K >= 16) {            // (NT > 1 is for K >= 16)
            // pieces that end behind the row are its last 16 bytes shifted down
            const int k = k0 + 16 * piece, at = k < g.K - 16 ? k : g.K - 16;
#pragma unroll
            for (int t = 0; t < NT + MT; ++t)
#pragma unroll
                for (int i = 0; i < 2; ++i) in[t][i] = reinterpret_cast<const AnyPiece*>(from(t, i) + at)->v;
            if (k > at) {
#pragma unroll
                for (int t = 0; t < NT + MT; ++t)
#pragma unroll
                    for (int i = 0; i < 2; ++i) in[t][i] = shift_down(in[t][i], k - at);
            }
        } else {
#pragma unroll
            for (int t = 0; t < NT + MT; ++t)
#pragma unroll
                for (int i = 0; i < 2; ++i) in[t][i] = first_bytes(from(t, i), k0 + 16 * piece, g.K);
        }
    };
    const auto between = [] {                        // the wavefront's accesses to LDS stay on their sides
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    };
    const auto operand = [&](int t) {
        const v4i p = own[t * ROWS16 + piece_at(lane & 15, lane >> 4)], q = own[t * ROWS16 + piece_at(lane & 15, (lane >> 4) + 4)];
        return v8i{p.x, p.y, p.z, p.w, q.x, q.y, q.z, q.w};
    };
    int k0 = wave * SLICE;
    if (k0 < g.K) load(k0);
    for (; k0 < g.K; k0 += FEW_WAVES * SLICE) {
#pragma unroll
        for (int t = 0; t < NT + MT; ++t)
#pragma unroll
            for (int i = 0; i < 2; ++i) own[t * ROWS16 + piece_at(8 * i + (lane >> 3), piece)] = in[t][i];
        between();
        if (k0 + FEW_WAVES * SLICE < g.K) load(k0 + FEW_WAVES * SLICE);
        v8i a[NT];
#pragma unroll
        for (int u = 0; u < NT; ++u) a[u] = operand(u);
        if constexpr (WIDENED<T, MT>) {
            // (quarter by quarter, so that the widened operands of one only are in registers)
            v8i b[MT];
#pragma unroll
            for (int t = 0; t < MT; ++t) b[t] = operand(NT + t);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v8h ah[NT];
#pragma unroll
                for (int u = 0; u < NT; ++u) ah[u] = widen8(a[u], i);
#pragma unroll
                for (int t = 0; t < MT; ++t) {
                    const v8h bh = widen8(b[t], i);
#pragma unroll
                    for (int u = 0; u < NT; ++u)
                        acc[t][u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ah[u], bh, acc[t][u], 0, 0, 0);
                }
            }
        } else {
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                const v8i b = operand(NT + t);
#pragma unroll
                for (int u = 0; u < NT; ++u)
                    acc[t][u] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a[u], b, acc[t][u], 0, 0, 0, 0, 0, 0);
            }
        }
        between();
    }
    __syncthreads();
    v4f(*sums)[MT * NT][64] = reinterpret_cast<v4f(*)[MT * NT][64]>(lds);
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int u = 0; u < NT; ++u) sums[wave][t * NT + u][lane] = acc[t][u];
    __syncthreads();
    for (int t = wave; t < MT * NT; t += FEW_WAVES) {
        v4f total = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int v = 0; v < FEW_WAVES; ++v) total += sums[v][t][lane];
        const float four[4] = {total.x, total.y, total.z, total.w};
        store4<T>(g, m0 + 16 * (t / NT) + (lane & 15), n0 + 16 * (t % NT) + 4 * (lane >> 4), four);
    }
}

template <typename T>
__global__ void __launch_bounds__(256, 3) linear_tile_kernel(LinearArgs g) {
    __shared__ v4i shared[2 * TILE * SLICE / 16];
    __shared__ Factors<TILE> factors;
    v4i *xs = shared, *ws = shared + TILE * SLICE / 16;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const long m0 = (long)blockIdx.y * TILE;
    const int n0 = blockIdx.x * TILE;
    const int wm = (wave >> 1) * 64, wn = (wave & 1) * 64;
    v16f acc[2][2];
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[a][b][i] = 0.f;
    // A thread's pieces: column tid % 8 of rows tid / 8 + 32 i, as 32-bit offsets from the tile's first
    // rows; rows that are not there repeat the last (their results are not stored).
    const uint8_t* xb = g.x + m0 * g.K;
    const uint8_t* wb = g.w + (long)n0 * g.K;
    const int col = (threadIdx.x & 7) * 16;
    unsigned x_row[4], w_row[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = (threadIdx.x >> 3) + 32 * i;
        x_row[i] = (unsigned)(r < g.M - m0 ? r : (int)(g.M - m0) - 1) * (unsigned)g.K;
        w_row[i] = (unsigned)(r < g.N - n0 ? r : g.N - n0 - 1) * (unsigned)g.K;
    }
    const auto multiply = [&] {
#pragma unroll
        for (int s = 0; s < SLICE / 64; ++s) {
            v8i a[2], b[2];
            const int c = s * 4 + (lane >> 5);
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const int ra = wn + 32 * t + (lane & 31), rb = wm + 32 * t + (lane & 31);
                const v4i p = ws[piece_at(ra, c)], q = ws[piece_at(ra, c + 2)];
                a[t] = v8i{p.x, p.y, p.z, p.w, q.x, q.y, q.z, q.w};
                const v4i u = xs[piece_at(rb, c)], v = xs[piece_at(rb, c + 2)];
                b[t] = v8i{u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
            }
            if constexpr (WIDENED<T>) {
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const v8h bh[2] = {widen8(b[0], q), widen8(b[1], q)};
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const v8h ah = widen8(a[i], q);
#pragma unroll
                        for (int j = 0; j < 2; ++j)
                            acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ah, bh[j], acc[i][j], 0, 0, 0);
                    }
                }
            } else {
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int j = 0; j < 2; ++j)
                        acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a[i], b[j], acc[i][j],
                                                                                    0, 0, 0, 0, 0, 0);
            }
        }
    };
    // The next slice is on its way in registers while the present one is multiplied.  Pieces that end
    // behind the row are its last 16 bytes (K >= 16 here), shifted down before they go to LDS, so that
    // there is zero behind the end of k in both operands.
    const int slices = (g.K + SLICE - 1) / SLICE;
    v4i xr[4], wr[4];
    const auto fetch = [&](int s) {
        const int k = s * SLICE + col;
        const unsigned at = (unsigned)(k < g.K - 16 ? k : g.K - 16);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            xr[i] = reinterpret_cast<const AnyPiece*>(xb + (x_row[i] + at))->v;
            wr[i] = reinterpret_cast<const AnyPiece*>(wb + (w_row[i] + at))->v;
        }
    };
    fetch(0);
    load_factors(g, m0, n0, factors);                // (read behind the loop's barriers)
    for (int s = 0; s < slices; ++s) {
        if ((s + 1) * SLICE > g.K) {
            const int behind = s * SLICE + col + 16 - g.K;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                xr[i] = behind > 0 ? shift_down(xr[i], behind) : xr[i];
                wr[i] = behind > 0 ? shift_down(wr[i], behind) : wr[i];
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int place = piece_at(threadIdx.x >> 3, threadIdx.x & 7) + 32 * i * (SLICE / 16);
            xs[place] = xr[i];
            ws[place] = wr[i];
        }
        __syncthreads();
        if (s + 1 < slices) fetch(s + 1);
        multiply();
        __syncthreads();
    }
    char* region = reinterpret_cast<char*>(shared) + wave * (32 * 64 * (int)sizeof(T));
#pragma unroll
    for (int j = 0; j < 2; ++j)
        write_rows<T, 64, 1>(g, factors, region, m0, n0, wm + 32 * j, wn, lane,
                             [&](int i, int, int e) { return acc[i][j][e]; });
}

// Large products: 256 x 256 tiles, four wavefronts of 128 x 128 each (their sums fill the accumulation
// registers, one wavefront per SIMD).  A 64-byte slice of k is sixteen 32x32x64 matrix instructions
// (1024 cycles) per wavefront on eight operands of 2 KB, so that the four wavefronts ask LDS for 64 bytes
// a cycle, half of what 64 x 64 wavefront tiles would.
//
// Double slices (128 bytes of each row: whole cache lines) go from memory straight into LDS, no registers
// in between, into two buffers in turn, and are multiplied half by half: while a half is multiplied, the
// operands of the next half are read into registers of their own.  When the second half of one double
// slice has been read by everybody, the double slice after next is asked for into its place: it has two
// steps (2048 cycles) to arrive.  One barrier per double slice, before its first half is read: a wavefront
// waits there until its own pieces have arrived, and behind the barrier everybody's have.  Double slices go
// in pairs, one for each buffer; behind an odd number of them comes one of zeros.  Two steps hide the way from
// the die's cache but not the one from memory, so a step also touches the lines of the double slice after
// that, shared out among the tiles of a die (inputs that were not used just before: 250 -> 230 us).
//
// Rows that are not there repeat the last one (their results are not stored).  Where k ends inside the
// last slice, pieces behind the end repeat the row's last piece and are replaced by zero on their way
// from LDS to the registers, in both operands (a NaN in one of them must not meet the other's zero).
constexpr int BIG = 256, BIG_SLICE = 128;
constexpr int OPERAND = BIG * BIG_SLICE / 16;        // pieces of one operand's double slice

template <typename T>
__global__ void __launch_bounds__(256, 1) linear_big_kernel(LinearArgs g, int tiles_n, int tiles_m) {
    static_assert(sizeof(T) == 2, "four wavefronts' results fill the LDS");
    // Two buffers of [x, w][row][8 pieces], 64 KB each.  They are two variables, and which one is meant is
    // known where the code is compiled: the compiler lets a read of LDS wait for every request into the same
    // variable that is under way (with one variable for both each half step waited for what it had just
    // asked for: 16384 x 4096 x 4096 264 us).
    __shared__ v4i buffer0[2 * OPERAND], buffer1[2 * OPERAND];
    __shared__ Factors<BIG> factors;
    __shared__ unsigned unread[64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // Workgroups go round the eight dies (blockIdx % 8): each die gets a run of neighbouring tiles, in
    // groups of eight rows of tiles, so that its cache serves the tiles that run together.
    const int total = tiles_n * tiles_m, per = (total + 7) / 8;
    const int id = (int)(blockIdx.x & 7) * per + (int)(blockIdx.x >> 3);
    if ((int)(blockIdx.x >> 3) >= per || id >= total) return;
    const int in_group = 8 * tiles_n, group = id / in_group, rest = id - group * in_group;
    const int rows = tiles_m - 8 * group < 8 ? tiles_m - 8 * group : 8;
    const long m0 = (long)(8 * group + rest % rows) * BIG;
    const int n0 = rest / rows * BIG;
    const int wm = (wave >> 1) * 128, wn = (wave & 1) * 128;

    // Pieces lie as in the small tiles.  An instruction moves 8 rows: lane l fills place l % 8 of row l / 8.
    const int piece = (lane & 7) ^ row_key(8 * wave + (lane >> 3)), last_piece = g.K / 16 - 1;
    const uint8_t* xb = g.x + m0 * g.K;
    const uint8_t* wb = g.w + (long)n0 * g.K;
    const long rows_x = g.M - m0, rows_w = g.N - n0;
    unsigned x_row[8], w_row[8];                     // byte offsets of the lane's rows
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const long r = 8 * (wave + 4 * i) + (lane >> 3);
        x_row[i] = (unsigned)(r < rows_x ? r : rows_x - 1) * (unsigned)g.K;
        w_row[i] = (unsigned)(r < rows_w ? r : rows_w - 1) * (unsigned)g.K;
    }
    // `b`: std::integral_constant of the buffer
    const auto fetch = [&](auto b, int d) {          // double slice d
        const int p = 8 * d + piece;
        const unsigned k = 16u * (unsigned)(p < last_piece ? p : last_piece);
        v4i* at = (decltype(b)::value ? buffer1 : buffer0) + wave * 64;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            __builtin_amdgcn_global_load_lds(
                (const __attribute__((address_space(1))) void*)(xb + (x_row[i] + k)),
                (__attribute__((address_space(3))) void*)(at + 256 * i), 16, 0, 0);
            __builtin_amdgcn_global_load_lds(
                (const __attribute__((address_space(1))) void*)(wb + (w_row[i] + k)),
                (__attribute__((address_space(3))) void*)(at + OPERAND + 256 * i), 16, 0, 0);
        }
    };
    // One word of a cache line of double slice d, so that it is in the die's cache when the slice is asked for.
    // The tiles that run together on a die lie four in a row and eight in a column, so each touches a quarter
    // of its rows of x and an eighth of its rows of w, and the others theirs of the same rows.
    const int xr = 64 * (rest / rows & 3) + 16 * wave + (lane & 15), wr = 32 * (rest % rows & 7) + 8 * wave + (lane & 7);
    const uint8_t* line = lane < 16 ? xb + (xr < rows_x ? xr : rows_x - 1) * g.K : wb + (wr < rows_w ? wr : rows_w - 1) * g.K;
    const auto warm = [&](int d) {
        __builtin_amdgcn_sched_barrier(0);           // (behind what was asked for before: see arrive)
        const int at = BIG_SLICE * d < g.K - 16 ? BIG_SLICE * d : g.K - 16;
        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(line + at),
                                         (__attribute__((address_space(3))) void*)unread, 4, 0, 0);
    };
    struct Operands {
        v8i a[4], b[4];
    };
    const int row8 = (lane & 31) * 8;
    const auto read = [&](auto b, int half, Operands& h) {
        const int turn = (half * 4 + (lane >> 5)) ^ row_key(lane & 31);
        const v4i* x = (decltype(b)::value ? buffer1 : buffer0) + wm * 8 + row8;
        const v4i* w = (decltype(b)::value ? buffer1 : buffer0) + OPERAND + wn * 8 + row8;
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            const v4i p = w[256 * t + turn], q = w[256 * t + (turn ^ 2)];
            h.a[t] = v8i{p.x, p.y, p.z, p.w, q.x, q.y, q.z, q.w};
            const v4i u = x[256 * t + turn], v = x[256 * t + (turn ^ 2)];
            h.b[t] = v8i{u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
        }
    };
    v16f acc[4][4];
#pragma unroll
    for (int a = 0; a < 4; ++a)
#pragma unroll
        for (int b = 0; b < 4; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[a][b][i] = 0.f;
    const auto multiply = [&](const Operands& h) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(h.a[i], h.b[j], acc[i][j], 0, 0, 0,
                                                                            0, 0, 0);
    };
    // Requests and reads go between the matrix instructions, requests first.
    const auto interleave = [](bool requests) {
        if (requests) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);   // a matrix instruction
                __builtin_amdgcn_sched_group_barrier(0x020, 2, 0);   // two requests
            }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);       // two reads
        }
        if (!requests) __builtin_amdgcn_sched_group_barrier(0x008, 8, 0);
        __builtin_amdgcn_sched_barrier(0);
    };
    // Everything asked for has arrived, for everybody, and everybody's reads are done.  BUT: the last requests
    // that need not have arrived (they come in order).
    const auto arrive = [](auto but) {
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_waitcnt(0x0070 | decltype(but)::value);   // vmcnt(BUT) lgkmcnt(0)
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    // zero where half `half` of double slice d is behind the end of k
    const auto cut = [&](int d, int half, Operands& h) {
        const int there = g.K / 16 - 8 * d - 4 * half - (lane >> 5);
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                h.a[t][i] = there > i / 4 * 2 ? h.a[t][i] : 0;
                h.b[t][i] = there > i / 4 * 2 ? h.b[t][i] : 0;
            }
    };
    const int doubles = (g.K + BIG_SLICE - 1) / BIG_SLICE;
    constexpr std::integral_constant<int, 0> b0{};
    constexpr std::integral_constant<int, 1> b1{};
    Operands first, second;
    const auto step = [&](auto b, int d) {
        constexpr std::integral_constant<int, 1 - decltype(b)::value> other{};
        const bool ends = (d + 1) * BIG_SLICE > g.K;
        if (ends) cut(d, 0, first);
        read(b, 1, second);
        multiply(first);
        interleave(false);
        if (ends) cut(d, 1, second);
        arrive(b1);                                  // d + 1 is there, nobody reads d any more
        fetch(b, d + 2);                             // (behind the end of k: not used)
        read(other, 0, first);
        multiply(second);
        interleave(true);
        warm(d + 3);
    };
    fetch(b0, 0);
    load_factors(g, m0, n0, factors);
    arrive(b0);
    fetch(b1, 1);
    warm(2);
    read(b0, 0, first);
    for (int d = 0; d < doubles; d += 2) step(b0, d), step(b1, d + 1);
    arrive(b0);                                      // nothing is under way, the operands' LDS is free
    // (a wavefront's 32 KB lie in one of the buffers)
    char* region = reinterpret_cast<char*>(wave < 2 ? buffer0 : buffer1) + (wave & 1) * (128 * 128 * (int)sizeof(T));
    write_rows<T, 128, 4>(g, factors, region, m0, n0, wm, wn, lane,
                          [&](int i, int j, int e) { return acc[i][j][e]; });
}

static bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace kvae

using namespace kvae;

extern "C" int kvae_linear_8bit(int64_t M, int64_t N, int64_t K, const void* x, const void* x_scale,
                                const void* w, const void* w_scale, const void* bias, int out_dtype,
                                void* y, void* stream) {
    if (M < 1 || N < 1 || K < 1 || !x || !x_scale || !w || !w_scale || !y) return KVAE_E_BADARG;
    // 32-bit offsets inside a tile of 256 rows, fewer than 2^32 threads in a launch (512 for 16 columns)
    if (N > (1 << 26) || K > (1 << 22) || M > (1L << 31) || M > (1L << 40) / N) return KVAE_E_TOOLARGE;
    return for_element_type(out_dtype, [&](auto e) {
        using T = decltype(e);
        const LinearArgs g{(long)M, (int)N, (int)K, static_cast<const uint8_t*>(x),
                           static_cast<const uint8_t*>(w), static_cast<const float*>(x_scale),
                           static_cast<const float*>(w_scale), static_cast<const float*>(bias), y};
        const hipStream_t s = static_cast<hipStream_t>(stream);
        const long tn = (N + TILE - 1) / TILE;
        const long bn = (N + BIG - 1) / BIG, bm = (M + BIG - 1) / BIG;
        // Which form, by sizes (bfloat16 results, us):
        // - a few rows: blocks of 16 columns by all rows up to 64, k shared out; 64 x 4096 x 4096 7 against 10 in
        //   blocks of 64 x 64 and 27 in tiles of 128, 512^3 3.9 against 6.1 and 6.2.  Also where k < 16.
        // - 64 x 64 blocks, k shared out, when there are 96 to 256 of them, one for a unit of the card (up to two
        //   if k is long): 128 x 4096 x 4096 10 against 13 in 16 columns and 27 in tiles, 256 x 4096 x 4096 12
        //   against 23 and 27, 1024^3 6.1 against 10 and 9.4; 512 of them with k = 4096 21 against 29 in tiles,
        //   with k = 1024 11.1 against 10.
        // - tiles of 256 x 256 whose results fill five eighths of the card's units in every round, k long
        //   enough to hide that such a tile neither starts nor ends under another one's work, and rows of
        //   whole 16-byte pieces: large tiles.  16384 x 4096: k = 1280 94 against 101 in tiles of 128,
        //   k = 1024 83 against 87, k = 768 75 against 69.  3328 x 3328 x 4096 (66 % of the units) 49 against
        //   54, 4352 x 4096 x 4096 (53 %) 92 against 84.
        // (blockIdx.y is 16 bits: rows beyond go in further launches)
        const auto in_parts = [&](long rows_each, auto&& launch) {
            for (long first = 0; first < M; first += 65535 * rows_each) {
                LinearArgs h = g;
                const long rows = M - first < 65535 * rows_each ? M - first : 65535 * rows_each;
                h.M = rows;
                h.x = g.x + first * K;
                h.sx = g.sx + first;
                h.y = static_cast<T*>(y) + first * N;
                launch(h, (unsigned)((rows + rows_each - 1) / rows_each));
            }
            return hipGetLastError() == hipSuccess ? KVAE_OK : KVAE_E_LAUNCH;
        };
        const long blocks64 = ((M + 63) / 64) * ((N + 63) / 64);
        const bool blocks = M > 32 && K >= 16 && blocks64 >= 96 && (blocks64 <= 256 || (blocks64 <= 512 && K >= 2048));
        if (blocks || M <= 64 || K < 16 || blocks64 < 96) {
            const auto go = [&](auto mt, auto nt) {
                constexpr int MT = decltype(mt)::value, NT = decltype(nt)::value;
                return in_parts(16 * MT, [&](const LinearArgs& h, unsigned count) {
                    linear_few_rows_kernel<T, MT, NT>
                        <<<dim3((unsigned)((N + 16 * NT - 1) / (16 * NT)), count), 64 * FEW_WAVES, 0, s>>>(h);
                });
            };
            constexpr std::integral_constant<int, 1> one{};
            constexpr std::integral_constant<int, 2> two{};
            constexpr std::integral_constant<int, 4> four{};
            if (blocks) return go(four, four);
            if (M <= 16) return go(one, one);
            if (M <= 32) return go(two, one);
            return go(four, one);
        }
        if constexpr (!WIDENED<T>) {
            const long units = device_compute_units(), rounds = (bn * bm + units - 1) / units;
            if (M * N * 8 >= rounds * units * (5 * BIG * BIG) && K >= 1024 && K % 16 == 0 && aligned16(x) && aligned16(w)) {
                const unsigned blocks = (unsigned)((bn * bm + 7) / 8 * 8);
                linear_big_kernel<T><<<dim3(blocks), 256, 0, s>>>(g, (int)bn, (int)bm);
                return hipGetLastError() == hipSuccess ? KVAE_OK : KVAE_E_LAUNCH;
            }
        }
        return in_parts(TILE, [&](const LinearArgs& h, unsigned count) {
            linear_tile_kernel<T><<<dim3((unsigned)tn, count), 256, 0, s>>>(h);
        });
    });
}
