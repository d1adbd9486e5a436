// AdamW step over many tensors in one launch, on gfx950, with the states in float or in 8 bits:
//
//   m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g^2
//   p = p (1 - lr wd) - (lr / (1 - b1^t)) m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// A stream over memory: parameter, gradient and both states are read once and written once (float:
// 28 bytes an element; 8-bit states: 16 bytes).  The tensors' addresses travel with the launch, so
// a model of some forty small tensors costs one launch; a workgroup finds its tensor by bisection.
// Measured: 40 float tensors of 250000 elements together 8.7 us; 60 million elements in 150 tensors with
// 8-bit states 212 us in four launches (964 MB, 4.5 TB/s, where a large copy moves 5.1: the hashes and
// conversions of two states take as long as their bytes), with float states 342 (1680 MB, 4.9); bfloat16 with
// float copies that follow the parameter 387 (1800 MB, 4.7), with 8-bit states 242 (1080 MB, 4.5).
//
// 8-bit states.  Blocks of 256 elements hold m and sqrt(v) as e4m3 values times one scale per
// block (max / 448).  sqrt(v) and not v: e4m3 spans 2^18 between its largest and its smallest
// positive value, so v spans 2^36 within a block.  Two rules keep training sound:
// - Rounding is stochastic.  v moves by a thousandth of itself a step (b2 = 0.999) and the code's
//   step is a sixteenth: to the nearest it would never move.  The random bits are a hash of
//   (seed, step, index), so a run can be repeated bit for bit.
// - The code of a positive sqrt(v) is never zero: the update divides by it, and a zero under an m
//   that was rounded up would make a step of a thousand times lr.
// The arithmetic of the states is written without contraction into fused multiply-adds and with
// correctly rounded roots and scales' reciprocals: codes come out the same as from the formulas
// above evaluated one operation at a time.
#include "narrow_types.h"

namespace kvae {

constexpr int ADAM_THREADS = 256;
constexpr int PER_LANE = 16;                         // elements: 16 lanes hold a block of 256
constexpr int ADAM_CHUNK = ADAM_THREADS * PER_LANE;  // elements of a workgroup
constexpr int QUANT_BLOCK = KVAE_ADAMW_BLOCK;
constexpr int TABLE = KVAE_ADAMW_MAX_TENSORS;
static_assert(QUANT_BLOCK == 16 * PER_LANE, "a block is one row of 16 lanes");

struct AdamArgs {
    kvae_adamw_tensor t[TABLE];
    int first_chunk[TABLE + 1];                      // workgroup -> tensor
    unsigned first_block[TABLE];                     // blocks of 256 of the tensors before (hash index)
    int count;
    float lr, beta1, beta2, eps, decay;              // decay: lr * weight_decay
    float one_minus_beta1, one_minus_beta2;
    float rate, root_fix;                            // lr / (1 - b1^t), 1 / sqrt(1 - b2^t)
    unsigned key;                                    // seed + t * 0x9E3779B9
    double dbeta1, dbeta2, dlr, ddecay;              // for a step count that lives on the device
    const int64_t* step;
    const float* lr_device;
    unsigned seed;
    int follow;
};

template <int CTRL>
__device__ __forceinline__ float row_exchange(float x) {
    return __builtin_bit_cast(
        float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ float max16(float v) {
    v = fmaxf(v, row_exchange<0xB1>(v));
    v = fmaxf(v, row_exchange<0x4E>(v));
    v = fmaxf(v, row_exchange<0x141>(v));
    return fmaxf(v, row_exchange<0x140>(v));
}

constexpr float E4M3_MAX = 448.f;
constexpr float SMALLEST_SCALE = 1.17549435e-38f;    // smallest normal: its reciprocal is finite

// Two rounds of multiply and shift (C. Wellons' 32-bit mix) over a multiplicative start.
constexpr unsigned INDEX_FACTOR = 0x9E3779B1u;
__device__ __forceinline__ unsigned random_bits(unsigned h) {   // h = index * INDEX_FACTOR + key
    h = (h ^ (h >> 16)) * 0x7FEB352Du;
    h = (h ^ (h >> 15)) * 0x846CA68Bu;
    return h ^ (h >> 16);
}

// x to an e4m3 byte, up or down by 16 random bits; POSITIVE (x >= 0): never to zero unless x is.
// Where the value is normal in e4m3 (2^-6 and more) its three mantissa bits are the float's first
// three: the random bits are added below them and cut off, and the exponent is moved from bias 127
// to 7.  Below, the code counts steps of 2^-9.
template <bool POSITIVE>
__device__ __forceinline__ unsigned round_e4m3(float x, unsigned random16) {
    const unsigned bits = __builtin_bit_cast(unsigned, x), size = bits & 0x7FFFFFFFu;
    const float t = fabsf(x);
    const unsigned normal = ((size + (random16 << 4) + 8u) >> 20) - (120u << 3);
    unsigned small = (unsigned)__fadd_rn(t * 512.f, __builtin_fmaf((float)random16, 1.f / 65536.f, 0.5f / 65536.f));
    if constexpr (POSITIVE) small = t > 0.f && small == 0u ? 1u : small;
    unsigned code = t < 0.015625f ? small : normal;
    code = code < 0x7Eu ? code : 0x7Eu;              // at most 448
    code = t == t ? code : 0x7Fu;
    return code | ((bits >> 24) & 0x80u);
}

// A lane's 16 elements are four groups of four, 64 elements apart: 16 lanes hold a block of 256, and
// every access of theirs is one contiguous run.  n: elements of the tensor from the lane's first on.
constexpr int GROUP = 4, GROUPS = PER_LANE / GROUP, APART = 16 * GROUP;

// FULL: all of the workgroup's elements are there.
template <bool FULL, typename T>
__device__ __forceinline__ void load16(const T* p, long n, float (&x)[PER_LANE]) {
#pragma unroll
    for (int k = 0; k < GROUPS; ++k) {
        if (FULL || n >= k * APART + GROUP) {
            const Pack<T, GROUP> q = load_pack<T, GROUP>(p + k * APART);
#pragma unroll
            for (int v = 0; v < GROUP; ++v) x[k * GROUP + v] = widen(q.v[v]);
        } else {
#pragma unroll
            for (int v = 0; v < GROUP; ++v) x[k * GROUP + v] = k * APART + v < n ? widen(p[k * APART + v]) : 0.f;
        }
    }
}
template <bool FULL, typename T>
__device__ __forceinline__ void store16(T* p, long n, const float (&x)[PER_LANE]) {
#pragma unroll
    for (int k = 0; k < GROUPS; ++k) {
        if (FULL || n >= k * APART + GROUP) {
            Pack<T, GROUP> q;
#pragma unroll
            for (int v = 0; v < GROUP; ++v) q.v[v] = narrow<T>(x[k * GROUP + v]);
            store_pack<T, GROUP>(p + k * APART, q);
        } else {
#pragma unroll
            for (int v = 0; v < GROUP; ++v)
                if (k * APART + v < n) p[k * APART + v] = narrow<T>(x[k * GROUP + v]);
        }
    }
}
// four e4m3 bytes at any address
struct __attribute__((packed)) Word { uint32_t w; };
template <bool FULL>
__device__ __forceinline__ void load_codes(const uint8_t* p, long n, float scale, float (&x)[PER_LANE]) {
#pragma unroll
    for (int k = 0; k < GROUPS; ++k) {
        uint32_t w = 0;
        if (FULL || n >= k * APART + GROUP) {
            w = reinterpret_cast<const Word*>(p + k * APART)->w;
        } else {
#pragma unroll
            for (int v = 0; v < GROUP; ++v)
                if (k * APART + v < n) w |= (uint32_t)p[k * APART + v] << (8 * v);
        }
        x[k * GROUP] = __builtin_amdgcn_cvt_f32_fp8(w, 0) * scale;
        x[k * GROUP + 1] = __builtin_amdgcn_cvt_f32_fp8(w, 1) * scale;
        x[k * GROUP + 2] = __builtin_amdgcn_cvt_f32_fp8(w, 2) * scale;
        x[k * GROUP + 3] = __builtin_amdgcn_cvt_f32_fp8(w, 3) * scale;
    }
}
// Codes and scale of a block of 256 over a row of 16 lanes.  SHIFT: which half of the hash decides.
template <bool FULL, bool POSITIVE, int SHIFT>
__device__ __forceinline__ void store_codes(uint8_t* p, float* scale_at, bool first, long n,
                                            const float (&x)[PER_LANE], const unsigned (&random)[PER_LANE]) {
    float big = 0.f;
#pragma unroll
    for (int i = 0; i < PER_LANE; ++i) big = fmaxf(big, fabsf(x[i]));
    big = max16(big);
    const float scale = fmaxf(big * (1.f / E4M3_MAX), SMALLEST_SCALE);
    const float inverse = 1.f / scale;
    if (first) *scale_at = scale;
#pragma unroll
    for (int k = 0; k < GROUPS; ++k) {
        uint32_t w = 0;
#pragma unroll
        for (int v = 0; v < GROUP; ++v) {
            const unsigned r = random[k * GROUP + v];
            w |= round_e4m3<POSITIVE>(x[k * GROUP + v] * inverse, SHIFT ? r >> 16 : r & 0xFFFFu) << (8 * v);
        }
        if (FULL || n >= k * APART + GROUP) {
            reinterpret_cast<Word*>(p + k * APART)->w = w;
        } else {
#pragma unroll
            for (int v = 0; v < GROUP; ++v)
                if (k * APART + v < n) p[k * APART + v] = (uint8_t)(w >> (8 * v));
        }
    }
}

template <typename T, bool EIGHT, bool MASTER>
__global__ void __launch_bounds__(ADAM_THREADS) adamw_kernel(const AdamArgs g) {
#pragma clang fp contract(off)
    __shared__ float fixes[2];
    float lr = g.lr, decay = g.decay, rate = g.rate, root_fix = g.root_fix;
    unsigned key = g.key;
    if (g.step) {                                    // captured: step count and rate live on the device
        if (threadIdx.x == 0) {
            const double t = (double)*g.step;
            const double rate1 = g.lr_device ? (double)*g.lr_device : g.dlr;
            fixes[0] = (float)(rate1 / -expm1(t * log(g.dbeta1)));
            fixes[1] = (float)(1.0 / sqrt(-expm1(t * log(g.dbeta2))));
        }
        __syncthreads();
        rate = fixes[0];
        root_fix = fixes[1];
        lr = g.lr_device ? *g.lr_device : lr;
        decay = (float)((g.lr_device ? (double)*g.lr_device : g.dlr) * g.ddecay);
        key = g.seed + (unsigned)*g.step * 0x9E3779B9u;
    }
    int low = 0, high = g.count;                     // first_chunk[low] <= blockIdx.x < first_chunk[high]
    while (high - low > 1) {
        const int mid = (low + high) / 2;
        if (g.first_chunk[mid] <= (int)blockIdx.x) low = mid; else high = mid;
    }
    const kvae_adamw_tensor t = g.t[low];
    const long block = (long)(blockIdx.x - g.first_chunk[low]) * (ADAM_CHUNK / QUANT_BLOCK) + threadIdx.x / 16;
    const int inside = (threadIdx.x & 15) * GROUP;
    const long at = block * QUANT_BLOCK + inside, n = t.numel - at;
    // a row of 16 lanes (one block) leaves together, so that max16 finds all its lanes
    if (block * QUANT_BLOCK >= t.numel) return;
    const auto update = [&](auto full) {
#pragma clang fp contract(off)
        constexpr bool FULL = decltype(full)::value;
        float p[PER_LANE], grad[PER_LANE], m[PER_LANE], v[PER_LANE];
        if constexpr (MASTER) {
            load16<FULL>(static_cast<const float*>(t.master) + at, n, p);
            if (g.follow) {                          // (2 bytes an element of 28 more to read)
                float q[PER_LANE];
                load16<FULL>(static_cast<const T*>(t.param) + at, n, q);
#pragma unroll
                for (int i = 0; i < PER_LANE; ++i) p[i] = widen(narrow<T>(p[i])) == q[i] ? p[i] : q[i];
            }
        } else {
            load16<FULL>(static_cast<const T*>(t.param) + at, n, p);
        }
        load16<FULL>(static_cast<const T*>(t.grad) + at, n, grad);
        if constexpr (EIGHT) {
            load_codes<FULL>(static_cast<const uint8_t*>(t.exp_avg) + at, n,
                             static_cast<const float*>(t.exp_avg_scale)[block], m);
            load_codes<FULL>(static_cast<const uint8_t*>(t.exp_avg_sq) + at, n,
                             static_cast<const float*>(t.exp_avg_sq_scale)[block], v);
#pragma unroll
            for (int i = 0; i < PER_LANE; ++i) v[i] = v[i] * v[i];
        } else {
            load16<FULL>(static_cast<const float*>(t.exp_avg) + at, n, m);
            load16<FULL>(static_cast<const float*>(t.exp_avg_sq) + at, n, v);
        }
#pragma unroll
        for (int i = 0; i < PER_LANE; ++i) {
            m[i] = m[i] * g.beta1 + grad[i] * g.one_minus_beta1;
            v[i] = v[i] * g.beta2 + (grad[i] * grad[i]) * g.one_minus_beta2;
            const float root = sqrtf(v[i]);
            if constexpr (EIGHT) v[i] = root;        // from here on sqrt(v)
            // (the reciprocal is within an ulp; a quotient to the last bit would cost eight
            // instructions and moves the update by 1e-7 of itself)
            p[i] = p[i] * (1.f - decay) - rate * (m[i] * __builtin_amdgcn_rcpf(root * root_fix + g.eps));
        }
        if constexpr (MASTER) store16<FULL>(static_cast<float*>(t.master) + at, n, p);
        store16<FULL>(static_cast<T*>(t.param) + at, n, p);
        if constexpr (EIGHT) {
            const bool first = inside == 0;
            // elements 2^32 apart have the same low half of the index: the high one gives them another key
            const unsigned long index = (unsigned long)g.first_block[low] * QUANT_BLOCK + (unsigned long)at;
            const unsigned high = (unsigned)(index >> 32);
            if (high) key = random_bits(key + high * INDEX_FACTOR);
            const unsigned h = (unsigned)index * INDEX_FACTOR + key;
            unsigned random[PER_LANE];
#pragma unroll
            for (int i = 0; i < PER_LANE; ++i)
                random[i] = random_bits(h + (unsigned)((i / GROUP) * APART + i % GROUP) * INDEX_FACTOR);
            store_codes<FULL, false, 0>(static_cast<uint8_t*>(t.exp_avg) + at,
                                        static_cast<float*>(t.exp_avg_scale) + block, first, n, m, random);
            store_codes<FULL, true, 1>(static_cast<uint8_t*>(t.exp_avg_sq) + at,
                                       static_cast<float*>(t.exp_avg_sq_scale) + block, first, n, v, random);
        } else {
            store16<FULL>(static_cast<float*>(t.exp_avg) + at, n, m);
            store16<FULL>(static_cast<float*>(t.exp_avg_sq) + at, n, v);
        }
    };
    if ((long)(blockIdx.x - g.first_chunk[low] + 1) * ADAM_CHUNK <= t.numel) {
        update(std::true_type{});
    } else {
        update(std::false_type{});
    }
}

}  // namespace kvae

using namespace kvae;

extern "C" int kvae_adamw_step(const kvae_adamw* d, void* stream) {
    if (!d || d->count < 1 || d->count > TABLE || !d->tensors) return KVAE_E_BADARG;
    if (d->state_bits != 32 && d->state_bits != 8) return KVAE_E_UNSUPPORTED;
    if (d->dtype != KVAE_F32 && d->dtype != KVAE_BF16 && d->dtype != KVAE_F16) return KVAE_E_UNSUPPORTED;
    if (!d->step_device && d->step < 1) return KVAE_E_BADARG;
    static_assert(sizeof(AdamArgs) <= 4096, "arguments of a launch");
    AdamArgs g{};
    long chunks = 0, blocks = d->first_block;
    const bool master = d->tensors[0].master != nullptr;
    for (int i = 0; i < d->count; ++i) {
        const kvae_adamw_tensor& t = d->tensors[i];
        if (t.numel < 1 || !t.param || !t.grad || !t.exp_avg || !t.exp_avg_sq) return KVAE_E_BADARG;
        if (d->state_bits == 8 && (!t.exp_avg_scale || !t.exp_avg_sq_scale)) return KVAE_E_BADARG;
        if ((t.master != nullptr) != master) return KVAE_E_BADARG;
        g.t[i] = t;
        g.first_chunk[i] = (int)chunks;
        g.first_block[i] = (unsigned)blocks;
        chunks += (t.numel + ADAM_CHUNK - 1) / ADAM_CHUNK;
        blocks += (t.numel + QUANT_BLOCK - 1) / QUANT_BLOCK;
        if (chunks >= (1L << 32) / ADAM_THREADS) return KVAE_E_TOOLARGE;   // a launch has fewer than 2^32 threads
    }
    g.first_chunk[d->count] = (int)chunks;
    g.count = d->count;
    g.lr = (float)d->lr, g.beta1 = (float)d->beta1, g.beta2 = (float)d->beta2, g.eps = (float)d->eps;
    g.one_minus_beta1 = (float)(1.0 - d->beta1), g.one_minus_beta2 = (float)(1.0 - d->beta2);
    g.decay = (float)(d->lr * d->weight_decay);
    g.dbeta1 = d->beta1, g.dbeta2 = d->beta2, g.dlr = d->lr, g.ddecay = d->weight_decay;
    g.step = static_cast<const int64_t*>(d->step_device);
    g.lr_device = static_cast<const float*>(d->lr_device);
    g.seed = d->seed;
    g.follow = d->follow_param;
    if (!g.step) {
        g.rate = (float)(d->lr / (1.0 - pow(d->beta1, (double)d->step)));
        g.root_fix = (float)(1.0 / sqrt(1.0 - pow(d->beta2, (double)d->step)));
        g.key = d->seed + (unsigned)d->step * 0x9E3779B9u;
    }
    return for_element_type(d->dtype, [&](auto e) {
        using T = decltype(e);
        const hipStream_t s = static_cast<hipStream_t>(stream);
        const auto go = [&](auto eight, auto with_master) {
            adamw_kernel<T, decltype(eight)::value, decltype(with_master)::value>
                <<<dim3((unsigned)chunks), ADAM_THREADS, 0, s>>>(g);
        };
        const auto with_bits = [&](auto with_master) {
            d->state_bits == 8 ? go(std::true_type{}, with_master) : go(std::false_type{}, with_master);
        };
        master ? with_bits(std::true_type{}) : with_bits(std::false_type{});
        return hipGetLastError() == hipSuccess ? KVAE_OK : KVAE_E_LAUNCH;
    });
}
