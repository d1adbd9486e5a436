// Gated linear recurrence over a sequence on gfx950, forward, backward and one step.
//
//   f = sigmoid(forget), c_t = f_t c_{t-1} + (1 - f_t) x_t, y_t = c_t silu(o_t) (or c_t)
//
// element-wise over (B,H): unlike the LSTM's recurrence there is no matrix product between steps,
// so the work is a stream over memory: the forward pass reads u = [x | forget | o] and writes y,
// the backward pass reads u and dy and writes du.  The state is float whatever the element type.
//
// Mapping.  A lane owns one channel (float) or two neighbouring ones (16-bit types) of one
// sequence, so that a wavefront moves 256 contiguous bytes per tensor and step.  It takes its steps
// in chunks (16 float, 8 16-bit), loads a whole chunk before using it, and keeps what a step needs
// in registers: f and (1 - f) x.  With many channels a wavefront walks over the sequence alone.
// With fewer, the four wavefronts of a workgroup take four consecutive chunks of the same channels
// at once: each composes its chunk to c_out = P c_in + S in registers, the compositions meet in LDS,
// and every wavefront then runs its chunk from its own start state, so that u is still read once.
// Only when even that does not fill the card is the sequence cut into segments for several
// workgroups: a launch that composes each segment, then the same kernel, which folds the
// compositions of the segments before its own into its start state.
//
// The backward pass does not read y (which is rounded to the element type, and gated): the
// forward pass leaves the float state before every chunk, and the backward pass runs a chunk's
// recurrence again from there in registers, on the x and forget it has to read anyway.
//
// Bound by memory.  1000 steps of 4096 x 64 float channels: 4.2 GB in 0.86 ms forward and 7.3 GB in
// 1.46 ms backward, 4.9 and 5.0 TB/s, where a large copy reaches 5.1; 1000 masked steps of 256 x 256
// bfloat16 channels 127 and 205 us; 20 steps of 32 x 128 float channels 4.4 and 6.8 us.
#include "narrow_types.h"

namespace kvae {

constexpr int SCAN_BLOCK = 256;
constexpr int TOGETHER = 4;                  // wavefronts that share a stretch of time
constexpr int MOST_SEGMENTS = 128;

struct ScanArgs {
    long T, B, H;
    const void* u;
    long u_t, u_b;               // strides of u in elements
    const uint8_t* mask;
    long mask_t, mask_b;
    const float* h0;
    void* y;
    float* last;
    float* states;
    const void* dy;
    long dy_t, dy_b;
    const float* dlast;
    void* du;
    float* dh0;
    long groups;                 // lanes per sequence
    long seg;                    // steps per segment, a multiple of the chunk
    int segs;
    float2* compose;             // (segs, B, H): P and S of each segment
};

// exp(z) from the hardware's 2^x.  The argument's one rounding is up to 2^-24 of it, which is a relative error of
// |z| 2^-24 of the result, to which the instruction adds an ulp: ten units at |z| = 10.  (Two terms of the argument
// would save that at a multiply-add an exponential; a gate of that size changes little by it.)
__device__ __forceinline__ float exp_of(float z) { return __builtin_amdgcn_exp2f(z * 1.44269504f); }

struct Gate {
    float f, keep;               // sigmoid(z), 1 - sigmoid(z), both without cancellation; NaN stays
};
__device__ __forceinline__ Gate sigmoid_pair(float z) {
    const float e = exp_of(-fabsf(z));
    const float big = __builtin_amdgcn_rcpf(1.f + e);
    const float small = e * big;
    return z >= 0.f ? Gate{big, small} : Gate{small, big};
}
__device__ __forceinline__ float sigmoid(float z) { return __builtin_amdgcn_rcpf(1.f + exp_of(-z)); }

// A lane's place: sequence b0 + b with b0 the workgroup's first, channels h .. h + V - 1.  Addresses
// are a uniform base (scalar registers, moved from step to step by scalar instructions) plus a
// 32-bit lane offset that stays: 64-bit lane pointers would be kept for every step and tensor and
// take more registers than the data.
// The last lane of a sequence is moved back so that its V channels end at H, and lanes behind the
// last sequence repeat its last lane (so that a workgroup stays whole): a channel that two lanes own
// gets the same values from both.
struct Place {
    long b0;
    unsigned b, h;
    unsigned seg;                // segment of the time axis
};
// Workgroups go round the eight dies (id % 8).  With segments each die gets a run of neighbouring channel
// groups: a group of 64 lanes begins anywhere in a 128-byte line, and the line that two of them share is
// then fetched into one cache (32768 steps of 520 half channels: 19 -> 17 us to compose, 28 -> 26 to run).
// Without, a whole sequence passes before its neighbour is far behind or ahead, and there is nothing to gain.
template <int V, int W>
__device__ __forceinline__ Place scan_place(const ScanArgs& g) {
    Place p;
    p.seg = 0;
    long first = (long)blockIdx.x * (W == 1 ? SCAN_BLOCK : 64);
    if (W > 1 && g.segs > 1) {
        const unsigned id = blockIdx.y * gridDim.x + blockIdx.x, total = gridDim.x * gridDim.y;
        const unsigned die = id & 7, each = total >> 3, longer = total & 7;
        const unsigned mine = die * each + (die < longer ? die : longer) + (id >> 3);
        p.seg = mine / gridDim.x;
        first = (long)(mine - p.seg * gridDim.x) * 64;
    }
    p.b0 = first / g.groups;
    const long left = g.B * g.groups - first;        // lanes from here to the last one
    unsigned lane = W == 1 ? threadIdx.x : threadIdx.x & 63;
    if (lane >= left) lane = (unsigned)left - 1;
    const unsigned groups = (unsigned)g.groups, inside = (unsigned)(first - p.b0 * g.groups) + lane;
    p.b = inside / groups;
    p.h = (inside - p.b * groups) * V;
    if (p.h > (unsigned)g.H - V) p.h = (unsigned)g.H - V;
    return p;
}
template <typename T, int V>
__device__ __forceinline__ Pack<T, V> load_off(const void* base, unsigned bytes) {
    return load_pack<T, V>(reinterpret_cast<const T*>(static_cast<const char*>(base) + bytes));
}
template <typename T, int V>
__device__ __forceinline__ void store_off(void* base, unsigned bytes, const Pack<T, V>& x) {
    store_pack<T, V>(reinterpret_cast<T*>(static_cast<char*>(base) + bytes), x);
}

template <int V>
struct Map {                     // c -> P c + S
    float P[V], S[V];
};
template <int V>
__device__ __forceinline__ Map<V> identity() {
    Map<V> m;
#pragma unroll
    for (int v = 0; v < V; ++v) m.P[v] = 1.f, m.S[v] = 0.f;
    return m;
}
// first `a`, then `b`
template <int V>
__device__ __forceinline__ Map<V> then(const Map<V>& a, const Map<V>& b) {
    Map<V> m;
#pragma unroll
    for (int v = 0; v < V; ++v) m.P[v] = a.P[v] * b.P[v], m.S[v] = b.P[v] * a.S[v] + b.S[v];
    return m;
}

// What the wavefronts of a workgroup tell each other: one map per wavefront and lane.
template <int V, int W>
struct Exchange {
    Map<V> m[W][64];
};

// State (or, REVERSE, gradient) that a segment starts from: `init`, then the maps of the
// segments that come before it in walking order.  With several wavefronts each takes every W-th of
// them in one stretch and the stretches meet in LDS.
template <int V, int W, bool REVERSE>
__device__ __forceinline__ void segment_start(const ScanArgs& g, int seg, int wave, long at, const float* init, Exchange<V, W>* ex,
                                              float (&c)[V]) {
#pragma unroll
    for (int v = 0; v < V; ++v) c[v] = init ? init[at + v] : 0.f;
    if (g.segs == 1) return;
    const long plane = g.B * g.H;
    const int before = REVERSE ? g.segs - 1 - seg : seg;
    const int each = (before + W - 1) / W;
    const int begin = wave * each < before ? wave * each : before;
    const int end = begin + each < before ? begin + each : before;
    Map<V> m = identity<V>();
#pragma unroll 8
    for (int i = begin; i < end; ++i) {
        const float2* p = g.compose + (REVERSE ? g.segs - 1 - i : i) * plane + at;
        Map<V> k;
#pragma unroll
        for (int v = 0; v < V; ++v) k.P[v] = p[v].x, k.S[v] = p[v].y;
        m = then<V>(m, k);
    }
    if constexpr (W > 1) {
        ex->m[wave][threadIdx.x & 63] = m;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const Map<V> k = ex->m[w][threadIdx.x & 63];
#pragma unroll
            for (int v = 0; v < V; ++v) c[v] = k.P[v] * c[v] + k.S[v];
        }
    } else {
#pragma unroll
        for (int v = 0; v < V; ++v) c[v] = m.P[v] * c[v] + m.S[v];
    }
}

// Chunks come in two forms of the same code.  FULL: all L steps are there.  Otherwise n of them are
// (possibly none): the loads of the others repeat the last step of the segment, so that they stay
// inside the tensors, and count as masked, so that no load waits behind a branch.

// The scheduler works step by step: left alone it computes all steps of a chunk side by side, which
// takes several times the registers (and spills) for no gain, as other wavefronts fill the gaps.
__device__ __forceinline__ void keep_order() { __builtin_amdgcn_sched_barrier(0); }

// p + by, a scalar address the compiler takes as new: it would otherwise work out the addresses of
// all steps of all tensors ahead of the loop and run out of scalar registers.
template <typename P>
__device__ __forceinline__ P* move_on(P* p, long by) {
    p += by;
    asm("" : "+s"(p));
    return p;
}

// A loaded word, unpacked from here on and not before (unpacked 16-bit pairs take twice the registers).
template <typename T, int V>
__device__ __forceinline__ Pack<T, V> now(const Pack<T, V>& x) {
    if constexpr (sizeof(x) == 4) {
        unsigned word = __builtin_bit_cast(unsigned, x);
        asm volatile("" : "+v"(word));
        return __builtin_bit_cast(Pack<T, V>, word);
    } else {
        return x;
    }
}

// A value computed here and not where it is used (what it is computed from would be kept instead).
__device__ __forceinline__ void settle(float& x) { asm volatile("" : "+v"(x)); }

// Steps t0 .. t0 + L - 1 of the lane's channels: x, forget, output gate and, BACKWARD, dy.
template <typename T, int V, int L, bool GATED, bool MASKED, bool FULL, bool WITH_X, bool WITH_GATE, bool WITH_DY>
__device__ __forceinline__ void load_steps(const ScanArgs& g, const Place& at, long t0, long t_end, int n,
                                           Pack<T, V> (&x)[L], Pack<T, V> (&z)[L], Pack<T, V> (&o)[L],
                                           Pack<T, V> (&d)[L], bool (&live)[L]) {
    const long t = FULL || t0 < t_end ? t0 : t_end - 1;
    const T* p = static_cast<const T*>(g.u) + at.b0 * g.u_b + t * g.u_t;
    const T* q = WITH_DY ? static_cast<const T*>(g.dy) + at.b0 * g.dy_b + t * g.dy_t : nullptr;
    const uint8_t* m = MASKED ? g.mask + t * g.mask_t + at.b0 * g.mask_b : nullptr;
    const unsigned pu = (at.b * (unsigned)g.u_b + at.h) * (unsigned)sizeof(T);
    const unsigned qu = WITH_DY ? (at.b * (unsigned)g.dy_b + at.h) * (unsigned)sizeof(T) : 0u;
    const unsigned mu = MASKED ? at.b * (unsigned)g.mask_b : 0u;
#pragma unroll
    for (int i = 0; i < L; ++i) {
        if constexpr (WITH_X) x[i] = load_off<T, V>(p, pu);
        z[i] = load_off<T, V>(p + g.H, pu);
        if constexpr (GATED && WITH_GATE) o[i] = load_off<T, V>(p + 2 * g.H, pu);
        if constexpr (WITH_DY) d[i] = load_off<T, V>(q, qu);
        live[i] = FULL || i < n;
        if constexpr (MASKED) live[i] = live[i] && m[mu] != 0;
        const bool on = FULL || i + 1 < n;
        p = move_on(p, on ? g.u_t : 0);
        if constexpr (WITH_DY) q = move_on(q, on ? g.dy_t : 0);
        if constexpr (MASKED) m = move_on(m, on ? g.mask_t : 0);
    }
    keep_order();
}

template <typename T, int V, int L, int W, bool GATED, bool MASKED>
__global__ void __launch_bounds__(W == 1 ? SCAN_BLOCK : 64 * W, 4) scan_forward_kernel(ScanArgs g) {
    __shared__ Exchange<V, W> ex[W == 1 ? 1 : 2];
    const Place place = scan_place<V, W>(g);
    const int lane = threadIdx.x & 63;
    const int wave = W == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const long t_begin = (long)place.seg * g.seg;
    const long t_end = t_begin + g.seg < g.T ? t_begin + g.seg : g.T;
    const long at = (place.b0 + place.b) * g.H + place.h, plane = g.B * g.H;
    const long at0 = place.b0 * g.H;                 // at = at0 + place.b H + place.h
    const unsigned inside = place.b * (unsigned)g.H + place.h;
    float c[V];
    segment_start<V, W, false>(g, (int)place.seg, wave, at, g.h0, &ex[0], c);
    int turn = 1;                                    // (segment_start has used ex[0])
    const auto chunk = [&](auto full, long t0, int n) {
        constexpr bool FULL = decltype(full)::value, SELECT = MASKED || !FULL;
        Pack<T, V> x[L], z[L], o[L], none[L];
        bool live[L];
        load_steps<T, V, L, GATED, MASKED, FULL, true, true, false>(g, place, t0, t_end, n, x, z, o, none, live);
        float f[L][V], add[L][V];
        Map<V> own = identity<V>();
#pragma unroll
        for (int i = 0; i < L; ++i) {
            const Pack<T, V> xi = now(x[i]), zi = now(z[i]);
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const Gate k = sigmoid_pair(widen(zi.v[v]));
                f[i][v] = k.f;
                add[i][v] = k.keep * widen(xi.v[v]);
                if constexpr (SELECT) {
                    f[i][v] = live[i] ? f[i][v] : 1.f;
                    add[i][v] = live[i] ? add[i][v] : 0.f;
                }
                if constexpr (W > 1) {
                    own.P[v] *= f[i][v];
                    own.S[v] = f[i][v] * own.S[v] + add[i][v];
                }
            }
            keep_order();
        }
        float s[V];
        if constexpr (W > 1) {
            Exchange<V, W>& e = ex[turn];
            e.m[wave][lane] = own;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < W; ++w) {
                if (w == wave) {
#pragma unroll
                    for (int v = 0; v < V; ++v) s[v] = c[v];
                }
                const Map<V> k = e.m[w][lane];
#pragma unroll
                for (int v = 0; v < V; ++v) c[v] = k.P[v] * c[v] + k.S[v];
            }
        } else {
#pragma unroll
            for (int v = 0; v < V; ++v) s[v] = c[v];
        }
        if (g.states && (FULL || n > 0)) {
            Pack<float, V> q;
#pragma unroll
            for (int v = 0; v < V; ++v) q.v[v] = s[v];
            store_off<float, V>(g.states + (t0 / L) * plane + at0, inside * 4u, q);
        }
        T* w = static_cast<T*>(g.y) + t0 * plane + at0;
#pragma unroll
        for (int i = 0; i < L; ++i) {
            Pack<T, V> out, oi;
            if constexpr (GATED) oi = now(o[i]);
#pragma unroll
            for (int v = 0; v < V; ++v) {
                s[v] = f[i][v] * s[v] + add[i][v];
                float r = s[v];
                if constexpr (GATED) {
                    const float ov = widen(oi.v[v]);
                    r = r * (ov * sigmoid(ov));
                }
                if constexpr (MASKED) r = live[i] ? r : 0.f;
                out.v[v] = narrow<T>(r);
            }
            if (FULL || i < n) store_off<T, V>(w, inside * (unsigned)sizeof(T), out);
            w = move_on(w, plane);
            keep_order();
        }
        if constexpr (W == 1) {
#pragma unroll
            for (int v = 0; v < V; ++v) c[v] = s[v];
        } else {
            // the sequence's last state comes from the wavefront that ran its last step
            if (g.last && n > 0 && t0 + n == g.T) {
#pragma unroll
                for (int v = 0; v < V; ++v) g.last[at + v] = s[v];
            }
        }
    };
    // (which form a round of chunks takes is the same for the whole workgroup: it holds a barrier)
    for (long base = t_begin; base < t_end; base += L * W, turn ^= 1) {
        const long t0 = base + L * wave;
        if (base + L * W <= t_end) {
            chunk(std::true_type{}, t0, L);
        } else {
            chunk(std::false_type{}, t0, t_end - t0 >= L ? L : (t_end > t0 ? (int)(t_end - t0) : 0));
        }
    }
    if (W == 1 && g.last && t_end == g.T) {
#pragma unroll
        for (int v = 0; v < V; ++v) g.last[at + v] = c[v];
    }
}

// A segment's map, for the state (forward) or its gradient (BACKWARD): the workgroup's wavefronts
// compose a stretch each, the first joins them.
template <typename T, int V, int L, int W, bool GATED, bool MASKED, bool BACKWARD>
__global__ void __launch_bounds__(64 * W) scan_compose_kernel(ScanArgs g) {
    __shared__ Exchange<V, W> ex;
    const Place place = scan_place<V, W>(g);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const long t_first = (long)place.seg * g.seg;
    const long t_last = t_first + g.seg < g.T ? t_first + g.seg : g.T;
    const long stretch = g.seg / W;                  // (a multiple of L)
    const long t_begin = t_first + wave * stretch < t_last ? t_first + wave * stretch : t_last;
    const long t_end = t_begin + stretch < t_last ? t_begin + stretch : t_last;
    Map<V> own = identity<V>();
    const auto chunk = [&](auto full, long t0, int n) {
        constexpr bool FULL = decltype(full)::value, SELECT = MASKED || !FULL;
        Pack<T, V> x[L], z[L], o[L], d[L];
        bool live[L];
        load_steps<T, V, L, GATED, MASKED, FULL, !BACKWARD, BACKWARD, BACKWARD>(g, place, t0, t_end, n, x, z, o, d,
                                                                               live);
#pragma unroll
        for (int j = 0; j < L; ++j) {
            const int i = BACKWARD ? L - 1 - j : j;
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const Gate k = sigmoid_pair(widen(z[i].v[v]));
                float P, S;
                if constexpr (BACKWARD) {            // carry -> f (dy silu(o) + carry)
                    float dc = widen(d[i].v[v]);
                    if constexpr (GATED) {
                        const float ov = widen(o[i].v[v]);
                        dc = dc * (ov * sigmoid(ov));
                    }
                    P = own.P[v] * k.f, S = k.f * (dc + own.S[v]);
                } else {
                    P = own.P[v] * k.f, S = k.f * own.S[v] + k.keep * widen(x[i].v[v]);
                }
                own.P[v] = !SELECT || live[i] ? P : own.P[v];
                own.S[v] = !SELECT || live[i] ? S : own.S[v];
            }
            keep_order();
        }
    };
    const long chunks = (t_end - t_begin + L - 1) / L;
    for (long k = 0; k < chunks; ++k) {
        const long t0 = t_begin + (BACKWARD ? chunks - 1 - k : k) * L;
        if (t_end - t0 >= L) {
            chunk(std::true_type{}, t0, L);
        } else {
            chunk(std::false_type{}, t0, (int)(t_end - t0));
        }
    }
    ex.m[wave][lane] = own;
    __syncthreads();
    if (wave != 0) return;
    Map<V> all = ex.m[BACKWARD ? W - 1 : 0][lane];
#pragma unroll
    for (int w = 1; w < W; ++w) all = then<V>(all, ex.m[BACKWARD ? W - 1 - w : w][lane]);
    const long at = (place.b0 + place.b) * g.H + place.h, plane = g.B * g.H;
#pragma unroll
    for (int v = 0; v < V; ++v) g.compose[place.seg * plane + at + v] = make_float2(all.P[v], all.S[v]);
}

// Adjoint.  carry = f_{t+1} G_{t+1}, the gradient that reaches c_t from later steps:
//   G_t = dy_t silu(o_t) + carry, dx = (1-f) G, dforget = f (1-f) (c_{t-1} - x) G, do = dy c silu'(o)
// Everything but G is known once a chunk's states have been run again: do goes out at once, and a
// step keeps f, dy silu(o), 1 - f and f (1-f) (c_{t-1} - x) until the gradient from behind is there.
template <typename T, int V, int L, int W, bool GATED, bool MASKED>
__global__ void __launch_bounds__(W == 1 ? SCAN_BLOCK : 64 * W, 4) scan_backward_kernel(ScanArgs g) {
    __shared__ Exchange<V, W> ex[W == 1 ? 1 : 2];
    const Place place = scan_place<V, W>(g);
    const int lane = threadIdx.x & 63;
    const int wave = W == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const long t_begin = (long)place.seg * g.seg;
    const long t_end = t_begin + g.seg < g.T ? t_begin + g.seg : g.T;
    const long at = (place.b0 + place.b) * g.H + place.h, plane = g.B * g.H;
    const long at0 = place.b0 * g.H;
    const unsigned inside = place.b * (unsigned)g.H + place.h;
    const long row = (GATED ? 3 : 2) * g.H;
    const unsigned du_inside = (place.b * (unsigned)row + place.h) * (unsigned)sizeof(T);
    float carry[V];
    segment_start<V, W, true>(g, (int)place.seg, wave, at, g.dlast, &ex[0], carry);
    int turn = 1;
    const auto chunk = [&](auto full, long t0, int n) {
        constexpr bool FULL = decltype(full)::value, SELECT = MASKED || !FULL;
        Pack<T, V> x[L], z[L], o[L], d[L];
        bool live[L];
        float c[V];
        const Pack<float, V> first =
            load_off<float, V>(g.states + ((FULL || n > 0 ? t0 : t_end - 1) / L) * plane + at0, inside * 4u);
#pragma unroll
        for (int v = 0; v < V; ++v) c[v] = first.v[v];
        load_steps<T, V, L, GATED, MASKED, FULL, true, true, true>(g, place, t0, t_end, n, x, z, o, d, live);
        float f[L][V], keep[L][V], slope[L][V], into[L][V];
        const long du_t = g.B * row;
        T* w = static_cast<T*>(g.du) + t0 * du_t + place.b0 * row;
#pragma unroll
        for (int i = 0; i < L; ++i) {
            Pack<T, V> dg, oi;
            const Pack<T, V> xi = now(x[i]), zi = now(z[i]), di = now(d[i]);
            if constexpr (GATED) oi = now(o[i]);
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const Gate k = sigmoid_pair(widen(zi.v[v]));
                const float xv = widen(xi.v[v]);
                const float next = k.f * c[v] + k.keep * xv;
                float dc = widen(di.v[v]), go = 0.f;
                if constexpr (GATED) {
                    const float ov = widen(oi.v[v]);
                    const Gate r = sigmoid_pair(ov);
                    go = dc * next * (r.f * (1.f + ov * r.keep));
                    dc = dc * (ov * r.f);
                }
                f[i][v] = k.f;
                keep[i][v] = k.keep;
                slope[i][v] = k.f * k.keep * (c[v] - xv);
                into[i][v] = dc;
                if constexpr (SELECT) {
                    f[i][v] = live[i] ? k.f : 1.f;
                    keep[i][v] = live[i] ? k.keep : 0.f;
                    slope[i][v] = live[i] ? slope[i][v] : 0.f;
                    into[i][v] = live[i] ? dc : 0.f;
                    go = live[i] ? go : 0.f;
                    c[v] = live[i] ? next : c[v];
                } else {
                    c[v] = next;
                }
                dg.v[v] = narrow<T>(go);
                settle(f[i][v]), settle(keep[i][v]), settle(slope[i][v]), settle(into[i][v]);
            }
            if constexpr (GATED) {
                if (FULL || i < n) store_off<T, V>(w + 2 * g.H, du_inside, dg);
            }
            w = move_on(w, du_t);
            keep_order();
        }
        float a[V];
        if constexpr (W > 1) {
            Map<V> own = identity<V>();
#pragma unroll
            for (int i = L - 1; i >= 0; --i) {
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    own.P[v] *= f[i][v];
                    own.S[v] = f[i][v] * (into[i][v] + own.S[v]);
                }
                keep_order();
            }
            Exchange<V, W>& e = ex[turn];
            e.m[wave][lane] = own;
            __syncthreads();
#pragma unroll
            for (int k = W - 1; k >= 0; --k) {
                if (k == wave) {
#pragma unroll
                    for (int v = 0; v < V; ++v) a[v] = carry[v];
                }
                const Map<V> r = e.m[k][lane];
#pragma unroll
                for (int v = 0; v < V; ++v) carry[v] = r.P[v] * carry[v] + r.S[v];
            }
        } else {
#pragma unroll
            for (int v = 0; v < V; ++v) a[v] = carry[v];
        }
#pragma unroll
        for (int i = L - 1; i >= 0; --i) {
            w = move_on(w, -du_t);
            Pack<T, V> dx, dz;
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const float G = into[i][v] + a[v];
                dx.v[v] = narrow<T>(keep[i][v] * G);
                dz.v[v] = narrow<T>(slope[i][v] * G);
                a[v] = f[i][v] * G;
            }
            if (FULL || i < n) {
                store_off<T, V>(w, du_inside, dx);
                store_off<T, V>(w + g.H, du_inside, dz);
            }
            keep_order();
        }
        if constexpr (W == 1) {
#pragma unroll
            for (int v = 0; v < V; ++v) carry[v] = a[v];
        } else {
            if (g.dh0 && t0 == 0) {
#pragma unroll
                for (int v = 0; v < V; ++v) g.dh0[at + v] = a[v];
            }
        }
    };
    constexpr long SPAN = L * W;
    for (long base = t_begin + ((t_end - t_begin - 1) / SPAN) * SPAN; base >= t_begin; base -= SPAN, turn ^= 1) {
        const long t0 = base + L * wave;
        if (base + SPAN <= t_end) {
            chunk(std::true_type{}, t0, L);
        } else {
            chunk(std::false_type{}, t0, t_end - t0 >= L ? L : (t_end > t0 ? (int)(t_end - t0) : 0));
        }
    }
    if (W == 1 && g.dh0 && t_begin == 0) {
#pragma unroll
        for (int v = 0; v < V; ++v) g.dh0[at + v] = carry[v];
    }
}

// One step with the state updated in place: a stream over u, state and y (262144 sequences of 128 channels,
// bfloat16: 99 us, 5.4 TB/s).  Here a channel has
// exactly one lane (the state is read and written), so an odd end goes element by element.
template <typename T, int V, bool GATED>
__global__ void __launch_bounds__(SCAN_BLOCK)
scan_step_kernel(long B, long H, const T* __restrict__ u, long u_b, const uint8_t* __restrict__ mask,
                 long mask_b, float* __restrict__ state, T* __restrict__ y, long groups) {
    const long idx = (long)blockIdx.x * SCAN_BLOCK + threadIdx.x;
    if (idx >= B * groups) return;
    const long b = idx / groups, h = (idx - b * groups) * V;
    const T* p = u + b * u_b + h;
    float* s = state + b * H + h;
    T* out = y + b * H + h;
    const bool live = !mask || mask[b * mask_b] != 0;
    const auto one = [&](float x, float z, float o, float c, float& r) {
        const Gate k = sigmoid_pair(z);
        const float next = k.f * c + k.keep * x;
        r = next;
        if constexpr (GATED) r = next * (o * sigmoid_pair(o).f);
        r = live ? r : 0.f;
        return live ? next : c;
    };
    if (h + V <= H) {
        const Pack<T, V> x = load_pack<T, V>(p), z = load_pack<T, V>(p + H);
        Pack<T, V> o = x, r;
        if constexpr (GATED) o = load_pack<T, V>(p + 2 * H);
        Pack<float, V> c = load_pack<float, V>(s);
#pragma unroll
        for (int v = 0; v < V; ++v) {
            float w;
            c.v[v] = one(widen(x.v[v]), widen(z.v[v]), widen(o.v[v]), c.v[v], w);
            r.v[v] = narrow<T>(w);
        }
        store_pack<float, V>(s, c);
        store_pack<T, V>(out, r);
        return;
    }
    for (int v = 0; h + v < H; ++v) {
        float w;
        s[v] = one(widen(p[v]), widen(p[H + v]), GATED ? widen(p[2 * H + v]) : 0.f, s[v], w);
        out[v] = narrow<T>(w);
    }
}

// How the work is laid out, from the sizes alone (times: forward / backward, H = 128, us).
// - 1024 wavefronts of channels or more (a SIMD has one): each walks over its sequence alone.  At
//   1024 the two forms meet (float, T = 1000: 208/329 alone, 217/368 with four).
// - Fewer: four wavefronts share the time axis, as long as there is more than one chunk.  At 256
//   wavefronts and T = 1000: 57/90 against 135/210 alone; T = 20, 64 wavefronts: 4.4/6.8 against
//   8.2/7.4.  (Eight: 5.1/8.7 there, and no faster on long sequences.)
// - Fewer than 600 (float; 850 of a 16-bit type, whose wavefronts have half the bytes under way) with that,
//   and six rounds of a workgroup or more: the sequence is cut into segments as well, up to 128, of at
//   least two rounds each, and u is read twice.  T = 2000, forward and backward: float, 480 wavefronts 196
//   against 235 uncut, 800 340 against 258; bfloat16, 600 250 against 342, 1000 460 against 382.  Float,
//   T = 300, 480 wavefronts: 41 against 34.  32768 steps of 520 half channels take 17 us to compose and 26 to
//   run (one wavefront per segment and a launch for the start states: 47 + 10 + 54).
// Asking for the next round's steps before a round is worked on was slower (21 + 30 there, 1000 masked steps
// 235 against 128): the barrier waits for what has been asked for.
struct Plan {
    int V, L, W, segs;
    long seg;                                        // steps per segment
};
static Plan scan_plan(long T, long B, long H, int dtype) {
    Plan p;
    p.V = dtype != KVAE_F32 && H >= 2 ? 2 : 1;
    p.L = KVAE_SCAN_CHUNK(dtype);
    const long waves = (B * ((H + p.V - 1) / p.V) + 63) / 64;
    p.W = waves < 1024 && T > p.L ? TOGETHER : 1;
    p.segs = 1;
    p.seg = T;
    const long round = (long)p.L * p.W;
    if (p.W > 1 && waves * p.W < (dtype == KVAE_F32 ? 600 : 850) && T >= 6 * round) {
        long want = (8192 + waves * p.W - 1) / (waves * p.W);
        if (want > MOST_SEGMENTS) want = MOST_SEGMENTS;
        if (want > T / (2 * round)) want = T / (2 * round);
        const long each = ((T + want - 1) / want + round - 1) / round * round;
        p.segs = (int)((T + each - 1) / each);
        p.seg = each;
    }
    return p;
}

// a launch has fewer than 2^32 threads, and a channel has up to four (wavefronts that share the time axis
// only do so where there are few channels)
constexpr long MOST_CHANNELS = (1L << 32) - SCAN_BLOCK;

static int check_scan(const kvae_gated_scan* d) {
    if (!d || d->T < 1 || d->B < 1 || d->H < 1 || !d->u) return KVAE_E_BADARG;
    if (d->dtype != KVAE_F32 && d->dtype != KVAE_BF16 && d->dtype != KVAE_F16)
        return KVAE_E_UNSUPPORTED;
    if (d->B > MOST_CHANNELS / d->H) return KVAE_E_TOOLARGE;
    // lane offsets are 32 bits: the sequences of a workgroup (up to 256 lanes of one channel) must
    // lie within 2^31 bytes of each other
    if (d->u_stride_b < 0 || d->dy_stride_b < 0 || d->mask_stride_b < 0) return KVAE_E_BADARG;
    long sequences = 2L * SCAN_BLOCK / d->H + 2;     // (a lane owns at most two channels)
    if (sequences > d->B) sequences = d->B;
    const long size = d->dtype == KVAE_F32 ? 4 : 2, most = (1L << 31) / size;
    const long stride = d->u_stride_b > d->dy_stride_b ? d->u_stride_b : d->dy_stride_b;
    if (3 * d->H > most / (sequences + 1)) return KVAE_E_TOOLARGE;
    if (sequences > 1 && (stride > (most - 3 * d->H) / (sequences - 1) ||
                          d->mask_stride_b > (1L << 31) / (sequences - 1)))
        return KVAE_E_TOOLARGE;
    return KVAE_OK;
}

static ScanArgs scan_args(const kvae_gated_scan* d) {
    ScanArgs g{};
    g.T = d->T, g.B = d->B, g.H = d->H;
    g.u = d->u, g.u_t = d->u_stride_t, g.u_b = d->u_stride_b;
    g.mask = static_cast<const uint8_t*>(d->mask);
    g.mask_t = d->mask_stride_t, g.mask_b = d->mask_stride_b;
    g.h0 = static_cast<const float*>(d->h0);
    g.y = d->y, g.last = static_cast<float*>(d->last), g.states = static_cast<float*>(d->states);
    g.dy = d->dy, g.dy_t = d->dy_stride_t, g.dy_b = d->dy_stride_b;
    g.dlast = static_cast<const float*>(d->dlast);
    g.du = d->du, g.dh0 = static_cast<float*>(d->dh0);
    return g;
}

template <typename T, int V, int W, bool BACKWARD, bool GATED, bool MASKED>
static void launch_scan(ScanArgs g, hipStream_t stream) {
    constexpr int L = KVAE_SCAN_CHUNK(sizeof(T) == 4 ? KVAE_F32 : KVAE_BF16);
    constexpr int BLOCK = W == 1 ? SCAN_BLOCK : 64 * W, LANES = W == 1 ? SCAN_BLOCK : 64;
    g.groups = (g.H + V - 1) / V;
    const dim3 grid((unsigned)((g.B * g.groups + LANES - 1) / LANES), (unsigned)g.segs);
    if constexpr (W > 1) {
        if (g.segs > 1)
            scan_compose_kernel<T, V, L, W, BACKWARD && GATED, MASKED, BACKWARD><<<grid, BLOCK, 0, stream>>>(g);
    }
    if constexpr (BACKWARD)
        scan_backward_kernel<T, V, L, W, GATED, MASKED><<<grid, BLOCK, 0, stream>>>(g);
    else
        scan_forward_kernel<T, V, L, W, GATED, MASKED><<<grid, BLOCK, 0, stream>>>(g);
}

// f(std::bool_constant<x>{})
template <typename F>
static void with_bool(bool x, F&& f) {
    x ? f(std::true_type{}) : f(std::false_type{});
}

template <bool BACKWARD>
static int run_scan(const kvae_gated_scan* d, void* workspace, size_t bytes, hipStream_t stream) {
    const size_t need = kvae_gated_scan_workspace_bytes(d->T, d->B, d->H, d->dtype);
    if (bytes < need || (need && !workspace)) return KVAE_E_WORKSPACE;
    const Plan plan = scan_plan(d->T, d->B, d->H, d->dtype);
    ScanArgs g = scan_args(d);
    g.seg = plan.seg, g.segs = plan.segs;
    g.compose = static_cast<float2*>(workspace);
    return for_element_type(d->dtype, [&](auto e) {
        using T = decltype(e);
        with_bool(d->gated, [&](auto gated) {
            with_bool(g.mask != nullptr, [&](auto masked) {
                with_bool(plan.W > 1, [&](auto together) {
                    constexpr int W = decltype(together)::value ? TOGETHER : 1;
                    constexpr bool GATED = decltype(gated)::value, MASKED = decltype(masked)::value;
                    if constexpr (sizeof(T) == 2) {
                        if (plan.V == 2) return launch_scan<T, 2, W, BACKWARD, GATED, MASKED>(g, stream);
                    }
                    launch_scan<T, 1, W, BACKWARD, GATED, MASKED>(g, stream);
                });
            });
        });
        return hipGetLastError() == hipSuccess ? KVAE_OK : KVAE_E_LAUNCH;
    });
}

}  // namespace kvae

using namespace kvae;

extern "C" size_t kvae_gated_scan_workspace_bytes(int64_t T, int64_t B, int64_t H, int dtype) {
    if (T < 1 || B < 1 || H < 1) return 0;
    const Plan p = scan_plan(T, B, H, dtype);
    return p.segs < 2 ? 0 : (size_t)p.segs * B * H * sizeof(float2);
}

extern "C" int kvae_gated_scan_forward(const kvae_gated_scan* d, void* workspace,
                                       size_t workspace_bytes, void* stream) {
    const int rc = check_scan(d);
    if (rc != KVAE_OK) return rc;
    if (!d->y) return KVAE_E_BADARG;
    return run_scan<false>(d, workspace, workspace_bytes, static_cast<hipStream_t>(stream));
}

extern "C" int kvae_gated_scan_backward(const kvae_gated_scan* d, void* workspace,
                                        size_t workspace_bytes, void* stream) {
    const int rc = check_scan(d);
    if (rc != KVAE_OK) return rc;
    if (!d->states || !d->dy || !d->du) return KVAE_E_BADARG;
    return run_scan<true>(d, workspace, workspace_bytes, static_cast<hipStream_t>(stream));
}

extern "C" int kvae_gated_scan_step(int64_t B, int64_t H, int dtype, int gated, const void* u,
                                    int64_t u_stride_b, const void* mask, int64_t mask_stride_b,
                                    void* state, void* y, void* stream) {
    if (B < 1 || H < 1 || !u || !state || !y) return KVAE_E_BADARG;
    if (B > MOST_CHANNELS / H) return KVAE_E_TOOLARGE;
    return for_element_type(dtype, [&](auto e) {
        using T = decltype(e);
        constexpr int V = 4;
        const long groups = (H + V - 1) / V;
        const dim3 grid((unsigned)((B * groups + SCAN_BLOCK - 1) / SCAN_BLOCK));
        const hipStream_t s = static_cast<hipStream_t>(stream);
        const auto go = [&](auto g) {
            scan_step_kernel<T, V, decltype(g)::value><<<grid, SCAN_BLOCK, 0, s>>>(
                B, H, static_cast<const T*>(u), u_stride_b, static_cast<const uint8_t*>(mask),
                mask_stride_b, static_cast<float*>(state), static_cast<T*>(y), groups);
        };
        gated ? go(std::true_type{}) : go(std::false_type{});
        return hipGetLastError() == hipSuccess ? KVAE_OK : KVAE_E_LAUNCH;
    });
}
