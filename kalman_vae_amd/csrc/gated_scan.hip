// Gated linear recurrence over a sequence on gfx950, forward, backward and one step.
//
//   f = sigmoid(forget), c_t = f_t c_{t-1} + (1 - f_t) x_t, y_t = c_t silu(o_t) (or c_t)
//
// element-wise over (B,H): unlike the LSTM's recurrence there is no matrix product between steps,
// so the work is a stream over memory: the forward pass reads u = [x | forget | o] and writes y,
// the backward pass reads u and dy and writes du.
//
// Mapping: a lane owns one channel (float) or two neighbouring ones (16-bit types) of one
// sequence, so that a wavefront moves 256 contiguous bytes per tensor and step, and walks its
// steps in chunks of CHUNK: the loads of a whole chunk are issued before the first is used.
// The state stays in registers in float, whatever the element type.
//
// The backward pass does not read y (which is rounded to the element type, and gated): the
// forward pass leaves the float state before every chunk, and the backward pass runs a chunk's
// recurrence again from there in registers, on the x and forget it has to read anyway.
//
// When B*H lanes do not fill the card, the time axis is cut into segments of whole chunks: one
// launch composes each segment's steps to c_out = P c_in + S, a second composes the segments, and
// the main kernel starts every segment from its state.
#include "narrow_types.h"

#include "device_info.h"

namespace kvae {

constexpr int CHUNK = KVAE_SCAN_CHUNK;   // steps whose loads are in flight together
constexpr int SCAN_BLOCK = 256;

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
    long seg;                    // steps per segment, a multiple of CHUNK
    long segs;
    float2* compose;             // (segs, B, H): P and S of each segment
    float* carry;                // (segs, B, H): state a segment starts from
};

struct Gate {
    float f, keep;               // sigmoid(z), 1 - sigmoid(z), both without cancellation
};
__device__ __forceinline__ Gate sigmoid_pair(float z) {
    const float e = __expf(-fabsf(z));
    const float big = __builtin_amdgcn_rcpf(1.f + e);
    const float small = e * big;
    return z >= 0.f ? Gate{big, small} : (z < 0.f ? Gate{small, big} : Gate{z, z});
}

// Lane -> (sequence, first channel).  The last lane of a sequence is moved back so that its V
// channels end at H: a channel that two lanes own gets the same values from both.
template <int V>
__device__ __forceinline__ bool scan_lane(const ScanArgs& g, long& b, long& h) {
    const long c = (long)blockIdx.x * SCAN_BLOCK + threadIdx.x;
    if (c >= g.B * g.groups) return false;
    b = c / g.groups;
    h = (c - b * g.groups) * V;
    if (h > g.H - V) h = g.H - V;
    return true;
}

template <typename T, int V, bool GATED, bool MASKED>
__global__ void __launch_bounds__(SCAN_BLOCK) scan_forward_kernel(ScanArgs g) {
    long b, h;
    if (!scan_lane<V>(g, b, h)) return;
    const long t_begin = (long)blockIdx.y * g.seg;
    const long t_end = t_begin + g.seg < g.T ? t_begin + g.seg : g.T;
    const long at = b * g.H + h, plane = g.B * g.H;
    float c[V];
#pragma unroll
    for (int v = 0; v < V; ++v)
        c[v] = g.carry ? g.carry[blockIdx.y * plane + at + v] : (g.h0 ? g.h0[at + v] : 0.f);
    const T* u = static_cast<const T*>(g.u) + b * g.u_b + h;
    T* y = static_cast<T*>(g.y) + at;
    for (long t0 = t_begin; t0 < t_end; t0 += CHUNK) {
        const int n = t_end - t0 < CHUNK ? (int)(t_end - t0) : CHUNK;
        if (g.states) {
            float* s = g.states + (t0 / CHUNK) * plane + at;
#pragma unroll
            for (int v = 0; v < V; ++v) s[v] = c[v];
        }
        Pack<T, V> x[CHUNK], z[CHUNK], o[CHUNK];
        bool live[CHUNK];
        const T* p = u + t0 * g.u_t;
        T* w = y + t0 * plane;
        const uint8_t* m = MASKED ? g.mask + t0 * g.mask_t + b * g.mask_b : nullptr;
#pragma unroll
        for (int i = 0; i < CHUNK; ++i) {
            if (i < n) {
                x[i] = load_pack<T, V>(p);
                z[i] = load_pack<T, V>(p + g.H);
                if constexpr (GATED) o[i] = load_pack<T, V>(p + 2 * g.H);
                if constexpr (MASKED) live[i] = *m != 0, m += g.mask_t;
                p += g.u_t;
            }
        }
#pragma unroll
        for (int i = 0; i < CHUNK; ++i) {
            if (i < n) {
                Pack<T, V> out;
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    const Gate k = sigmoid_pair(widen(z[i].v[v]));
                    const float next = k.f * c[v] + k.keep * widen(x[i].v[v]);
                    float r = next;
                    if constexpr (GATED) {
                        const float ov = widen(o[i].v[v]);
                        r = next * (ov * sigmoid_pair(ov).f);
                    }
                    if constexpr (MASKED) {
                        c[v] = live[i] ? next : c[v];
                        r = live[i] ? r : 0.f;
                    } else {
                        c[v] = next;
                    }
                    out.v[v] = narrow<T>(r);
                }
                store_pack<T, V>(w, out);
                w += plane;
            }
        }
    }
    if (g.last && t_end == g.T) {
#pragma unroll
        for (int v = 0; v < V; ++v) g.last[at + v] = c[v];
    }
}

// A segment's composition for the forward pass: c_out = P c_in + S.
template <typename T, int V, bool MASKED>
__global__ void __launch_bounds__(SCAN_BLOCK) scan_forward_compose_kernel(ScanArgs g) {
    long b, h;
    if (!scan_lane<V>(g, b, h)) return;
    const long t_begin = (long)blockIdx.y * g.seg;
    const long t_end = t_begin + g.seg < g.T ? t_begin + g.seg : g.T;
    const long at = b * g.H + h, plane = g.B * g.H;
    float P[V], S[V];
#pragma unroll
    for (int v = 0; v < V; ++v) P[v] = 1.f, S[v] = 0.f;
    const T* u = static_cast<const T*>(g.u) + b * g.u_b + h;
    for (long t0 = t_begin; t0 < t_end; t0 += CHUNK) {
        const int n = t_end - t0 < CHUNK ? (int)(t_end - t0) : CHUNK;
        Pack<T, V> x[CHUNK], z[CHUNK];
        bool live[CHUNK];
        const T* p = u + t0 * g.u_t;
        const uint8_t* m = MASKED ? g.mask + t0 * g.mask_t + b * g.mask_b : nullptr;
#pragma unroll
        for (int i = 0; i < CHUNK; ++i) {
            if (i < n) {
                x[i] = load_pack<T, V>(p);
                z[i] = load_pack<T, V>(p + g.H);
                if constexpr (MASKED) live[i] = *m != 0, m += g.mask_t;
                p += g.u_t;
            }
        }
#pragma unroll
        for (int i = 0; i < CHUNK; ++i) {
            if (i < n) {
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    const Gate k = sigmoid_pair(widen(z[i].v[v]));
                    const float p = P[v] * k.f, s = k.f * S[v] + k.keep * widen(x[i].v[v]);
                    if (!MASKED || live[i]) P[v] = p, S[v] = s;
                }
            }
        }
    }
#pragma unroll
    for (int v = 0; v < V; ++v) g.compose[blockIdx.y * plane + at + v] = make_float2(P[v], S[v]);
}

// Adjoint.  carry = f_{t+1} G_{t+1}, the gradient that reaches c_t from later steps:
//   G_t = dy_t silu(o_t) + carry, dx = (1-f) G, dforget = f (1-f) (c_{t-1} - x) G, do = dy c silu'(o)
template <typename T, int V, bool GATED, bool MASKED>
__global__ void __launch_bounds__(SCAN_BLOCK) scan_backward_kernel(ScanArgs g) {
    long b, h;
    if (!scan_lane<V>(g, b, h)) return;
    const long t_begin = (long)blockIdx.y * g.seg;
    const long t_end = t_begin + g.seg < g.T ? t_begin + g.seg : g.T;
    const long at = b * g.H + h, plane = g.B * g.H;
    const long row = (GATED ? 3 : 2) * g.H;
    float carry[V];
#pragma unroll
    for (int v = 0; v < V; ++v)
        carry[v] = g.carry ? g.carry[blockIdx.y * plane + at + v] : (g.dlast ? g.dlast[at + v] : 0.f);
    const T* u = static_cast<const T*>(g.u) + b * g.u_b + h;
    const T* dy = static_cast<const T*>(g.dy) + b * g.dy_b + h;
    T* du = static_cast<T*>(g.du) + b * row + h;
    for (long t0 = t_begin + ((t_end - t_begin - 1) / CHUNK) * CHUNK; t0 >= t_begin; t0 -= CHUNK) {
        const int n = t_end - t0 < CHUNK ? (int)(t_end - t0) : CHUNK;
        Pack<T, V> x[CHUNK], z[CHUNK], o[CHUNK], d[CHUNK];
        float c[CHUNK][V], last[V];
        bool live[CHUNK];
        const float* s = g.states + (t0 / CHUNK) * plane + at;
#pragma unroll
        for (int v = 0; v < V; ++v) last[v] = s[v];
        const T* p = u + t0 * g.u_t;
        const T* q = dy + t0 * g.dy_t;
        const uint8_t* m = MASKED ? g.mask + t0 * g.mask_t + b * g.mask_b : nullptr;
#pragma unroll
        for (int i = 0; i < CHUNK; ++i) {
            if (i < n) {
                x[i] = load_pack<T, V>(p);
                z[i] = load_pack<T, V>(p + g.H);
                if constexpr (GATED) o[i] = load_pack<T, V>(p + 2 * g.H);
                d[i] = load_pack<T, V>(q);
                q += g.dy_t;
                if constexpr (MASKED) live[i] = *m != 0, m += g.mask_t;
                p += g.u_t;
            }
        }
        // c[i]: the state BEFORE step t0 + i
#pragma unroll
        for (int i = 0; i < CHUNK; ++i) {
            if (i < n) {
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    c[i][v] = last[v];
                    const Gate k = sigmoid_pair(widen(z[i].v[v]));
                    const float next = k.f * last[v] + k.keep * widen(x[i].v[v]);
                    if (!MASKED || live[i]) last[v] = next;
                }
            }
        }
        T* w = du + (t0 + n - 1) * g.B * row;
#pragma unroll
        for (int i = CHUNK - 1; i >= 0; --i) {
            if (i < n) {
                Pack<T, V> dx, dz, dg;
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    const Gate k = sigmoid_pair(widen(z[i].v[v]));
                    const float xv = widen(x[i].v[v]), before = c[i][v];
                    float dc = widen(d[i].v[v]), go = 0.f;
                    if constexpr (GATED) {
                        const float ov = widen(o[i].v[v]);
                        const Gate q = sigmoid_pair(ov);
                        const float now = k.f * before + k.keep * xv;
                        go = dc * now * (q.f * (1.f + ov * q.keep));
                        dc = dc * (ov * q.f);
                    }
                    const float G = dc + carry[v];
                    float gx = k.keep * G, gz = k.f * k.keep * (before - xv) * G, on = k.f * G;
                    if constexpr (MASKED) {
                        gx = live[i] ? gx : 0.f;
                        gz = live[i] ? gz : 0.f;
                        go = live[i] ? go : 0.f;
                        on = live[i] ? on : carry[v];
                    }
                    carry[v] = on;
                    dx.v[v] = narrow<T>(gx);
                    dz.v[v] = narrow<T>(gz);
                    dg.v[v] = narrow<T>(go);
                }
                store_pack<T, V>(w, dx);
                store_pack<T, V>(w + g.H, dz);
                if constexpr (GATED) store_pack<T, V>(w + 2 * g.H, dg);
                w -= g.B * row;
            }
        }
    }
    if (g.dh0 && t_begin == 0) {
#pragma unroll
        for (int v = 0; v < V; ++v) g.dh0[at + v] = carry[v];
    }
}

// A segment's composition for the backward pass: carry_out = P carry_in + S.
template <typename T, int V, bool GATED, bool MASKED>
__global__ void __launch_bounds__(SCAN_BLOCK) scan_backward_compose_kernel(ScanArgs g) {
    long b, h;
    if (!scan_lane<V>(g, b, h)) return;
    const long t_begin = (long)blockIdx.y * g.seg;
    const long t_end = t_begin + g.seg < g.T ? t_begin + g.seg : g.T;
    const long at = b * g.H + h, plane = g.B * g.H;
    float P[V], S[V];
#pragma unroll
    for (int v = 0; v < V; ++v) P[v] = 1.f, S[v] = 0.f;
    const T* u = static_cast<const T*>(g.u) + b * g.u_b + h;
    const T* dy = static_cast<const T*>(g.dy) + b * g.dy_b + h;
    for (long t0 = t_begin + ((t_end - t_begin - 1) / CHUNK) * CHUNK; t0 >= t_begin; t0 -= CHUNK) {
        const int n = t_end - t0 < CHUNK ? (int)(t_end - t0) : CHUNK;
        Pack<T, V> z[CHUNK], o[CHUNK], d[CHUNK];
        bool live[CHUNK];
        const T* p = u + t0 * g.u_t;
        const T* q = dy + t0 * g.dy_t;
        const uint8_t* m = MASKED ? g.mask + t0 * g.mask_t + b * g.mask_b : nullptr;
#pragma unroll
        for (int i = 0; i < CHUNK; ++i) {
            if (i < n) {
                z[i] = load_pack<T, V>(p + g.H);
                if constexpr (GATED) o[i] = load_pack<T, V>(p + 2 * g.H);
                d[i] = load_pack<T, V>(q);
                q += g.dy_t;
                if constexpr (MASKED) live[i] = *m != 0, m += g.mask_t;
                p += g.u_t;
            }
        }
#pragma unroll
        for (int i = CHUNK - 1; i >= 0; --i) {
            if (i < n) {
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    const Gate k = sigmoid_pair(widen(z[i].v[v]));
                    float dc = widen(d[i].v[v]);
                    if constexpr (GATED) {
                        const float ov = widen(o[i].v[v]);
                        dc = dc * (ov * sigmoid_pair(ov).f);
                    }
                    const float p = k.f * P[v], s = k.f * (dc + S[v]);
                    if (!MASKED || live[i]) P[v] = p, S[v] = s;
                }
            }
        }
    }
#pragma unroll
    for (int v = 0; v < V; ++v) g.compose[blockIdx.y * plane + at + v] = make_float2(P[v], S[v]);
}

// State every segment starts from, in walking order (forward: first to last; backward: last to
// first).  One workgroup has 64 channels; its 16 wavefronts share the segments, compose their own
// stretch, exchange the compositions through LDS and walk the stretch again.
constexpr int CARRY_WAVES = 16;
template <bool REVERSE>
__global__ void __launch_bounds__(64 * CARRY_WAVES)
scan_carry_kernel(long channels, long segs, const float2* __restrict__ compose,
                  const float* __restrict__ init, float* __restrict__ carry) {
    __shared__ float2 stretch[CARRY_WAVES][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const long c = (long)blockIdx.x * 64 + lane;
    const bool in = c < channels;
    const long each = (segs + CARRY_WAVES - 1) / CARRY_WAVES;
    const long begin = wave * each < segs ? wave * each : segs;
    const long end = begin + each < segs ? begin + each : segs;
    float P = 1.f, S = 0.f;
    if (in) {
#pragma unroll 8
        for (long i = begin; i < end; ++i) {
            const float2 k = compose[(REVERSE ? segs - 1 - i : i) * channels + c];
            S = k.x * S + k.y;
            P *= k.x;
        }
    }
    stretch[wave][lane] = make_float2(P, S);
    __syncthreads();
    if (!in) return;
    float v = init ? init[c] : 0.f;
    for (int w = 0; w < wave; ++w) v = stretch[w][lane].x * v + stretch[w][lane].y;
#pragma unroll 8
    for (long i = begin; i < end; ++i) {
        const long s = REVERSE ? segs - 1 - i : i;
        const float2 k = compose[s * channels + c];
        carry[s * channels + c] = v;
        v = k.x * v + k.y;
    }
}

// One step with the state updated in place: a stream over u, state and y.  Here a channel has
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

// Channels per lane: two 16-bit ones or one float make a dword per lane and load.
template <typename T>
int scan_width(long H) {
    return sizeof(T) == 2 && H >= 2 ? 2 : 1;
}

// Segments of the time axis.  A wavefront keeps about 12 KB of loads in flight, so some 2000
// wavefronts (two per SIMD) cover the memory's latency; with fewer channels the time axis is cut,
// which reads part of the input twice: not before there are fewer than 512 wavefronts, and never
// into segments of under two chunks.
static long scan_segments(long T, long B, long H, int dtype) {
    const long width = dtype != KVAE_F32 && H >= 2 ? 2 : 1;
    const long waves = (B * ((H + width - 1) / width) + 63) / 64;
    if (waves >= 512) return 1;
    long segs = (2048 + waves - 1) / waves;
    const long most = T / (2 * CHUNK);
    if (segs > most) segs = most;
    if (segs > 32768) segs = 32768;
    return segs < 2 ? 1 : segs;
}
static long segment_steps(long T, long segs) {
    const long each = (T + segs - 1) / segs;
    return (each + CHUNK - 1) / CHUNK * CHUNK;
}

static int check_scan(const kvae_gated_scan* d) {
    if (!d || d->T < 1 || d->B < 1 || d->H < 1 || !d->u || (d->mask && d->mask_stride_b < 0))
        return KVAE_E_BADARG;
    if (d->dtype != KVAE_F32 && d->dtype != KVAE_BF16 && d->dtype != KVAE_F16)
        return KVAE_E_UNSUPPORTED;
    // a workgroup holds 256 lanes and blockIdx.x is 31 bits
    if (d->B > (1L << 38) / d->H) return KVAE_E_TOOLARGE;
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

static void cut_time(ScanArgs& g, int dtype, void* workspace) {
    const long segs = scan_segments(g.T, g.B, g.H, dtype);
    g.seg = segment_steps(g.T, segs);
    g.segs = (g.T + g.seg - 1) / g.seg;
    if (g.segs > 1) {
        g.compose = static_cast<float2*>(workspace);
        g.carry = reinterpret_cast<float*>(g.compose + g.segs * g.B * g.H);
    }
}

template <typename T, int V, bool BACKWARD, bool GATED, bool MASKED>
static void launch_scan(ScanArgs g, hipStream_t stream) {
    g.groups = (g.H + V - 1) / V;
    const dim3 grid((unsigned)((g.B * g.groups + SCAN_BLOCK - 1) / SCAN_BLOCK), (unsigned)g.segs);
    if (g.segs > 1) {
        const long channels = g.B * g.H;
        const dim3 cgrid((unsigned)((channels + 63) / 64));
        if constexpr (BACKWARD) {
            scan_backward_compose_kernel<T, V, GATED, MASKED><<<grid, SCAN_BLOCK, 0, stream>>>(g);
            scan_carry_kernel<true><<<cgrid, 64 * CARRY_WAVES, 0, stream>>>(channels, g.segs, g.compose,
                                                                          g.dlast, g.carry);
        } else {
            scan_forward_compose_kernel<T, V, MASKED><<<grid, SCAN_BLOCK, 0, stream>>>(g);
            scan_carry_kernel<false><<<cgrid, 64 * CARRY_WAVES, 0, stream>>>(channels, g.segs, g.compose,
                                                                           g.h0, g.carry);
        }
    }
    if constexpr (BACKWARD)
        scan_backward_kernel<T, V, GATED, MASKED><<<grid, SCAN_BLOCK, 0, stream>>>(g);
    else
        scan_forward_kernel<T, V, GATED, MASKED><<<grid, SCAN_BLOCK, 0, stream>>>(g);
}

template <bool BACKWARD>
static int run_scan(const kvae_gated_scan* d, void* workspace, size_t bytes, hipStream_t stream) {
    if (bytes < kvae_gated_scan_workspace_bytes(d->T, d->B, d->H, d->dtype)) return KVAE_E_WORKSPACE;
    return for_element_type(d->dtype, [&](auto e) {
        using T = decltype(e);
        ScanArgs g = scan_args(d);
        cut_time(g, d->dtype, workspace);
        const auto go = [&](auto width, auto gated, auto masked) {
            launch_scan<T, decltype(width)::value, BACKWARD, decltype(gated)::value,
                        decltype(masked)::value>(g, stream);
        };
        const auto with_width = [&](auto gated, auto masked) {
            if constexpr (sizeof(T) == 2) {
                if (scan_width<T>(g.H) == 2) return go(std::integral_constant<int, 2>{}, gated, masked);
            }
            go(std::integral_constant<int, 1>{}, gated, masked);
        };
        const auto with_mask = [&](auto gated) {
            g.mask ? with_width(gated, std::true_type{}) : with_width(gated, std::false_type{});
        };
        d->gated ? with_mask(std::true_type{}) : with_mask(std::false_type{});
        return hipGetLastError() == hipSuccess ? KVAE_OK : KVAE_E_LAUNCH;
    });
}

}  // namespace kvae

using namespace kvae;

extern "C" size_t kvae_gated_scan_workspace_bytes(int64_t T, int64_t B, int64_t H, int dtype) {
    if (T < 1 || B < 1 || H < 1) return 0;
    const long segs = scan_segments(T, B, H, dtype);
    if (segs < 2) return 0;
    return (size_t)segs * B * H * (sizeof(float2) + sizeof(float));
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
    if (B > (1L << 38) / H) return KVAE_E_TOOLARGE;
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
