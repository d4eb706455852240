// A residual block's norms, gate and residual scale (include/wc_b200.h,
// wc_block_norm), forward and backward.
//
// With hats for normalised values, r the reciprocal deviations and means over
// the width (the mean terms for LayerNorm only):
//   u = wp hhat + bp, y = c x + g u, n = wn yhat + bn
//   dY = dy + rn (wn dn - mean(wn dn) - yhat mean(wn dn yhat))
//   dx = c dY, dg = sum dY u, dU = g dY
//   dh = rp (wp dU - mean(wp dU) - hhat mean(wp dU hhat))
//   dwn = sum dn yhat, dbn = sum dn, dwp = sum dU hhat, dbp = sum dU
//
// Both directions are bound by the bytes of the [rows, width] matrices (two in
// and two out; four in and two out), each read and written once here. A unit is
// 8 columns of a row (16 bytes of a 16-bit type).
//   forward: a row in the registers of a part of a warp, or of a CTA; means and
//     deviations from the registers, in two passes.
//   backward, widths up to 256: a part of a warp a row, a unit a thread, which
//     also keeps that unit's sums over the rows (weights' and gate's).
//   backward, widths up to 4096: a CTA a row, a unit a thread, rows brought to
//     shared memory by bulk copies some rows ahead.
//   other widths, strides and addresses: kernels that read an element at a
//     time, and in the backward pass all inputs twice (rows, then columns).
#include <algorithm>

#include "colsum.cuh"
#include "kernels.h"
#include "umma.cuh"

namespace wctrain {

namespace {

constexpr int THREADS = 256;

struct Row {
    float pm, pr, nm, nr;
};

template <class T>
struct Args {
    wc_block_norm_args a;
    __device__ const T* gate(int64_t t) const {
        return a.gate ? static_cast<const T*>(a.gate) + t / a.rows_per_gate * a.width : nullptr;
    }
    __device__ float hhat(int64_t t, int64_t j, const Row& r) const {
        return (to_f(static_cast<const T*>(a.h)[t * a.ld_h + j]) - r.pm) * r.pr;
    }
    __device__ float u(float hh, int64_t j) const {
        return a.post_weight ? fmaf(hh, a.post_weight[j], a.post_bias ? a.post_bias[j] : 0.0f) : hh;
    }
    __device__ float y(int64_t t, int64_t j, float u, const T* gate) const {
        return a.residual_scale * to_f(static_cast<const T*>(a.x)[t * a.ld_x + j]) + (gate ? to_f(gate[j]) * u : u);
    }
};

template <class T>
__global__ void __launch_bounds__(THREADS) k_block_norm(Args<T> q) {
    __shared__ float s[32];
    const wc_block_norm_args& a = q.a;
    const int64_t D = a.width, blocks = (D + 31) / 32;
    const float inv = 1.0f / (float)D;
    for (int64_t t = blockIdx.x; t < a.rows; t += gridDim.x) {
        Row r{0.0f, 1.0f, 0.0f, 1.0f};
        const T* gate = q.gate(t);
        if (a.post_weight) {
            float v = 0.0f;
            if (a.kind == WC_NORM_LAYER) {
                for (int64_t j = threadIdx.x; j < D; j += THREADS) v += q.hhat(t, j, r);
                r.pm = cta_sum(v, s) * inv;
            }
            v = 0.0f;
            for (int64_t j = threadIdx.x; j < D; j += THREADS) v += q.hhat(t, j, r) * q.hhat(t, j, r);
            r.pr = rsqrtf(cta_sum(v, s) * inv + a.eps);
        }
        auto y_at = [&](int64_t j) { return q.y(t, j, q.u(q.hhat(t, j, r), j), gate); };
        if (a.pre_weight) {
            float v = 0.0f;
            if (a.kind == WC_NORM_LAYER) {
                for (int64_t j = threadIdx.x; j < D; j += THREADS) v += y_at(j);
                r.nm = cta_sum(v, s) * inv;
            }
            v = 0.0f;
            for (int64_t j = threadIdx.x; j < D; j += THREADS) v += (y_at(j) - r.nm) * (y_at(j) - r.nm);
            r.nr = rsqrtf(cta_sum(v, s) * inv + a.eps);
        }
        for (int64_t b = threadIdx.x / 32; b < blocks; b += THREADS / 32) {
            const int64_t j = b * 32 + (threadIdx.x & 31);
            float n = 0.0f;
            if (j < D) {
                const float y = y_at(j);
                static_cast<T*>(a.y)[t * a.ld_y + j] = from_f<T>(y);
                if (a.pre_weight) {
                    n = fmaf((y - r.nm) * r.nr, a.pre_weight[j], a.pre_bias ? a.pre_bias[j] : 0.0f);
                    if (a.n) static_cast<T*>(a.n)[t * a.ld_n + j] = from_f<T>(n);
                }
            }
            if (a.n_q) {
                const uint32_t code = act8_code(__uint_as_float(__reduce_max_sync(~0u, __float_as_uint(n) & 0x7fffffffu)));
                a.n_q[(t * blocks + b) * 32 + (threadIdx.x & 31)] =
                    code == 255 ? (int8_t)0 : (int8_t)__float2int_rn(n * act8_inverse(code));
                if ((threadIdx.x & 31) == 0) a.n_scale[t * blocks + b] = (uint8_t)code;
            }
        }
        if (threadIdx.x == 0) reinterpret_cast<float4*>(a.stats)[t] = make_float4(r.pm, r.pr, r.nm, r.nr);
    }
}

template <class T>
__device__ float at(const void* p, int64_t ld, int64_t t, int64_t j) {
    return p ? to_f(static_cast<const T*>(p)[t * ld + j]) : 0.0f;
}

// dx and dh, and per row the two means that dY needs
template <class T>
__global__ void __launch_bounds__(THREADS) k_block_norm_rows(Args<T> q, wc_block_norm_grads g, float2* means) {
    __shared__ float s[32];
    const wc_block_norm_args& a = q.a;
    const int64_t D = a.width;
    const float inv = 1.0f / (float)D;
    const bool layer = a.kind == WC_NORM_LAYER, pre = a.pre_weight && g.dn;
    for (int64_t t = blockIdx.x; t < a.rows; t += gridDim.x) {
        const float4 st = reinterpret_cast<const float4*>(a.stats)[t];
        const Row r{st.x, st.y, st.z, st.w};
        const T* gate = q.gate(t);
        auto yhat = [&](int64_t j) { return (q.y(t, j, q.u(q.hhat(t, j, r), j), gate) - r.nm) * r.nr; };
        float m0 = 0.0f, m1 = 0.0f;
        if (pre) {
            for (int64_t j = threadIdx.x; j < D; j += THREADS) {
                const float d = at<T>(g.dn, g.ld_dn, t, j) * a.pre_weight[j];
                m0 += d, m1 += d * yhat(j);
            }
            m0 = layer ? cta_sum(m0, s) * inv : 0.0f;
            m1 = cta_sum(m1, s) * inv;
        }
        if (threadIdx.x == 0) means[t] = make_float2(m0, m1);
        auto dY = [&](int64_t j) {
            float d = at<T>(g.dy, g.ld_dy, t, j);
            if (pre) d += r.nr * (at<T>(g.dn, g.ld_dn, t, j) * a.pre_weight[j] - m0 - yhat(j) * m1);
            return d;
        };
        auto dU = [&](int64_t j) { return dY(j) * (gate ? to_f(gate[j]) : 1.0f) * (a.post_weight ? a.post_weight[j] : 1.0f); };
        float c0 = 0.0f, c1 = 0.0f;
        if (a.post_weight && g.dh) {
            for (int64_t j = threadIdx.x; j < D; j += THREADS) {
                const float d = dU(j);
                c0 += d, c1 += d * q.hhat(t, j, r);
            }
            c0 = layer ? cta_sum(c0, s) * inv : 0.0f;
            c1 = cta_sum(c1, s) * inv;
        }
        for (int64_t j = threadIdx.x; j < D; j += THREADS) {
            if (g.dx) static_cast<T*>(g.dx)[t * g.ld_dx + j] = from_f<T>(a.residual_scale * dY(j));
            if (g.dh) static_cast<T*>(g.dh)[t * g.ld_dh + j] =
                from_f<T>(a.post_weight ? r.pr * (dU(j) - c0 - q.hhat(t, j, r) * c1) : dU(j));
        }
    }
}

// Items are (group, segment of its rows); a CTA column y takes items y, y +
// gridDim.y, ... It keeps the weights' sums over all of them and writes the
// gate's sum of each.
template <class T>
__global__ void __launch_bounds__(THREADS) k_block_norm_cols(Args<T> q, wc_block_norm_grads g, const float2* means,
                                                             int64_t items, int segments, int64_t per, float* gate_part,
                                                             float* weight_part) {
    __shared__ float s[5][8][32];
    const wc_block_norm_args& a = q.a;
    const int64_t D = a.width, j = (int64_t)blockIdx.x * 32 + (threadIdx.x & 31);
    const int w = threadIdx.x / 32;
    const int64_t R = a.gate ? a.rows_per_gate : a.rows;
    float acc[4] = {};
    for (int64_t i = blockIdx.y; i < items; i += gridDim.y) {
        const int64_t group = i / segments, first = group * R + (i - group * segments) * per;
        const int64_t last = min(min(first + per, (group + 1) * R), a.rows);
        float dg = 0.0f;
        if (j < D)
            for (int64_t t = first + w; t < last; t += 8) {
                const float4 st = reinterpret_cast<const float4*>(a.stats)[t];
                const Row r{st.x, st.y, st.z, st.w};
                const T* gate = q.gate(t);
                const float hh = q.hhat(t, j, r), u = q.u(hh, j), yh = (q.y(t, j, u, gate) - r.nm) * r.nr;
                const float dn = at<T>(g.dn, g.ld_dn, t, j);
                float d = at<T>(g.dy, g.ld_dy, t, j);
                if (a.pre_weight && g.dn) d += r.nr * (dn * a.pre_weight[j] - means[t].x - yh * means[t].y);
                dg += d * u;
                const float du = d * (gate ? to_f(gate[j]) : 1.0f);
                acc[0] += du * hh, acc[1] += du, acc[2] += dn * yh, acc[3] += dn;
            }
        if (g.dgate) {
            __syncthreads();
            s[4][w][threadIdx.x & 31] = dg;
            __syncthreads();
            if (w == 0 && j < D) {
                for (int k = 1; k < 8; ++k) dg += s[4][k][threadIdx.x];
                if (segments == 1) static_cast<T*>(g.dgate)[group * D + j] = from_f<T>(dg);
                else gate_part[i * D + j] = dg;
            }
        }
    }
    for (int k = 0; k < 4; ++k) s[k][w][threadIdx.x & 31] = acc[k];
    __syncthreads();
    if (w == 0 && j < D)
        for (int k = 0; k < 4; ++k) {
            float v = acc[k];
            for (int i = 1; i < 8; ++i) v += s[k][i][threadIdx.x];
            weight_part[(blockIdx.y * 4 + k) * D + j] = v;
        }
}

// the segments of a group joined
template <class T>
__global__ void k_gate_sum(const float* part, int segments, int64_t D, int64_t total, T* out) {
    for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
        const int64_t group = i / D, j = i - group * D;
        float v = 0.0f;
        for (int k = 0; k < segments; ++k) v += part[(group * segments + k) * D + j];
        out[i] = from_f<T>(v);
    }
}

// ---- units -------------------------------------------------------------------
template <class T>
struct Unit {
    uint4 w[sizeof(T) / 2];
    __device__ __forceinline__ void load(const T* p) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) w[i] = reinterpret_cast<const uint4*>(p)[i];
    }
    __device__ __forceinline__ void stream(const T* p) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) w[i] = __ldcs(reinterpret_cast<const uint4*>(p) + i);
    }
    __device__ __forceinline__ void get(float* v) const {
        alignas(16) T e[8];
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) reinterpret_cast<uint4*>(e)[i] = w[i];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = to_f(e[i]);
    }
    // the same in pairs
    __device__ __forceinline__ void get(unsigned long long* v) const {
        float f[8];
        get(f);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = umma::f2(f[2 * i], f[2 * i + 1]);
    }
    __device__ __forceinline__ static void put(T* p, const unsigned long long* v) {
        float f[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) f[2 * i] = umma::f2_lo(v[i]), f[2 * i + 1] = umma::f2_hi(v[i]);
        put(p, f);
    }
    __device__ __forceinline__ static void put(T* p, const float* v) {
        alignas(16) T e[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = from_f<T>(v[i]);
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) __stcs(reinterpret_cast<uint4*>(p) + i, reinterpret_cast<const uint4*>(e)[i]);
    }
};
__device__ __forceinline__ void load8(const float* p, float* v) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
}
__device__ __forceinline__ void store8(float* p, const float* v) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    *reinterpret_cast<float4*>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
}
__device__ __forceinline__ void fill8(float* v, float x) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = x;
}

// Sums over the threads that share a row: `lanes` of a warp, or the CTA (each
// warp's sum through shared memory, two arrays in turn so that one barrier a
// sum is enough).
template <int WARPS>
struct Group {
    float2 (*s)[32];
    int lanes, turn = 0;
    __device__ __forceinline__ float2 sum(float2 v) {
        for (int o = WARPS ? 16 : lanes >> 1; o; o >>= 1) v.x += __shfl_xor_sync(~0u, v.x, o), v.y += __shfl_xor_sync(~0u, v.y, o);
        if (!WARPS) return v;
        const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
        if (lane == 0) s[turn][threadIdx.x >> 5] = v;
        __syncthreads();
        v = lane < warps ? s[turn][lane] : make_float2(0.0f, 0.0f);
#pragma unroll
        for (int o = WARPS > 16 ? 16 : WARPS > 8 ? 8 : WARPS > 4 ? 4 : 2; o; o >>= 1) v.x += __shfl_xor_sync(~0u, v.x, o), v.y += __shfl_xor_sync(~0u, v.y, o);
        v.x = __shfl_sync(~0u, v.x, 0), v.y = __shfl_sync(~0u, v.y, 0);
        turn ^= 1;
        return v;
    }
    __device__ __forceinline__ float sum(float v) { return sum(make_float2(v, 0.0f)).x; }
};

// WARPS = 0: `lanes` threads of a warp a row, else a CTA of up to WARPS warps;
// NV units a thread, `lanes` (or blockDim.x) apart.
template <class T, int WARPS, int NV>
__global__ void __launch_bounds__(WARPS ? WARPS * 32 : 256, WARPS ? (WARPS < 32 ? 40 / (WARPS ? WARPS : 1) : 1) : 4) k_norm_units(wc_block_norm_args a, int lanes) {
    __shared__ float2 s[2][32];
    Group<WARPS> group{s, lanes};
    const int D = (int)a.width, at = WARPS ? threadIdx.x : (int)(threadIdx.x & (lanes - 1)), apart = WARPS ? (int)blockDim.x : lanes;
    const int per = WARPS ? 1 : 256 / lanes, slot = WARPS ? 0 : (int)threadIdx.x / lanes;
    const int blocks = (D + 31) / 32;
    const float inv = 1.0f / (float)D;
    const bool layer = a.kind == WC_NORM_LAYER;
    for (int64_t t0 = (int64_t)blockIdx.x * per; t0 < a.rows; t0 += (int64_t)gridDim.x * per) {
        const int64_t t = t0 + slot;
        const bool in = t < a.rows;
        Unit<T> x[NV];
        float v[NV][8];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * apart + at) * 8;
            fill8(v[i], 0.0f);
            if (in && c < D) {
                Unit<T> h;
                h.stream(static_cast<const T*>(a.h) + t * a.ld_h + c);
                x[i].stream(static_cast<const T*>(a.x) + t * a.ld_x + c);
                h.get(v[i]);
            }
        }
        // moments of what is in v; columns past the width are 0 and count for nothing
        auto moments = [&](float& mean, float& r) {
            if (layer) {
                float m = 0.0f;
#pragma unroll
                for (int i = 0; i < NV; ++i)
#pragma unroll
                    for (int k = 0; k < 8; ++k) m += v[i][k];
                mean = group.sum(m) * inv;
            }
            float q = 0.0f;
#pragma unroll
            for (int i = 0; i < NV; ++i)
                if ((i * apart + at) * 8 < D)
#pragma unroll
                    for (int k = 0; k < 8; ++k) q = fmaf(v[i][k] - mean, v[i][k] - mean, q);
            r = rsqrtf(group.sum(q) * inv + a.eps);
        };
        Row r{0.0f, 1.0f, 0.0f, 1.0f};
        if (a.post_weight) moments(r.pm, r.pr);
        const T* gate = a.gate && in ? static_cast<const T*>(a.gate) + t / a.rows_per_gate * D : nullptr;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * apart + at) * 8;
            if (!in || c >= D) continue;
            if (a.post_weight) {
                float w[8], b[8];
                load8(a.post_weight + c, w);
                if (a.post_bias) load8(a.post_bias + c, b);
                else fill8(b, 0.0f);
#pragma unroll
                for (int k = 0; k < 8; ++k) v[i][k] = fmaf((v[i][k] - r.pm) * r.pr, w[k], b[k]);
            }
            float xf[8];
            x[i].get(xf);
            if (gate) {
                Unit<T> gu;
                gu.load(gate + c);
                float g[8];
                gu.get(g);
#pragma unroll
                for (int k = 0; k < 8; ++k) v[i][k] = fmaf(a.residual_scale, xf[k], g[k] * v[i][k]);
            } else {
#pragma unroll
                for (int k = 0; k < 8; ++k) v[i][k] = fmaf(a.residual_scale, xf[k], v[i][k]);
            }
            Unit<T>::put(static_cast<T*>(a.y) + t * a.ld_y + c, v[i]);
        }
        if (a.pre_weight) {
            moments(r.nm, r.nr);
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int c = (i * apart + at) * 8;
                const bool here = in && c < D;
                if (here) {
                    float w[8], b[8];
                    load8(a.pre_weight + c, w);
                    if (a.pre_bias) load8(a.pre_bias + c, b);
                    else fill8(b, 0.0f);
#pragma unroll
                    for (int k = 0; k < 8; ++k) v[i][k] = fmaf((v[i][k] - r.nm) * r.nr, w[k], b[k]);
                    if (a.n) Unit<T>::put(static_cast<T*>(a.n) + t * a.ld_n + c, v[i]);
                }
                if (a.n_q) {  // 4 threads next to each other hold a block (lanes is at least 4 then)
                    uint32_t code;
                    const uint2 q = quantise8(v[i], &code);
                    if (in && c < blocks * 32) {
                        *reinterpret_cast<uint2*>(a.n_q + t * blocks * 32 + c) = q;
                        if ((c & 31) == 0) a.n_scale[t * blocks + c / 32] = (uint8_t)code;
                    }
                }
            }
        }
        if (in && at == 0) reinterpret_cast<float4*>(a.stats)[t] = make_float4(r.pm, r.pr, r.nm, r.nr);
    }
}

// ---- the backward pass -----------------------------------------------------------
// Rows come in items, a segment of a group of rows with the same gate. Worker w
// takes items w, w + workers, ...: it keeps the weights' sums over all of them
// and hands on the gate's sum of each.
struct Plan {
    int64_t R, groups, per, items;
    int segments, workers, lanes, parts;  // lanes of a warp a row (0: a CTA a row, -1: the general kernels)
    Plan(const wc_block_norm_args& a, bool units) {
        R = a.gate ? a.rows_per_gate : a.rows;
        groups = a.rows ? (a.rows + R - 1) / R : 0;
        lanes = !units || a.width > 4096 ? -1 : 0;
        if (units && a.width <= 256)
            for (lanes = 1; lanes * 8 < a.width;) lanes *= 2;
        const int64_t most = lanes > 0 ? 148 * 2 * 8 : lanes == 0 ? (a.width <= 2048 ? 296 : 148) : 512;
        const int64_t longest = R < a.rows ? R : a.rows, want = groups ? (most + groups - 1) / groups : 1;
        const int64_t fit = (longest + 7) / 8;
        segments = (int)(fit < 1 ? 1 : fit < want ? fit : want);
        per = longest ? (longest + segments - 1) / segments : 1;
        items = groups * segments;
        workers = (int)(items < most ? items : most);
        parts = lanes > 0 ? (workers + 7) / 8 : workers;  // partial sums of the weights
    }
    uint64_t floats(const wc_block_norm_args& a) const {
        return 2 * (uint64_t)(a.rows + 1) + (uint64_t)parts * 4 * a.width + (segments > 1 ? (uint64_t)items * a.width : 0);
    }
};
struct Items {
    int64_t items, per, R, rows;
    int segments, workers;
    __device__ __forceinline__ void range(int64_t i, int64_t& group, int64_t& first, int64_t& last) const {
        group = i / segments, first = group * R + (i - group * segments) * per;
        last = min(min(first + per, (group + 1) * R), rows);
    }
};

// Arithmetic on pairs of 32-bit numbers (umma.cuh), each rounded as the scalar form: the backward pass has some 30
// operations a column, which would bound it before the bytes do.
using Pair = unsigned long long;
__device__ __forceinline__ Pair twice(float v) { return umma::f2(v, v); }
__device__ __forceinline__ Pair mul(Pair a, Pair b) {
    Pair d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ Pair add(Pair a, Pair b) { return umma::f2_add(a, b); }
__device__ __forceinline__ Pair fma(Pair a, Pair b, Pair c) { return umma::f2_fma(a, b, c); }
__device__ __forceinline__ float both(Pair a) { return umma::f2_lo(a) + umma::f2_hi(a); }

// What a thread keeps of its unit: the parameters and their gradients' sums.
struct Column {
    Pair wp[4], bp[4], wn[4], g[4];
    Pair dwp[4], dbp[4], dwn[4], dbn[4], dg[4];
    __device__ __forceinline__ static void fill(Pair* v, float x) {
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = twice(x);
    }
    __device__ __forceinline__ static void load(Pair* v, const float* p) {
        const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
        v[0] = umma::f2(a.x, a.y), v[1] = umma::f2(a.z, a.w), v[2] = umma::f2(b.x, b.y), v[3] = umma::f2(b.z, b.w);
    }
    __device__ __forceinline__ static void unpack(const Pair* v, float* f) {
#pragma unroll
        for (int k = 0; k < 4; ++k) f[2 * k] = umma::f2_lo(v[k]), f[2 * k + 1] = umma::f2_hi(v[k]);
    }
    __device__ __forceinline__ void load(const wc_block_norm_args& a, int c, bool in) {
        fill(wp, 1.0f), fill(bp, 0.0f), fill(wn, 0.0f), fill(g, 1.0f);
        fill(dwp, 0.0f), fill(dbp, 0.0f), fill(dwn, 0.0f), fill(dbn, 0.0f), fill(dg, 0.0f);
        if (!in) return;
        if (a.post_weight) load(wp, a.post_weight + c);
        if (a.post_bias) load(bp, a.post_bias + c);
        if (a.pre_weight) load(wn, a.pre_weight + c);
    }
    // A row's unit. get(i, v) reads its x, h, dy or dn (i = 0 .. 3; zeros past the width and for a gradient that is not
    // there), when it is needed: what is not held meanwhile leaves room for the sums. put(i, v) takes dx, then dh.
    template <class G, class Get, class Put>
    __device__ __forceinline__ void row(const wc_block_norm_args& a, const float4& st, bool pre, bool in, float inv, G& group, Get&& get,
                                        Put&& put) {
        const bool layer = a.kind == WC_NORM_LAYER;
        Pair hh[4], yh[4], d[4];
        get(1, hh), get(0, yh);
        const Pair pr = twice(st.y), pm = twice(-st.x), nr = twice(st.w), nm = twice(-st.z), rs = twice(a.residual_scale);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            hh[k] = mul(add(hh[k], pm), pr);
            yh[k] = mul(add(fma(rs, yh[k], mul(g[k], fma(hh[k], wp[k], bp[k]))), nm), nr);
        }
        if (pre) {
            Pair m0 = 0, m1 = 0;  // pairs of zeros
            get(3, d);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                dwn[k] = fma(d[k], yh[k], dwn[k]), dbn[k] = add(dbn[k], d[k]);
                d[k] = mul(d[k], wn[k]);
                m0 = add(m0, d[k]), m1 = fma(d[k], yh[k], m1);
            }
            const float2 m = group.sum(make_float2(both(m0), both(m1)));
            const Pair a0 = twice(layer ? -m.x * inv : 0.0f), a1 = twice(-m.y * inv);
#pragma unroll
            for (int k = 0; k < 4; ++k) yh[k] = mul(nr, fma(yh[k], a1, add(d[k], a0)));
        } else {
            fill(yh, 0.0f);
        }
        get(2, d);
        const Pair live = twice(in ? 1.0f : 0.0f);
#pragma unroll
        for (int k = 0; k < 4; ++k) yh[k] = mul(live, add(d[k], yh[k])), d[k] = mul(rs, yh[k]);  // dY
        put(0, d);
        Pair c0 = 0, c1 = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            dg[k] = fma(yh[k], fma(hh[k], wp[k], bp[k]), dg[k]);
            const Pair du = mul(yh[k], g[k]);
            dwp[k] = fma(du, hh[k], dwp[k]), dbp[k] = add(dbp[k], du);
            yh[k] = mul(du, wp[k]);
            c0 = add(c0, yh[k]), c1 = fma(yh[k], hh[k], c1);
        }
        if (a.post_weight) {
            const float2 c = group.sum(make_float2(both(c0), both(c1)));
            const Pair a0 = twice(layer ? -c.x * inv : 0.0f), a1 = twice(-c.y * inv);
#pragma unroll
            for (int k = 0; k < 4; ++k) yh[k] = mul(pr, fma(hh[k], a1, add(yh[k], a0)));
        }
        put(1, yh);
    }
};

// A part of a warp a row; a warp is a worker.
template <class T>
__global__ void __launch_bounds__(256, 2) k_norm_backward_warp(wc_block_norm_args a, wc_block_norm_grads g, Items q, int lanes,
                                                               float* gate_part, float* weight_part) {
    __shared__ float s[8][8][33];
    const int D = (int)a.width, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, at = lane & (lanes - 1), c = at * 8;
    const int slots = 32 / lanes, slot = lane / lanes, worker = blockIdx.x * 8 + warp;
    const bool in = c < D, pre = a.pre_weight && g.dn;
    const float inv = 1.0f / (float)D;
    Group<0> group{nullptr, lanes};
    Column col;
    col.load(a, c, in);
    for (int64_t i = worker; i < q.items; i += q.workers) {
        int64_t item_group, first, last;
        q.range(i, item_group, first, last);
        if (a.gate && in) {
            Unit<T> gate;
            gate.load(static_cast<const T*>(a.gate) + item_group * D + c);
            gate.get(col.g);
        }
        Unit<T> u[4];  // x, h, dy, dn: the next row's from when dx is out
        float4 next = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        auto fetch = [&](int64_t t) {
            const bool here = in && t < last;
#pragma unroll
            for (int k = 0; k < 4; ++k) u[k] = Unit<T>{};
            if (here) {
                u[0].stream(static_cast<const T*>(a.x) + t * a.ld_x + c);
                u[1].stream(static_cast<const T*>(a.h) + t * a.ld_h + c);
                if (g.dy) u[2].stream(static_cast<const T*>(g.dy) + t * g.ld_dy + c);
                if (g.dn) u[3].stream(static_cast<const T*>(g.dn) + t * g.ld_dn + c);
            }
            if (t < last) next = reinterpret_cast<const float4*>(a.stats)[t];
        };
        fetch(first + slot);
        for (int64_t t0 = first; t0 < last; t0 += slots) {
            const int64_t t = t0 + slot;
            const float4 st = next;
            const bool here = in && t < last;
            col.row(a, st, pre, here, inv, group, [&](int i, Pair* v) { u[i].get(v); },
                    [&](int i, const Pair* v) {
                        if (i == 0 && here && g.dx) Unit<T>::put(static_cast<T*>(g.dx) + t * g.ld_dx + c, v);
                        if (i == 0) fetch(t + slots);
                        if (i == 1 && here && g.dh) Unit<T>::put(static_cast<T*>(g.dh) + t * g.ld_dh + c, v);
                    });
        }
        if (g.dgate) {
            float dg[8];
            Column::unpack(col.dg, dg);
#pragma unroll
            for (int k = 0; k < 8; ++k)
                for (int o = 16; o >= lanes; o >>= 1) dg[k] += __shfl_xor_sync(~0u, dg[k], o);
            if (slot == 0 && in) {
                if (q.segments == 1) Unit<T>::put(static_cast<T*>(g.dgate) + item_group * D + c, dg);
                else store8(gate_part + i * D + c, dg);
            }
            Column::fill(col.dg, 0.0f);
        }
    }
    // the slots of a warp, then the warps
    auto flush = [&](const Pair* sum, int which) {
        float v[8];
        Column::unpack(sum, v);
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            for (int o = 16; o >= lanes; o >>= 1) v[k] += __shfl_xor_sync(~0u, v[k], o);
            s[warp][k][lane] = v[k];
        }
        __syncthreads();
        const int k = warp;
        if (slot == 0 && in) {
            float t = 0.0f;
#pragma unroll
            for (int w = 0; w < 8; ++w) t += s[w][k][lane];
            weight_part[((int64_t)blockIdx.x * 4 + which) * D + c + k] = t;
        }
    };
    flush(col.dwp, 0), flush(col.dbp, 1), flush(col.dwn, 2), flush(col.dbn, 3);
}

// A CTA a row, one unit a thread; a CTA is a worker. Its rows in order come to
// shared memory by bulk copies: x, h, dy, dn and the statistics.
constexpr int MAX_RING = 8;
template <class T>
__global__ void __launch_bounds__(512) k_norm_backward_cta(wc_block_norm_args a, wc_block_norm_grads g, Items q, int stages,
                                                           float* gate_part, float* weight_part) {
    extern __shared__ __align__(128) uint8_t ring[];
    __shared__ float2 s[2][32];
    __shared__ uint64_t full[MAX_RING];
    const int D = (int)a.width, c = threadIdx.x * 8, row_bytes = D * (int)sizeof(T), stage_bytes = 4 * row_bytes + 16;
    const bool in = c < D, pre = a.pre_weight && g.dn;
    const float inv = 1.0f / (float)D;
    Group<16> group{s, 32};
    Column col;
    col.load(a, c, in);
    if (threadIdx.x == 0) {
        for (int i = 0; i < stages; ++i) umma::mbar_init(&full[i], 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    // thread 0 walks ahead of the rows
    int64_t copy_item = blockIdx.x, copy_row = 0, copy_last = 0, copy_group;
    int copied = 0;
    auto copy = [&] {
        while (copy_row >= copy_last) {
            if (copy_item >= q.items) return;
            q.range(copy_item, copy_group, copy_row, copy_last);
            copy_item += q.workers;
        }
        const int slot = copied % stages;
        uint8_t* to = ring + slot * stage_bytes;
        umma::expect_tx(&full[slot], (2 + (g.dy != nullptr) + (g.dn != nullptr)) * row_bytes + 16);
        umma::bulk_g2s(to, static_cast<const T*>(a.x) + copy_row * a.ld_x, row_bytes, &full[slot]);
        umma::bulk_g2s(to + row_bytes, static_cast<const T*>(a.h) + copy_row * a.ld_h, row_bytes, &full[slot]);
        if (g.dy) umma::bulk_g2s(to + 2 * row_bytes, static_cast<const T*>(g.dy) + copy_row * g.ld_dy, row_bytes, &full[slot]);
        if (g.dn) umma::bulk_g2s(to + 3 * row_bytes, static_cast<const T*>(g.dn) + copy_row * g.ld_dn, row_bytes, &full[slot]);
        umma::bulk_g2s(to + 4 * row_bytes, a.stats + copy_row * 4, 16, &full[slot]);
        ++copied, ++copy_row;
    };
    if (threadIdx.x == 0)
        for (int i = 0; i + 1 < stages; ++i) copy();
    int done = 0;
    bool bad = false;
    for (int64_t i = blockIdx.x; i < q.items; i += q.workers) {
        int64_t item_group, first, last;
        q.range(i, item_group, first, last);
        if (a.gate && in) {
            Unit<T> u;
            u.load(static_cast<const T*>(a.gate) + item_group * D + c);
            u.get(col.g);
        }
        for (int64_t t = first; t < last; ++t, ++done) {
            const int slot = done % stages;
            // a copy that does not come (umma.cuh) leaves NaN from here on
            if (!bad && !umma::mbar_wait(&full[slot], (uint32_t)(done / stages) & 1)) bad = true;
            const T* from = reinterpret_cast<const T*>(ring + slot * stage_bytes);
            float4 st = *reinterpret_cast<const float4*>(ring + slot * stage_bytes + 4 * row_bytes);
            if (bad) st.y = st.w = __uint_as_float(0x7fffffffu);
            __syncthreads();  // all have done with the row before this one: its stage takes another
            if (threadIdx.x == 0 && !bad) copy();
            col.row(a, st, pre, in, inv, group,
                    [&](int i, Pair* v) {
                        Column::fill(v, 0.0f);
                        if (!in || (i == 2 && !g.dy) || (i == 3 && !g.dn)) return;
                        Unit<T> u;
                        u.load(from + i * D + c), u.get(v);
                    },
                    [&](int i, const Pair* v) {
                        if (!in) return;
                        if (i == 0 && g.dx) Unit<T>::put(static_cast<T*>(g.dx) + t * g.ld_dx + c, v);
                        if (i == 1 && g.dh) Unit<T>::put(static_cast<T*>(g.dh) + t * g.ld_dh + c, v);
                    });
        }
        if (g.dgate && in) {
            float dg[8];
            Column::unpack(col.dg, dg);
            if (q.segments == 1) Unit<T>::put(static_cast<T*>(g.dgate) + item_group * D + c, dg);
            else store8(gate_part + i * D + c, dg);
        }
        Column::fill(col.dg, 0.0f);
    }
    if (bad && threadIdx.x == 0)
        for (int k = 0; k < stages; ++k) umma::mbar_wait(&full[k], 0, umma::DRAIN_NS / 4), umma::mbar_wait(&full[k], 1, umma::DRAIN_NS / 4);
    if (in) {
        float* to = weight_part + (int64_t)blockIdx.x * 4 * D + c;
        const Pair* sums[4] = {col.dwp, col.dbp, col.dwn, col.dbn};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            float v[8];
            Column::unpack(sums[k], v);
            store8(to + k * D, v);
        }
    }
}

bool unit_rows(const void* p, int64_t ld, size_t e) { return !p || (((uintptr_t)p & 15) == 0 && (ld * e) % 16 == 0); }
// whether the shared matrices and the parameters can be read in units
bool units_ok(const wc_block_norm_args& a) {
    const size_t e = a.type == WC_F32 ? 4 : 2;
    const auto fine = [](const float* p) { return ((uintptr_t)p & 15) == 0; };
    return a.width % 8 == 0 && unit_rows(a.x, a.ld_x, e) && unit_rows(a.h, a.ld_h, e) && unit_rows(a.gate, a.width, e) &&
           fine(a.post_weight) && fine(a.post_bias) && fine(a.pre_weight) && fine(a.pre_bias);
}

template <class T>
void backward(const wc_block_norm_args& a, const wc_block_norm_grads& g, cudaStream_t s) {
    const size_t e = sizeof(T);
    const bool units = units_ok(a) && unit_rows(g.dy, g.ld_dy, e) && unit_rows(g.dn, g.ld_dn, e) && unit_rows(g.dx, g.ld_dx, e) &&
                       unit_rows(g.dh, g.ld_dh, e) && unit_rows(g.dgate, a.width, e);
    const Plan p(a, units);
    float* ws = static_cast<float*>(g.workspace);
    const int64_t D = a.width;
    float2* means = reinterpret_cast<float2*>(ws);
    float *weights = ws + (a.rows + 1) / 2 * 4, *gates = weights + (int64_t)p.parts * 4 * D;  // both 16-byte aligned where D is a multiple of 4
    if (a.rows) {
        const Items q{p.items, p.per, p.R, a.rows, p.segments, p.workers};
        if (p.lanes > 0) {
            k_norm_backward_warp<T><<<p.parts, 256, 0, s>>>(a, g, q, p.lanes, gates, weights);
        } else if (p.lanes == 0) {
            const int stage = 4 * (int)D * (int)e + 16, threads = (int)(D / 8 + 31) / 32 * 32;
            const int stages = std::min(MAX_RING, (D <= 2048 ? 100 : 200) * 1024 / stage);
            if (wcdev::raise_smem_limit(reinterpret_cast<const void*>(k_norm_backward_cta<T>), 200 * 1024))
                k_norm_backward_cta<T><<<p.workers, threads, (size_t)stages * stage, s>>>(a, g, q, stages, gates, weights);
        } else {
            k_block_norm_rows<T><<<(unsigned)(a.rows < 148 * 8 ? a.rows : 148 * 8), THREADS, 0, s>>>(Args<T>{a}, g, means);
            k_block_norm_cols<T><<<dim3((unsigned)((D + 31) / 32), p.workers), THREADS, 0, s>>>(
                Args<T>{a}, g, means, p.items, p.segments, p.per, gates, weights);
        }
        if (g.dgate && p.segments > 1)
            k_gate_sum<T><<<148 * 4, 256, 0, s>>>(gates, p.segments, D, p.groups * D, static_cast<T*>(g.dgate));
    }
    float* to[4] = {g.dpost_weight, g.dpost_bias, g.dpre_weight, g.dpre_bias};
    for (int k = 0; k < 4; ++k)
        if (to[k]) launch_colsum<float>(weights + k * D, p.parts, 4 * D, D, to[k], s);
}

template <class T>
void forward(const wc_block_norm_args& a, cudaStream_t s) {
    if (!a.rows) return;
    const size_t e = sizeof(T);
    if (!units_ok(a) || !unit_rows(a.y, a.ld_y, e) || !unit_rows(a.n, a.ld_n, e)) {
        k_block_norm<T><<<(unsigned)(a.rows < 148 * 8 ? a.rows : 148 * 8), THREADS, 0, s>>>(Args<T>{a});
        return;
    }
    // units of a row, whole blocks of 32 columns where it is packed
    const int units = (int)(a.n_q ? (a.width + 31) / 32 * 4 : a.width / 8);
    if (units <= 64) {
        int lanes = a.n_q ? 4 : 1;
        while (lanes < 32 && lanes * 2 < units) lanes *= 2;
        const int64_t per = 256 / lanes;
        const unsigned n = (unsigned)std::min<int64_t>(148 * 16, (a.rows + per - 1) / per);
        if (units <= lanes) k_norm_units<T, 0, 1><<<n, 256, 0, s>>>(a, lanes);
        else k_norm_units<T, 0, 2><<<n, 256, 0, s>>>(a, lanes);
        return;
    }
    // two units a thread
    const int threads = (units + 63) / 64 * 32;
    const unsigned n = (unsigned)std::min<int64_t>(148 * std::max(1, 2048 / threads), a.rows);
    if (threads <= 128) k_norm_units<T, 4, 2><<<n, threads, 0, s>>>(a, 32);
    else if (threads <= 256) k_norm_units<T, 8, 2><<<n, threads, 0, s>>>(a, 32);
    else if (threads <= 512) k_norm_units<T, 16, 2><<<n, threads, 0, s>>>(a, 32);
    else k_norm_units<T, 32, 2><<<n, threads, 0, s>>>(a, 32);
}

}  // namespace

// for either path: which one the gradients' addresses decide
uint64_t block_norm_workspace(const wc_block_norm_args& a) {
    return std::max(Plan(a, true).floats(a), Plan(a, false).floats(a)) * sizeof(float) + 16;
}

void launch_block_norm(const wc_block_norm_args& a, cudaStream_t s) {
    if (a.type == WC_F32) forward<float>(a, s);
    else if (a.type == WC_F16) forward<__half>(a, s);
    else forward<__nv_bfloat16>(a, s);
}

void launch_block_norm_backward(const wc_block_norm_args& a, const wc_block_norm_grads& g, cudaStream_t s) {
    if (a.type == WC_F32) backward<float>(a, g, s);
    else if (a.type == WC_F16) backward<__half>(a, g, s);
    else backward<__nv_bfloat16>(a, g, s);
}

}  // namespace wctrain
