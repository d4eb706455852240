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
#include "colsum.cuh"

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

struct Plan {
    int64_t groups, per, items;
    int segments, workers;
    explicit Plan(const wc_block_norm_args& a) {
        const int64_t R = a.gate ? a.rows_per_gate : a.rows;
        groups = a.rows ? (a.rows + R - 1) / R : 0;
        const int64_t longest = R < a.rows ? R : a.rows, want = groups ? (512 + groups - 1) / groups : 1;
        const int64_t most = (longest + 7) / 8;
        segments = (int)(most < 1 ? 1 : most < want ? most : want);
        per = longest ? (longest + segments - 1) / segments : 1;
        items = groups * segments;
        workers = (int)(items < 512 ? items : 512);
    }
    uint64_t floats(const wc_block_norm_args& a) const {
        return 2 * (uint64_t)a.rows + (uint64_t)workers * 4 * a.width + (segments > 1 ? (uint64_t)items * a.width : 0);
    }
};

template <class T>
void backward(const wc_block_norm_args& a, const wc_block_norm_grads& g, cudaStream_t s) {
    const Plan p(a);
    float* ws = static_cast<float*>(g.workspace);
    float2* means = reinterpret_cast<float2*>(ws);
    float *weights = ws + 2 * a.rows, *gates = weights + (int64_t)p.workers * 4 * a.width;
    const int64_t D = a.width;
    if (a.rows) {
        k_block_norm_rows<T><<<(unsigned)(a.rows < 148 * 8 ? a.rows : 148 * 8), THREADS, 0, s>>>(Args<T>{a}, g, means);
        k_block_norm_cols<T><<<dim3((unsigned)((D + 31) / 32), p.workers), THREADS, 0, s>>>(
            Args<T>{a}, g, means, p.items, p.segments, p.per, gates, weights);
        if (g.dgate && p.segments > 1)
            k_gate_sum<T><<<148 * 4, 256, 0, s>>>(gates, p.segments, D, p.groups * D, static_cast<T*>(g.dgate));
    }
    float* to[4] = {g.dpost_weight, g.dpost_bias, g.dpre_weight, g.dpre_bias};
    for (int k = 0; k < 4; ++k)
        if (to[k]) launch_colsum<float>(weights + k * D, p.workers, 4 * D, D, to[k], s);
}

template <class T>
void forward(const wc_block_norm_args& a, cudaStream_t s) {
    if (a.rows) k_block_norm<T><<<(unsigned)(a.rows < 148 * 8 ? a.rows : 148 * 8), THREADS, 0, s>>>(Args<T>{a});
}

}  // namespace

uint64_t block_norm_workspace(const wc_block_norm_args& a) { return Plan(a).floats(a) * sizeof(float); }

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
