// The clipped policy loss with a KL term, and its gradient at the logits.
//
// With base-2 logits x_j = (z_j - max) log2(e): S = sum 2^x_j, p_j = 2^x_j / S,
// l = (x_a - log2 S) ln 2, H = (log2 S - sum p_j x_j) ln 2. The row's loss
// depends on the logits through l and H only, so
//   dloss/dz_j = g (delta_ja - p_j) + w c p_j (ln p_j + H),
//   g = w (-ratio A [not clipped] - kl_coef (exp(r - l) - 1)).
#include "train.cuh"

namespace wctrain {

namespace {

constexpr int THREADS = 256;
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

// running maximum of the base-2 logits, sum of powers, and sum of powers times exponent
struct Run {
    float m, s, w;
    __device__ void join(const Run& o) {
        const float hi = fmaxf(m, o.m);
        if (hi == -INFINITY) return;
        const float ra = exp2f(m - hi), rb = exp2f(o.m - hi);
        const float wa = m == -INFINITY ? 0.0f : (w + s * (m - hi)) * ra;
        const float wb = o.m == -INFINITY ? 0.0f : (o.w + o.s * (o.m - hi)) * rb;
        s = s * ra + o.s * rb, w = wa + wb, m = hi;
    }
    __device__ void add(float x) { join(Run{x, 1.0f, 0.0f}); }
};

// per-row scalars of the loss from l and H
struct RowLoss {
    float row, kl, pull;  // pull: dloss/dl without the weight
    __device__ RowLoss(float l, float H, float old, float A, bool has_ref, float ref, const wc_policy_loss_args& a) {
        const float ratio = expf(l - old), lo = 1.0f - a.clip_low, hi = 1.0f + a.clip_high;
        const float gain = fminf(ratio * A, fminf(fmaxf(ratio, lo), hi) * A);
        const bool held = (A > 0.0f && ratio > hi) || (A < 0.0f && ratio < lo);
        const float d = has_ref ? ref - l : 0.0f, em = has_ref ? expm1f(d) : 0.0f;
        kl = em - d;
        row = -gain + a.kl_coef * kl - a.entropy_coef * H;
        pull = (held ? 0.0f : -ratio * A) - a.kl_coef * em;
    }
};

__device__ int64_t action_of(const wc_policy_loss_args& a, int64_t t) {
    return a.action_bytes == 8 ? static_cast<const int64_t*>(a.actions)[t]
                               : (int64_t) static_cast<const int32_t*>(a.actions)[t];
}

template <class T>
__global__ void __launch_bounds__(THREADS) k_policy_rows(wc_policy_loss_args a, float* part) {
    __shared__ Run sr[THREADS / 32];
    const int64_t V = a.width;
    float total = 0.0f;
    for (int64_t t = blockIdx.x; t < a.rows; t += gridDim.x) {
        const T* z = static_cast<const T*>(a.logits) + t * a.ld_logits;
        const uint8_t* legal = a.legal ? a.legal + t * a.ld_legal : nullptr;
        T* dz = a.dlogits ? static_cast<T*>(a.dlogits) + t * a.ld_dlogits : nullptr;
        const float w = a.weights ? a.weights[t] : 1.0f;
        const int64_t act = action_of(a, t);
        const bool live = w != 0.0f && act >= 0 && act < V && (!legal || legal[act]) && to_f(z[act]) != -INFINITY;
        if (!live) {
            if (dz)
                for (int64_t j = threadIdx.x; j < V; j += THREADS) dz[j] = from_f<T>(0.0f);
            if (threadIdx.x < 4) a.row_out[threadIdx.x * a.rows + t] = 0.0f;
            continue;
        }
        Run r{-INFINITY, 0.0f, 0.0f};
        bool bad = false;
        for (int64_t j = threadIdx.x; j < V; j += THREADS) {
            if (legal && !legal[j]) continue;
            const float x = to_f(z[j]) * LOG2E;
            bad |= isnan(x) || x == INFINITY;
            if (x != -INFINITY && !isnan(x)) r.add(x);
        }
        for (int o = 16; o; o >>= 1)
            r.join(Run{__shfl_xor_sync(~0u, r.m, o), __shfl_xor_sync(~0u, r.s, o), __shfl_xor_sync(~0u, r.w, o)});
        if ((threadIdx.x & 31) == 0) sr[threadIdx.x >> 5] = r;
        bad = __syncthreads_or(bad);
        r = sr[0];
        for (int i = 1; i < THREADS / 32; ++i) r.join(sr[i]);
        __syncthreads();
        if (bad) r.s = r.w = __uint_as_float(0x7fffffffu);
        const float logs = log2f(r.s), l = (fmaf(to_f(z[act]), LOG2E, -r.m) - logs) * LN2;
        const float H = (logs - r.w / r.s) * LN2;
        const RowLoss q(l, H, a.old_logp[t], a.advantages[t], a.ref_logp != nullptr, a.ref_logp ? a.ref_logp[t] : 0.0f, a);
        if (threadIdx.x == 0) {
            a.row_out[t] = q.row, a.row_out[a.rows + t] = l;
            a.row_out[2 * a.rows + t] = H, a.row_out[3 * a.rows + t] = q.kl;
            total += w * q.row;
        }
        if (!dz) continue;
        const float up = (a.upstream ? *a.upstream : 1.0f) * w, g = up * q.pull, ce = up * a.entropy_coef, inv = 1.0f / r.s;
        for (int64_t j = threadIdx.x; j < V; j += THREADS) {
            float d = 0.0f;
            if ((!legal || legal[j]) && to_f(z[j]) != -INFINITY) {
                const float x = fmaf(to_f(z[j]), LOG2E, -r.m), p = exp2f(x) * inv;
                d = p * (ce * fmaf(x - logs, LN2, H) - g);
                if (j == act) d += g;
            }
            dz[j] = from_f<T>(d);
        }
    }
    if (threadIdx.x == 0) part[blockIdx.x] = total;
}

__global__ void k_policy_total(const float* part, int n, float* loss) {
    float v = 0.0f;
    for (int i = threadIdx.x; i < n; i += 32) v += part[i];
    v = warp_sum(v);
    if (threadIdx.x == 0) *loss = v;
}

int policy_ctas(int64_t rows) { return rows < 148 * 8 ? (int)(rows ? rows : 1) : 148 * 8; }

}  // namespace

uint64_t policy_loss_workspace(int64_t rows, int64_t) { return (uint64_t)policy_ctas(rows) * sizeof(float); }

void launch_policy_loss(const wc_policy_loss_args& a, cudaStream_t s) {
    float* part = static_cast<float*>(a.workspace);
    const int n = policy_ctas(a.rows);
    if (a.type == WC_F32) k_policy_rows<float><<<n, THREADS, 0, s>>>(a, part);
    else if (a.type == WC_F16) k_policy_rows<__half><<<n, THREADS, 0, s>>>(a, part);
    else k_policy_rows<__nv_bfloat16><<<n, THREADS, 0, s>>>(a, part);
    k_policy_total<<<1, 32, 0, s>>>(part, n, a.loss);
}

}  // namespace wctrain
