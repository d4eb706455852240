// The clipped policy loss with a KL term, and its gradient at the logits, in
// one pass over the logits.
//
// With m the row's maximum, e_j = exp(z_j - m) and S = sum e_j:
//   l = (z_a - m) - ln S,  H = ln S - sum e_j (z_j - m) / S,  p_j = e_j / S.
// The row's loss depends on the logits through l and H only, so
//   dloss/dz_j = g (delta_ja - p_j) + w c p_j (ln p_j + H),
//   g = w (-ratio A [not clipped] - kl_coef (exp(r - l) - 1)).
// Powers are taken in base 2, 2^(z_j log2 e - c) with c = m log2 e rounded; the
// factor that the rounding of c puts on every e_j is taken out of ln S again.
//
// What bounds it is the bytes: each logit is read once and its gradient written
// once. A row stays in registers as it was loaded (16 bytes of logits and their
// legal bytes a chunk): a part of a warp for the narrowest rows, then a warp, a
// CTA, and for long rows a cluster of CTAs, which exchange (m, S, sum) through
// distributed shared memory. Rows that no cluster can hold, and rows whose
// stride or address keeps 16-byte loads off them, are read twice by one CTA
// (the second time mostly from L2).
#include <cooperative_groups.h>

#include <algorithm>
#include <type_traits>

#include "train.cuh"

namespace cg = cooperative_groups;

namespace wctrain {

namespace {

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// What a row needs besides its logits
struct RowIn {
    float w;
    int64_t act;
};
__device__ __forceinline__ RowIn row_in(const wc_policy_loss_args& a, int64_t t) {
    RowIn r;
    r.w = a.weights ? a.weights[t] : 1.0f;
    r.act = a.action_bytes == 8 ? static_cast<const int64_t*>(a.actions)[t] : (int64_t) static_cast<const int32_t*>(a.actions)[t];
    return r;
}

// A row's loss from its parts (m the maximum of all, S and W sums over all
// relative to it) and the logit of its action.
struct Row {
    float loss, l, H, kl;   // results
    float c, inv, g, ce, lH; // gradient: p = 2^(z log2 e - c) inv;  d = p (ce (ln p + H) - g) + [action] g
    __device__ __forceinline__ Row(const wc_policy_loss_args& a, int64_t t, float w, float m, float S, float W, float za) {
        c = m * LOG2E;
        const float off = fmaf(m, LOG2E, -c) * LN2;  // ln S = ln(sum of the rounded powers) - off
        const float lnS = logf(S) - off;
        l = (za - m) - lnS;
        H = lnS - W / S * LN2 + off;  // W counts from c as well
        const float A = a.advantages[t], lo = 1.0f - a.clip_low, hi = 1.0f + a.clip_high;
        const float ratio = expf(l - a.old_logp[t]);
        const float free = ratio * A, clipped = fminf(fmaxf(ratio, lo), hi) * A;
        const bool held = (A > 0.0f && ratio > hi) || (A < 0.0f && ratio < lo);
        const float d = a.ref_logp ? a.ref_logp[t] - l : 0.0f, em = a.ref_logp ? expm1f(d) : 0.0f;
        kl = em - d;
        loss = -(free < clipped || isnan(free) ? free : clipped) + a.kl_coef * kl - a.entropy_coef * H;
        const float up = (a.upstream ? *a.upstream : 1.0f) * w;
        g = up * ((held ? 0.0f : -free) - a.kl_coef * em);
        ce = up * a.entropy_coef;
        inv = 1.0f / S;
        lH = H - lnS - off;  // ln p + H = (z log2 e - c) ln 2 + lH
    }
    __device__ __forceinline__ void put(const wc_policy_loss_args& a, int64_t t) const {
        a.row_out[t] = loss, a.row_out[a.rows + t] = l, a.row_out[2 * a.rows + t] = H, a.row_out[3 * a.rows + t] = kl;
    }
    __device__ __forceinline__ float grad(float z) const {
        const float x = fmaf(z, LOG2E, -c), p = ex2(x) * inv;
        return p * (ce != 0.0f ? fmaf(ce, fmaf(x, LN2, lH), -g) : -g);
    }
};
__device__ __forceinline__ void put_void(const wc_policy_loss_args& a, int64_t t) {
    a.row_out[t] = 0.0f, a.row_out[a.rows + t] = 0.0f, a.row_out[2 * a.rows + t] = 0.0f, a.row_out[3 * a.rows + t] = 0.0f;
}

// 16 bytes of logits, and their legal bytes where the call has such
template <class T, bool MASK>
struct Chunk {
    static constexpr int N = 16 / sizeof(T);
    uint4 z;
    uint2 legal;
    __device__ __forceinline__ void load(const T* row, const uint8_t* mask, int64_t at) {
        z = __ldcs(reinterpret_cast<const uint4*>(row + at));
        if constexpr (MASK && N == 8) legal = __ldcs(reinterpret_cast<const uint2*>(mask + at));
        if constexpr (MASK && N == 4) legal.x = __ldcs(reinterpret_cast<const unsigned int*>(mask + at));
    }
    // entries that do not count
    __device__ __forceinline__ void none() {
        const uint32_t inf = sizeof(T) == 4 ? 0xff800000u : std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;
        z = make_uint4(inf, inf, inf, inf), legal = make_uint2(0, 0);
    }
    __device__ __forceinline__ void get(float* v) const {
        alignas(16) T e[N];
        *reinterpret_cast<uint4*>(e) = z;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            v[i] = to_f(e[i]);
            if (MASK && !((i < 4 ? legal.x : legal.y) >> (8 * (i & 3)) & 0xffu)) v[i] = -INFINITY;
        }
    }
};

template <class C, int NV>
__device__ __forceinline__ float local_max(const C* q) {
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        float v[C::N];
        q[i].get(v);
#pragma unroll
        for (int k = 0; k < C::N; ++k) m = fmaxf(m, v[k]);
    }
    return m;
}
// One entry's share of the sums from c on. A NaN, and +inf (inf - inf), reach s; an entry that does not count has
// x = -inf and e = 0.
__device__ __forceinline__ void add_entry(float v, float c, float& s, float& w) {
    const float x = fmaf(v, LOG2E, -c), e = ex2(x);
    s += e;
    w = fmaf(e, fmaxf(x, -1000.0f), w);
}
template <class C, int NV>
__device__ __forceinline__ float2 local_sums(const C* q, float m) {
    const float c = m * LOG2E;
    float s = 0.0f, w = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        float v[C::N];
        q[i].get(v);
#pragma unroll
        for (int k = 0; k < C::N; ++k) add_entry(v[k], c, s, w);
    }
    return make_float2(s, w);
}
template <class C, int NV, class T>
__device__ __forceinline__ void local_grad(const C* q, const Row& r, T* out, int first, int step, int width, int act) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int at = first + i * step;
        if (at >= width) break;
        float v[C::N];
        q[i].get(v);
#pragma unroll
        for (int k = 0; k < C::N; ++k) v[k] = v[k] == -INFINITY ? 0.0f : r.grad(v[k]);
        if ((unsigned)(act - at) < (unsigned)C::N)
#pragma unroll
            for (int k = 0; k < C::N; ++k)
                if (at + k == act) v[k] += r.g;
        alignas(16) T e[C::N];
#pragma unroll
        for (int k = 0; k < C::N; ++k) e[k] = from_f<T>(v[k]);
        __stcs(reinterpret_cast<uint4*>(out + at), *reinterpret_cast<const uint4*>(e));
    }
}
// Parts of a row (each relative to its own maximum) joined, in order
__device__ __forceinline__ void join(const float* pm, const float* ps, const float* pw, int n, float& M, float& S, float& W) {
    M = -INFINITY;
    for (int i = 0; i < n; ++i) M = fmaxf(M, pm[i]);
    S = W = 0.0f;
    const float C = M * LOG2E;
    for (int i = 0; i < n; ++i) {
        const bool none = pm[i] == -INFINITY;
        const float d = none ? 0.0f : pm[i] * LOG2E - C, f = none ? 0.0f : ex2(d);
        S = fmaf(ps[i], f, S);
        W = fmaf(fmaf(ps[i], d, pw[i]), f, W);
    }
}

// Rows of up to 32 NV chunks: `lanes` threads of a warp a row (a power of two).
template <class T, bool MASK, int NV>
__global__ void __launch_bounds__(256) k_policy_warp(wc_policy_loss_args a, int lanes, double* part) {
    using C = Chunk<T, MASK>;
    __shared__ double s[8];
    const int lane = threadIdx.x & 31, at = lane & (lanes - 1), per = 256 / lanes, width = (int)a.width;
    double total = 0.0;
    for (int64_t t0 = (int64_t)blockIdx.x * per; t0 < a.rows; t0 += (int64_t)gridDim.x * per) {
        const int64_t t = t0 + threadIdx.x / lanes;
        const bool in = t < a.rows;
        const T* z = static_cast<const T*>(a.logits) + (in ? t : 0) * a.ld_logits;
        const uint8_t* legal = MASK ? a.legal + (in ? t : 0) * a.ld_legal : nullptr;
        RowIn r{0.0f, -1};
        if (in) r = row_in(a, t);
        bool live = r.w != 0.0f && r.act >= 0 && r.act < width;
        C q[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * lanes + at) * C::N;
            if (live && c < width) q[i].load(z, legal, c);
            else q[i].none();
        }
        float za = -INFINITY;
        if (live && (!MASK || legal[r.act])) za = to_f(z[r.act]);
        live = live && za != -INFINITY;
        float m = local_max<C, NV>(q);
        for (int o = lanes >> 1; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
        float2 sw = local_sums<C, NV>(q, live ? m : 0.0f);
        for (int o = lanes >> 1; o; o >>= 1) sw.x += __shfl_xor_sync(~0u, sw.x, o), sw.y += __shfl_xor_sync(~0u, sw.y, o);
        if (!in) continue;
        T* out = a.dlogits ? static_cast<T*>(a.dlogits) + t * a.ld_dlogits : nullptr;
        if (live) {
            const Row row(a, t, r.w, m, sw.x, sw.y, za);
            if (at == 0) row.put(a, t), total += (double)(r.w * row.loss);
            if (out) local_grad<C, NV>(q, row, out, at * C::N, lanes * C::N, width, (int)r.act);
        } else {
            if (at == 0) put_void(a, t);
            if (out)
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    const int c = (i * lanes + at) * C::N;
                    if (c < width) __stcs(reinterpret_cast<uint4*>(out + c), make_uint4(0, 0, 0, 0));
                }
        }
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) total += __shfl_xor_sync(~0u, total, o);
    if (lane == 0) s[threadIdx.x >> 5] = total;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < 8; ++i) total += s[i];
        part[blockIdx.x] = total;
    }
}

// Longer rows: one CTA, or the CTAs of a cluster, a row. Warps, then the CTAs
// of the cluster, join their parts through shared memory; every thread joins
// them in the same order.
template <class T, bool MASK, int NV, int THREADS>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS) k_policy_cluster(wc_policy_loss_args a, int ctas, double* part) {
    using C = Chunk<T, MASK>;
    constexpr int WARPS = THREADS / 32;
    __shared__ float sm[WARPS], ss[WARPS], sw[WARPS];
    __shared__ float cm[2][8], cs[2][8], cw[2][8];  // the cluster's, two rows in turn
    cg::cluster_group cluster = cg::this_cluster();
    const int rank = ctas > 1 ? (int)cluster.block_rank() : 0, width = (int)a.width;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int step = ctas * THREADS * C::N, first = (rank * THREADS + (int)threadIdx.x) * C::N;
    double total = 0.0;
    int turn = 0;
    for (int64_t t = blockIdx.x / ctas; t < a.rows; t += gridDim.x / ctas) {
        const T* z = static_cast<const T*>(a.logits) + t * a.ld_logits;
        const uint8_t* legal = MASK ? a.legal + t * a.ld_legal : nullptr;
        T* out = a.dlogits ? static_cast<T*>(a.dlogits) + t * a.ld_dlogits : nullptr;
        const RowIn r = row_in(a, t);
        C q[NV];
        const bool read = r.w != 0.0f && r.act >= 0 && r.act < width;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if (read && first + i * step < width) q[i].load(z, legal, first + i * step);
            else q[i].none();
        }
        float za = -INFINITY;
        if (read && (!MASK || legal[r.act])) za = to_f(z[r.act]);
        if (za == -INFINITY) {  // void, for every thread of the cluster
            if (out)
#pragma unroll
                for (int i = 0; i < NV; ++i)
                    if (first + i * step < width) __stcs(reinterpret_cast<uint4*>(out + first + i * step), make_uint4(0, 0, 0, 0));
            if (rank == 0 && threadIdx.x == 0) put_void(a, t);
            continue;
        }
        float m = local_max<C, NV>(q);
#pragma unroll
        for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
        float2 v = local_sums<C, NV>(q, m == -INFINITY ? 0.0f : m);
        v.x = warp_sum(v.x), v.y = warp_sum(v.y);
        __syncthreads();  // the last row's parts have been read
        if (lane == 0) sm[warp] = m, ss[warp] = v.x, sw[warp] = v.y;
        __syncthreads();
        float M, S, W;
        join(sm, ss, sw, WARPS, M, S, W);
        if (ctas > 1) {
            if (threadIdx.x < ctas) {
                cluster.map_shared_rank(cm[turn], threadIdx.x)[rank] = M;
                cluster.map_shared_rank(cs[turn], threadIdx.x)[rank] = S;
                cluster.map_shared_rank(cw[turn], threadIdx.x)[rank] = W;
            }
            cluster.sync();
            join(cm[turn], cs[turn], cw[turn], ctas, M, S, W);
            turn ^= 1;
        }
        const Row row(a, t, r.w, M, S, W, za);
        if (rank == 0 && threadIdx.x == 0) row.put(a, t), total += (double)(r.w * row.loss);
        if (out) local_grad<C, NV>(q, row, out, first, step, width, (int)r.act);
    }
    if (rank == 0 && threadIdx.x == 0) part[blockIdx.x / ctas] = total;
    if (ctas > 1) cluster.sync();  // no CTA leaves while another may still write to it
}

// Any row: one CTA reads it twice, an entry at a time.
template <class T>
__global__ void __launch_bounds__(512) k_policy_long(wc_policy_loss_args a, double* part) {
    __shared__ float sm[16], ss[16], sw[16];
    const int64_t V = a.width;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    double total = 0.0;
    for (int64_t t = blockIdx.x; t < a.rows; t += gridDim.x) {
        const T* z = static_cast<const T*>(a.logits) + t * a.ld_logits;
        const uint8_t* legal = a.legal ? a.legal + t * a.ld_legal : nullptr;
        T* out = a.dlogits ? static_cast<T*>(a.dlogits) + t * a.ld_dlogits : nullptr;
        const RowIn r = row_in(a, t);
        float za = -INFINITY;
        if (r.w != 0.0f && r.act >= 0 && r.act < V && (!legal || legal[r.act])) za = to_f(z[r.act]);
        if (za == -INFINITY) {
            if (out)
                for (int64_t j = threadIdx.x; j < V; j += 512) out[j] = from_f<T>(0.0f);
            if (threadIdx.x == 0) put_void(a, t);
            continue;
        }
        // eight entries at a time: their maximum moves the running one, then their powers are added
        float m = -INFINITY, s = 0.0f, w = 0.0f;
        for (int64_t j = threadIdx.x; j < V; j += 8 * 512) {
            float v[8], top = m;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const int64_t i = j + k * 512;
                v[k] = i < V && (!legal || legal[i]) ? to_f(z[i]) : -INFINITY;
                top = fmaxf(top, v[k]);
            }
            const float c = top == -INFINITY ? 0.0f : top * LOG2E, d = m == -INFINITY ? 0.0f : m * LOG2E - c, f = ex2(d);
            w = fmaf(s, d, w) * f, s *= f, m = top;
#pragma unroll
            for (int k = 0; k < 8; ++k) add_entry(v[k], c, s, w);
        }
        float top = m;
#pragma unroll
        for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
        const float d = m == -INFINITY ? 0.0f : m * LOG2E - top * LOG2E, f = m == -INFINITY ? 0.0f : ex2(d);
        w = warp_sum(fmaf(s, d, w) * f), s = warp_sum(s * f);
        __syncthreads();
        if (lane == 0) sm[warp] = top, ss[warp] = s, sw[warp] = w;
        __syncthreads();
        float M, S, W;
        join(sm, ss, sw, 16, M, S, W);
        const Row row(a, t, r.w, M, S, W, za);
        if (threadIdx.x == 0) row.put(a, t), total += (double)(r.w * row.loss);
        if (out)
            for (int64_t j = threadIdx.x; j < V; j += 512) {
                const float v = !legal || legal[j] ? to_f(z[j]) : -INFINITY;
                float d = v == -INFINITY ? 0.0f : row.grad(v);
                if (j == r.act) d += row.g;
                out[j] = from_f<T>(d);
            }
    }
    if (threadIdx.x == 0) part[blockIdx.x] = total;
}

// the CTAs' totals, in order
__global__ void k_policy_total(const double* part, int n, float* loss) {
    double v = 0.0;
    for (int i = threadIdx.x; i < n; i += 32) v += part[i];
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
    if (threadIdx.x == 0) *loss = (float)v;
}

constexpr int MOST_CTAS = 148 * 8;

template <class T, bool MASK>
int launch_vec(const wc_policy_loss_args& a, double* part, cudaStream_t s) {
    constexpr int N = Chunk<T, MASK>::N;
    const int64_t chunks = a.width / N;
    if (chunks <= 32 * 4) {
        int lanes = 1;
        while (lanes < 32 && lanes * 4 < chunks) lanes *= 2;
        const int64_t per = 256 / lanes;
        const int n = (int)std::min<int64_t>(MOST_CTAS, (a.rows + per - 1) / per);
        const int nv = (int)((chunks + lanes - 1) / lanes);
        if (nv <= 1) k_policy_warp<T, MASK, 1><<<n, 256, 0, s>>>(a, lanes, part);
        else if (nv == 2) k_policy_warp<T, MASK, 2><<<n, 256, 0, s>>>(a, lanes, part);
        else if (nv == 3) k_policy_warp<T, MASK, 3><<<n, 256, 0, s>>>(a, lanes, part);
        else k_policy_warp<T, MASK, 4><<<n, 256, 0, s>>>(a, lanes, part);
        return n;
    }
    // 4 chunks a thread, up to 8 CTAs a row
    int ctas = 1;
    while (ctas < 8 && (int64_t)ctas * 512 * 4 < chunks) ctas *= 2;
    const int n = (int)std::min<int64_t>(MOST_CTAS / ctas, a.rows);
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim = {(unsigned)ctas, 1, 1};
    cfg.gridDim = n * ctas, cfg.stream = s, cfg.attrs = &attr, cfg.numAttrs = 1;
    cfg.blockDim = chunks <= 128 * 4 ? 128 : 512;
    if (chunks <= 128 * 4) cudaLaunchKernelEx(&cfg, k_policy_cluster<T, MASK, 4, 128>, a, ctas, part);
    else cudaLaunchKernelEx(&cfg, k_policy_cluster<T, MASK, 4, 512>, a, ctas, part);
    return n;
}

template <class T>
int launch_type(const wc_policy_loss_args& a, double* part, cudaStream_t s) {
    constexpr int N = 16 / sizeof(T);
    const auto fits = [&](const void* p, int64_t ld, size_t e) { return ((uintptr_t)p & 15) == 0 && (ld * e) % 16 == 0; };
    const bool vec = a.width % N == 0 && fits(a.logits, a.ld_logits, sizeof(T)) &&
                     (!a.dlogits || fits(a.dlogits, a.ld_dlogits, sizeof(T))) &&
                     (!a.legal || (((uintptr_t)a.legal & 7) == 0 && a.ld_legal % 8 == 0));
    if (vec && a.width / N <= 8 * 512 * 4) return a.legal ? launch_vec<T, true>(a, part, s) : launch_vec<T, false>(a, part, s);
    const int n = (int)std::min<int64_t>(148 * 4, a.rows);
    k_policy_long<T><<<n, 512, 0, s>>>(a, part);
    return n;
}

}  // namespace

uint64_t policy_loss_workspace(int64_t, int64_t) { return MOST_CTAS * sizeof(double); }

void launch_policy_loss(const wc_policy_loss_args& a, cudaStream_t s) {
    double* part = static_cast<double*>(a.workspace);
    int n = 0;
    if (a.rows) n = a.type == WC_F32   ? launch_type<float>(a, part, s)
                    : a.type == WC_F16 ? launch_type<__half>(a, part, s)
                                       : launch_type<__nv_bfloat16>(a, part, s);
    k_policy_total<<<1, 32, 0, s>>>(part, n, a.loss);
}

}  // namespace wctrain
