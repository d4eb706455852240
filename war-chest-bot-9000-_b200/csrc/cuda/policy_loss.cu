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
#include "umma.cuh"

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
    // the gradient at an entry other than the action
    __device__ __forceinline__ float grad(float z) const {
        const float x = fmaf(z, LOG2E, -c), p = ex2(x) * inv;
        return ce != 0.0f ? p * fmaf(ce, fmaf(fmaxf(x, -1000.0f), LN2, lH), -g) : p * -g;
    }
};
__device__ __forceinline__ void put_void(const wc_policy_loss_args& a, int64_t t) {
    a.row_out[t] = 0.0f, a.row_out[a.rows + t] = 0.0f, a.row_out[2 * a.rows + t] = 0.0f, a.row_out[3 * a.rows + t] = 0.0f;
}

using umma::f2;
using umma::f2_add;
using umma::f2_fma;
__device__ __forceinline__ unsigned long long f2_mul(unsigned long long a, unsigned long long b) {
    unsigned long long d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}

// 16 bytes of logits as they lie in memory, what does not count as -inf
template <class T>
struct Chunk {
    static constexpr int N = 16 / sizeof(T);
    static constexpr uint32_t INF = sizeof(T) == 4 ? 0xff800000u : std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;
    uint32_t z[4];
    __device__ __forceinline__ void load(const T* at) { *reinterpret_cast<uint4*>(z) = __ldcs(reinterpret_cast<const uint4*>(at)); }
    __device__ __forceinline__ void none() { z[0] = z[1] = z[2] = z[3] = INF; }
    // legal bytes, in the order of the entries
    __device__ __forceinline__ void mask(uint2 legal) {
        const uint32_t off[2] = {__vcmpeq4(legal.x, 0), __vcmpeq4(legal.y, 0)};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t m = N == 8 ? __byte_perm(off[i >> 1], 0, i & 1 ? 0x3322 : 0x1100) : __byte_perm(off[0], 0, 0x1111 * i);
            z[i] = (z[i] & ~m) | (INF & m);
        }
    }
    __device__ __forceinline__ static uint2 load_legal(const uint8_t* at) {
        if constexpr (N == 8) return __ldcs(reinterpret_cast<const uint2*>(at));
        return make_uint2(__ldcs(reinterpret_cast<const unsigned int*>(at)), 0);
    }
    // entries 2 i and 2 i + 1
    __device__ __forceinline__ float2 pair(int i) const {
        if constexpr (sizeof(T) == 4) return make_float2(__uint_as_float(z[2 * i]), __uint_as_float(z[2 * i + 1]));
        else if constexpr (std::is_same<T, __half>::value) return __half22float2(*reinterpret_cast<const __half2*>(&z[i]));
        else return make_float2(__uint_as_float(z[i] << 16), __uint_as_float(z[i] & 0xffff0000u));
    }
};

template <class T, int NV>
__device__ __forceinline__ float local_max(const Chunk<T>* q) {
    if constexpr (sizeof(T) == 4) {
        float m = -INFINITY;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int k = 0; k < 4; ++k) m = fmaxf(m, __uint_as_float(q[i].z[k]));
        return m;
    } else {
        using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
        T2 m = *reinterpret_cast<const T2*>(&q[0].z[0]);
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int k = 0; k < 4; ++k) m = __hmax2(m, *reinterpret_cast<const T2*>(&q[i].z[k]));
        return fmaxf(to_f(m.x), to_f(m.y));
    }
}
// One entry's share of the sums from c on. A NaN, and +inf (inf - inf), reach s; an entry that does not count has
// x = -inf and e = 0.
__device__ __forceinline__ void add_entry(float v, float c, float& s, float& w) {
    const float x = fmaf(v, LOG2E, -c), e = ex2(x);
    s += e;
    w = fmaf(e, fmaxf(x, -1000.0f), w);
}
template <class T, int NV>
__device__ __forceinline__ float2 local_sums(const Chunk<T>* q, float m) {
    const float c = m * LOG2E;
    const unsigned long long L = f2(LOG2E, LOG2E), C = f2(-c, -c);
    unsigned long long s = 0, w = 0;  // pairs of zeros
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int k = 0; k < Chunk<T>::N / 2; ++k) {  // add_entry for two
            const float2 v = q[i].pair(k);
            const unsigned long long x = f2_fma(f2(v.x, v.y), L, C);
            const float x0 = umma::f2_lo(x), x1 = umma::f2_hi(x);
            const unsigned long long e = f2(ex2(x0), ex2(x1));
            s = f2_add(s, e);
            w = f2_fma(e, f2(fmaxf(x0, -1000.0f), fmaxf(x1, -1000.0f)), w);
        }
    return make_float2(umma::f2_lo(s) + umma::f2_hi(s), umma::f2_lo(w) + umma::f2_hi(w));
}
template <class T, int NV>
__device__ __forceinline__ void local_grad(const Chunk<T>* q, const Row& r, T* out, int first, int step, int width, int act) {
    const unsigned long long L = f2(LOG2E, LOG2E), C = f2(-r.c, -r.c);
    const bool entropy = r.ce != 0.0f;
    const float f = -r.g * r.inv;  // p times -g
    const unsigned long long F = f2(f, f), E = f2(r.ce * LN2 * r.inv, r.ce * LN2 * r.inv), K = f2(fmaf(r.ce, r.lH, -r.g) * r.inv, fmaf(r.ce, r.lH, -r.g) * r.inv);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int at = first + i * step;
        if (at >= width) break;
        float v[Chunk<T>::N];
#pragma unroll
        for (int k = 0; k < Chunk<T>::N / 2; ++k) {
            const float2 z = q[i].pair(k);
            const unsigned long long x = f2_fma(f2(z.x, z.y), L, C);
            const float x0 = umma::f2_lo(x), x1 = umma::f2_hi(x);
            const unsigned long long e = f2(ex2(x0), ex2(x1));
            // e inv (ce (x ln 2 + lH) - g)
            const unsigned long long d = f2_mul(e, entropy ? f2_fma(f2(fmaxf(x0, -1000.0f), fmaxf(x1, -1000.0f)), E, K) : F);
            v[2 * k] = umma::f2_lo(d), v[2 * k + 1] = umma::f2_hi(d);
        }
        if ((unsigned)(act - at) < (unsigned)Chunk<T>::N)
#pragma unroll
            for (int k = 0; k < Chunk<T>::N; ++k)
                if (at + k == act) v[k] += r.g;
        alignas(16) T e[Chunk<T>::N];
#pragma unroll
        for (int k = 0; k < Chunk<T>::N; ++k) e[k] = from_f<T>(v[k]);
        __stcs(reinterpret_cast<uint4*>(out + at), *reinterpret_cast<const uint4*>(e));
    }
}
// A row's logits in registers: NV chunks, `step` entries apart
template <class T, bool MASK, int NV>
__device__ __forceinline__ void load_row(Chunk<T>* q, const T* z, const uint8_t* legal, bool read, int first, int step, int width) {
    uint2 on[MASK ? NV : 1];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int at = first + i * step;
        if (read && at < width) {
            q[i].load(z + at);
            if constexpr (MASK) on[i] = Chunk<T>::load_legal(legal + at);
        } else {
            q[i].none();
            if constexpr (MASK) on[i] = make_uint2(0, 0);
        }
    }
    if constexpr (MASK)
#pragma unroll
        for (int i = 0; i < NV; ++i) q[i].mask(on[i]);
}
// Parts of a row (m, s, w: sums relative to the part's own maximum), up to 4 a lane, joined over the warp.
template <int EACH>
__device__ __forceinline__ void join(const float4* parts, int n, float& M, float& S, float& W) {
    const int lane = threadIdx.x & 31;
    float4 p[EACH];
    M = -INFINITY;
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
        p[i] = lane + 32 * i < n ? parts[lane + 32 * i] : make_float4(-INFINITY, 0.0f, 0.0f, 0.0f);
        M = fmaxf(M, p[i].x);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) M = fmaxf(M, __shfl_xor_sync(~0u, M, o));
    S = W = 0.0f;
    const float C = M * LOG2E;
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
        const bool none = p[i].x == -INFINITY;
        const float d = none ? 0.0f : p[i].x * LOG2E - C, f = none ? 0.0f : ex2(d);
        S = fmaf(p[i].y, f, S);
        W = fmaf(fmaf(p[i].y, d, p[i].z), f, W);
    }
    S = warp_sum(S), W = warp_sum(W);
}

// Rows of up to 32 NV chunks: `lanes` threads of a warp a row (a power of two).
template <class T, bool MASK, int NV>
__global__ void __launch_bounds__(256) k_policy_warp(wc_policy_loss_args a, int lanes, double* part) {
    constexpr int N = Chunk<T>::N;
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
        Chunk<T> q[NV];
        load_row<T, MASK, NV>(q, z, legal, live, at * N, lanes * N, width);
        float za = -INFINITY;
        if (live && (!MASK || legal[r.act])) za = to_f(z[r.act]);
        live = live && za != -INFINITY;
        float m = local_max<T, NV>(q);
        for (int o = lanes >> 1; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
        float2 sw = local_sums<T, NV>(q, live ? m : 0.0f);
        for (int o = lanes >> 1; o; o >>= 1) sw.x += __shfl_xor_sync(~0u, sw.x, o), sw.y += __shfl_xor_sync(~0u, sw.y, o);
        if (!in) continue;
        T* out = a.dlogits ? static_cast<T*>(a.dlogits) + t * a.ld_dlogits : nullptr;
        if (live) {
            const Row row(a, t, r.w, m, sw.x, sw.y, za);
            if (at == 0) row.put(a, t), total += (double)(r.w * row.loss);
            if (out) local_grad<T, NV>(q, row, out, at * N, lanes * N, width, (int)r.act);
        } else {
            if (at == 0) put_void(a, t);
            if (out)
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    const int c = (i * lanes + at) * N;
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
template <class T, bool MASK, int NV, int THREADS, int CTAS>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS) k_policy_cluster(wc_policy_loss_args a, double* part) {
    constexpr int N = Chunk<T>::N, WARPS = THREADS / 32;
    __shared__ float4 parts[2][CTAS * WARPS];  // of every warp of the cluster, two rows in turn
    cg::cluster_group cluster = cg::this_cluster();
    const int rank = CTAS > 1 ? (int)cluster.block_rank() : 0, width = (int)a.width;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int step = CTAS * THREADS * N, first = (rank * THREADS + (int)threadIdx.x) * N;
    double total = 0.0;
    int turn = 0;
    for (int64_t t = blockIdx.x / CTAS; t < a.rows; t += gridDim.x / CTAS) {
        const T* z = static_cast<const T*>(a.logits) + t * a.ld_logits;
        const uint8_t* legal = MASK ? a.legal + t * a.ld_legal : nullptr;
        T* out = a.dlogits ? static_cast<T*>(a.dlogits) + t * a.ld_dlogits : nullptr;
        const RowIn r = row_in(a, t);
        Chunk<T> q[NV];
        const bool read = r.w != 0.0f && r.act >= 0 && r.act < width;
        load_row<T, MASK, NV>(q, z, legal, read, first, step, width);
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
        float m = local_max<T, NV>(q);
#pragma unroll
        for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
        float2 v = local_sums<T, NV>(q, m == -INFINITY ? 0.0f : m);
        v.x = warp_sum(v.x), v.y = warp_sum(v.y);
        // to every CTA of the cluster; what they read of the row before last they have read before the last barrier
        if (lane < CTAS) {
            float4* to = CTAS > 1 ? cluster.map_shared_rank(parts[turn], lane) : parts[turn];
            to[rank * WARPS + warp] = make_float4(m, v.x, v.y, 0.0f);
        }
        if (CTAS > 1) cluster.sync();
        else __syncthreads();
        float M, S, W;
        join<(CTAS * WARPS + 31) / 32>(parts[turn], CTAS * WARPS, M, S, W);
        turn ^= 1;
        const Row row(a, t, r.w, M, S, W, za);
        if (rank == 0 && threadIdx.x == 0) row.put(a, t), total += (double)(r.w * row.loss);
        if (out) local_grad<T, NV>(q, row, out, first, step, width, (int)r.act);
    }
    if (rank == 0 && threadIdx.x == 0) part[blockIdx.x / CTAS] = total;
    if (CTAS > 1) cluster.sync();  // no CTA leaves while another may still write to it
}

// Any row: one CTA reads it twice, an entry at a time.
template <class T>
__global__ void __launch_bounds__(512) k_policy_long(wc_policy_loss_args a, double* part) {
    __shared__ float4 parts[16];
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
        __syncthreads();  // the last row's parts have been read
        if (lane == 0) parts[warp] = make_float4(top, s, w, 0.0f);
        __syncthreads();
        float M, S, W;
        join<1>(parts, 16, M, S, W);
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

template <class T, bool MASK, int THREADS, int CTAS>
int launch_cluster(const wc_policy_loss_args& a, double* part, cudaStream_t s) {
    const int n = (int)std::min<int64_t>(148 * 1024 / THREADS / CTAS, a.rows);  // what is resident
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim = {CTAS, 1, 1};
    cfg.gridDim = n * CTAS, cfg.blockDim = THREADS, cfg.stream = s, cfg.attrs = &attr, cfg.numAttrs = 1;
    cudaLaunchKernelEx(&cfg, k_policy_cluster<T, MASK, 4, THREADS, CTAS>, a, part);
    return n;
}

template <class T, bool MASK>
int launch_vec(const wc_policy_loss_args& a, double* part, cudaStream_t s) {
    constexpr int N = Chunk<T>::N;
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
    if (chunks <= 128 * 4) return launch_cluster<T, MASK, 128, 1>(a, part, s);
    if (chunks <= 512 * 4) return launch_cluster<T, MASK, 512, 1>(a, part, s);
    if (chunks <= 512 * 8) return launch_cluster<T, MASK, 512, 2>(a, part, s);
    if (chunks <= 512 * 16) return launch_cluster<T, MASK, 512, 4>(a, part, s);
    return launch_cluster<T, MASK, 512, 8>(a, part, s);
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
