// The clipped policy loss with a KL term, and its gradient at the logits, in
// one pass over the logits.
//
// With m the row's maximum, e_j = exp(z_j - m) and S = sum e_j:
//   l = (z_a - m) - ln S,  H = ln S - sum e_j (z_j - m) / S,  p_j = e_j / S.
// The row's loss depends on the logits through l and H only, so
//   dloss/dz_j = g (delta_ja - p_j) + w c p_j (ln p_j + H),
//   g = w (-ratio A [not clipped] - kl_coef (exp(r - l) - 1)).
// A power is 2^x with x = z log2 e - c in one rounding, c = m log2 e rounded. The
// maximum's own x is what c was rounded by: S is divided by its power, which takes
// the rounding out again and, with it, the error of the hardware's power there (one
// entry left of a row has l = 0 and H = 0 exactly). The rounding of x, at most
// 2^-25 |x|, moves S by at most about 4e-8: the entries that weigh have small x, or
// are many. Where m log2 e would overflow (a row of nothing but the type's lowest
// value) x is z - m: such logits are equal or too far apart for a power to show.
//
// What bounds it is the bytes: each logit is read once and its gradient written
// once. Rows of up to 1024 entries (512 of 32 bits) stay in the registers of a
// part of a warp; longer ones in the shared memory of a CTA, or of a cluster of
// CTAs that exchange (m, S, sum) through distributed shared memory, until the
// gradient is written. Entries are handled in chunks of 16 bytes; rows that
// chunks do not fit have the chunks they lie in. Rows that no cluster can hold
// are read twice by one CTA (the second time mostly from L2).
//
// On a B200 131072 x 512 in bf16 with legal bytes takes 94 to 96 us (3.5 TB/s of the 6.5
// that a copy reaches: the SMs issue in 65% of the cycles, 30 instructions an entry
// with what a row costs by itself), 2048 x 131072 306 to 308 us (3.5 TB/s: 20 an
// entry, two of them powers), 512 x 300000 in f32, which no cluster holds, 642.
#include <cooperative_groups.h>

#include <algorithm>
#include <type_traits>

#include "kernels.h"
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

// x, no lower than what makes 2^x 0 in 32 bits: an entry that does not count (-inf) then adds 0 to every sum. NaN, and
// +inf - inf, stay NaN.
__device__ __forceinline__ float above(float x) {
    float y;
    asm("max.NaN.f32 %0, %1, 0fC47A0000;" : "=f"(y) : "f"(x));  // -1000
    return y;
}

// The factor of the logits, and c of a maximum: the same number wherever it is formed (a product fused into a sum would
// not be rounded)
__device__ __forceinline__ float factor(float m) { return fabsf(m) < 2e38f ? LOG2E : 1.0f; }
__device__ __forceinline__ float scaled(float m) { return __fmul_rn(m, factor(m)); }
// what sums from the maximum m on lack to those from `top` on, as a power of 2
__device__ __forceinline__ float shift(float m, float top) {
    return m == -INFINITY ? 0.0f : above(__fmul_rn(m, factor(top)) - scaled(top));
}

// What a row needs besides its logits: loaded a row ahead, since the logits' loads wait for it (a row that is void
// reads none)
struct RowIn {
    float w, old, A, r;
    int act;  // -1: void
    __device__ __forceinline__ RowIn(const wc_policy_loss_args& a, int64_t t) : w(0.0f), old(0.0f), A(0.0f), r(0.0f), act(-1) {
        if (t >= a.rows) return;
        w = a.weights ? a.weights[t] : 1.0f;
        const int64_t at = a.action_bytes == 8 ? static_cast<const int64_t*>(a.actions)[t]
                                               : (int64_t) static_cast<const int32_t*>(a.actions)[t];
        if (at >= 0 && at < a.width && w != 0.0f) act = (int)at;
        old = a.old_logp[t], A = a.advantages[t];
        if (a.ref_logp) r = a.ref_logp[t];
    }
};

// A row's loss from its parts (m the maximum of all, S and W sums of e and e x)
// and the logit of its action. l is kept in 64 bits up to its differences with
// the other log-probabilities: they are small, and what rounding l first would
// add to them is not.
struct Row {
    float loss, l, H, kl;   // results
    float c, f, g, e, k;    // gradient: d = 2^x (e x + k) + [action] g, x = z f - c
    float ce;
    Row() = default;
    __device__ __forceinline__ Row(const wc_policy_loss_args& a, const RowIn& in, float m, float S, float W, float za) : c(scaled(m)), f(factor(m)) {
        const float top = fmaf(m, f, -c), eTop = ex2(top);  // x and the power of the maximum
        const float inv = __frcp_rn(S), mean = S == eTop ? 0.0f : fmaf(W, inv, -top);  // of x, from the maximum's on
        // ln of S / eTop = 2^n q, q about 1; LOG2E as a float is 1.34e-8 (relative) low, which mean puts right to first order
        int n;
        float q = frexpf(S / eTop, &n);
        if (q < 0.75f) q *= 2.0f, --n;
        const double lnS = (double)n * 0.6931471805599453 + (double)fmaf(mean, 9.25e-9f, logf(q));
        const double ld = ((double)za - (double)m) - lnS;
        l = (float)ld;
        H = fmaf(mean, -LN2, (float)lnS);
        const float lo = 1.0f - a.clip_low, hi = 1.0f + a.clip_high, A = in.A;
        const float ratio = expf((float)(ld - (double)in.old));
        const float free = ratio * A, clipped = fminf(fmaxf(ratio, lo), hi) * A;
        const bool held = (A > 0.0f && ratio > hi) || (A < 0.0f && ratio < lo);
        const float d = a.ref_logp ? (float)((double)in.r - ld) : 0.0f, em = a.ref_logp ? expm1f(d) : 0.0f;
        // exp(d) - 1 - d: for a small d by its series (nine terms: 2^-28 at 1/2), since the difference leaves nothing of it
        float series = 1.0f / 3628800.0f;
        const float n1[8] = {1.0f / 362880.0f, 1.0f / 40320.0f, 1.0f / 5040.0f, 1.0f / 720.0f, 1.0f / 120.0f, 1.0f / 24.0f, 1.0f / 6.0f, 0.5f};
#pragma unroll
        for (int i = 0; i < 8; ++i) series = fmaf(series, d, n1[i]);
        kl = fabsf(d) < 0.5f ? d * d * series : em - d;
        loss = -(free < clipped || isnan(free) ? free : clipped) + (a.kl_coef == 0.0f ? 0.0f : a.kl_coef * kl) - a.entropy_coef * H;  // (kl may be past 32 bits)
        const float up = (a.upstream ? *a.upstream : 1.0f) * in.w;
        g = up * ((held ? 0.0f : -free) - (a.kl_coef == 0.0f ? 0.0f : a.kl_coef * em));
        ce = up * a.entropy_coef;
        // p = 2^x / S and ln p = (x - top) ln 2 - ln (S / eTop)
        e = ce * LN2 * inv, k = fmaf(ce, -LN2 * (mean + top), -g) * inv;
    }
    __device__ __forceinline__ void put(const wc_policy_loss_args& a, int64_t t) const {
        a.row_out[t] = loss, a.row_out[a.rows + t] = l, a.row_out[2 * a.rows + t] = H, a.row_out[3 * a.rows + t] = kl;
    }
    // the gradient at an entry other than the action; one that does not count has 2^x = 0 (and needs a finite x where
    // x is a factor)
    template <bool ENTROPY>
    __device__ __forceinline__ float grad(float z) const {
        const float x = fmaf(z, f, -c);
        if (!ENTROPY) return ex2(x) * k;
        const float y = above(x);
        return ex2(y) * fmaf(y, e, k);
    }
};
__device__ __forceinline__ void put_void(const wc_policy_loss_args& a, int64_t t) {
    a.row_out[t] = 0.0f, a.row_out[a.rows + t] = 0.0f, a.row_out[2 * a.rows + t] = 0.0f, a.row_out[3 * a.rows + t] = 0.0f;
}

// 16 bytes of logits as they lie in memory, what does not count as -inf
template <class T>
struct Chunk {
    static constexpr int N = 16 / sizeof(T);
    static constexpr uint32_t INF = sizeof(T) == 4 ? 0xff800000u : std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;
    alignas(16) uint32_t z[4];
    __device__ __forceinline__ void load(const T* at) { *reinterpret_cast<uint4*>(z) = __ldcs(reinterpret_cast<const uint4*>(at)); }
    // from and to shared memory, by its own addresses
    __device__ __forceinline__ void read(uint32_t at) {
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(z[0]), "=r"(z[1]), "=r"(z[2]), "=r"(z[3]) : "r"(at) : "memory");
    }
    __device__ __forceinline__ void write(uint32_t at) const {
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(z[0]), "r"(z[1]), "r"(z[2]), "r"(z[3]) : "memory");
    }
    __device__ __forceinline__ void none() { z[0] = z[1] = z[2] = z[3] = INF; }
    // legal bytes, in the order of the entries
    __device__ __forceinline__ void mask(uint2 legal) {
        // a byte that is not 0 gets its top bit, which the permutation spreads over the entry's bytes
        const uint32_t on[2] = {((legal.x & 0x7f7f7f7fu) + 0x7f7f7f7fu) | legal.x, ((legal.y & 0x7f7f7f7fu) + 0x7f7f7f7fu) | legal.y};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t m = N == 8 ? spread(on[i >> 1], i & 1 ? 0xbbaa : 0x9988) : spread(on[0], 0x8888 + 0x1111 * i);
            z[i] = (z[i] & m) | (INF & ~m);
        }
    }
    __device__ __forceinline__ static uint2 load_legal(const uint8_t* at) {
        if constexpr (N == 8) return __ldcs(reinterpret_cast<const uint2*>(at));
        return make_uint2(__ldcs(reinterpret_cast<const unsigned int*>(at)), 0);
    }
    __device__ __forceinline__ static uint32_t spread(uint32_t v, uint32_t how) {
        uint32_t r;
        asm("prmt.b32 %0, %1, 0, %2;" : "=r"(r) : "r"(v), "r"(how));
        return r;
    }
    // entries 2 i and 2 i + 1
    __device__ __forceinline__ Pair pair(int i) const {
        if constexpr (sizeof(T) == 4) {
            return umma::f2(z[2 * i], z[2 * i + 1]);
        } else if constexpr (std::is_same<T, __half>::value) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&z[i]));
            return umma::f2(f.x, f.y);
        } else {
            return umma::f2(z[i] << 16, z[i] & 0xffff0000u);
        }
    }
};

// The largest entry of chunks (NaN is left to the sums)
template <class T>
struct Largest {
    using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
    static constexpr bool WIDE = sizeof(T) == 4;
    uint32_t m = Chunk<T>::INF;
    __device__ __forceinline__ void add(const Chunk<T>& q) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if constexpr (WIDE) m = __float_as_uint(fmaxf(__uint_as_float(m), __uint_as_float(q.z[k])));
            else {
                const T2 v = __hmax2(*reinterpret_cast<const T2*>(&m), *reinterpret_cast<const T2*>(&q.z[k]));
                m = *reinterpret_cast<const uint32_t*>(&v);
            }
        }
    }
    __device__ __forceinline__ float get() const {
        if constexpr (WIDE) return __uint_as_float(m);
        else {
            const T2 v = *reinterpret_cast<const T2*>(&m);
            return fmaxf(to_f(v.x), to_f(v.y));
        }
    }
};
// One entry's share of the sums from c on
__device__ __forceinline__ void add_entry(float z, float f, float c, float& s, float& w) {
    const float x = above(fmaf(z, f, -c)), e = ex2(x);
    s += e;
    w = fmaf(e, x, w);
}
// ... of a chunk, by pairs
template <class T>
__device__ __forceinline__ void add_chunk(const Chunk<T>& q, Pair f, Pair c, Pair& s, Pair& w) {
#pragma unroll
    for (int k = 0; k < Chunk<T>::N / 2; ++k) {
        const Pair t = fma(q.pair(k), f, c), x = umma::f2(above(umma::f2_lo(t)), above(umma::f2_hi(t)));
        const Pair e = umma::f2(ex2(umma::f2_lo(x)), ex2(umma::f2_hi(x)));
        s = add(s, e), w = fma(e, x, w);
    }
}
// The gradient of a chunk. (At the action it is not all: the thread that writes the action's chunk writes that entry
// after it, which costs one store a row and nothing an entry.)
template <class T, bool ENTROPY>
__device__ __forceinline__ void chunk_grad(const Chunk<T>& q, const Row& r, T* e) {
    const Pair f = twice(r.f), c = twice(-r.c);
#pragma unroll
    for (int k = 0; k < Chunk<T>::N / 2; ++k) {
        const Pair t = fma(q.pair(k), f, c);
        Pair d;
        if constexpr (ENTROPY) {
            const Pair y = umma::f2(above(umma::f2_lo(t)), above(umma::f2_hi(t)));
            d = mul(umma::f2(ex2(umma::f2_lo(y)), ex2(umma::f2_hi(y))), fma(y, twice(r.e), twice(r.k)));
        } else {
            d = mul(umma::f2(ex2(umma::f2_lo(t)), ex2(umma::f2_hi(t))), twice(r.k));
        }
        if constexpr (sizeof(T) == 4) e[2 * k] = umma::f2_lo(d), e[2 * k + 1] = umma::f2_hi(d);
        else if constexpr (std::is_same<T, __half>::value) reinterpret_cast<__half2*>(e)[k] = __floats2half2_rn(umma::f2_lo(d), umma::f2_hi(d));
        else reinterpret_cast<__nv_bfloat162*>(e)[k] = __floats2bfloat162_rn(umma::f2_lo(d), umma::f2_hi(d));
    }
}
template <class T>
__device__ __forceinline__ void put_chunk(T* out, const T* e) {
    __stcs(reinterpret_cast<uint4*>(out), *reinterpret_cast<const uint4*>(e));
}
// The bytes of entries col .. col + 7 that lie in a row: all bits, or none
__device__ __forceinline__ uint2 inside(int col, int width) {
    const uint64_t m = (~0ull << (8 * max(0, -col))) & (~0ull >> (8 * max(0, min(7, col + 8 - width))));
    return make_uint2((uint32_t)m, (uint32_t)(m >> 32));
}
// A row's logits in registers: NV chunks of `lanes` threads. VEC: the row starts and ends with a chunk. Else it starts
// `before` entries into its first, and chunks are read with what lies there of the rows before and after (`edge`: a row
// that has too little of them around is read entry by entry); the legal bytes of a chunk start anywhere.
template <class T, bool MASK, bool VEC, int NV>
__device__ __forceinline__ void load_row(Chunk<T>* q, const T* z, const uint8_t* legal, bool read, int at, int lanes, int width, int before, bool edge) {
    constexpr int N = Chunk<T>::N;
    if (!VEC && edge) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * lanes + at) * N - before;
            alignas(16) T e[N];
#pragma unroll
            for (int k = 0; k < N; ++k) {
                e[k] = from_f<T>(-INFINITY);
                if (read && c + k >= 0 && c + k < width && (!MASK || legal[c + k])) e[k] = z[c + k];
            }
            *reinterpret_cast<uint4*>(q[i].z) = *reinterpret_cast<const uint4*>(e);
        }
        return;
    }
    uint2 on[MASK ? NV : 1];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (i * lanes + at) * N - before;
        if (read && c < width) {
            q[i].load(z + c);
            if constexpr (MASK && VEC) on[i] = Chunk<T>::load_legal(legal + c);
            if constexpr (MASK && !VEC) {
                const uint32_t* w = reinterpret_cast<const uint32_t*>(reinterpret_cast<uintptr_t>(legal + c) & ~3ull);
                const int by = 8 * (int)(reinterpret_cast<uintptr_t>(legal + c) & 3);
                const uint32_t w1 = __ldg(w + 1);
                on[i] = make_uint2(__funnelshift_r(__ldg(w), w1, by), N == 8 ? __funnelshift_r(w1, __ldg(w + 2), by) : 0u);
            }
        } else {
            q[i].none();
            if constexpr (MASK) on[i] = make_uint2(0, 0);
        }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        if constexpr (VEC) {
            if constexpr (MASK) q[i].mask(on[i]);
        } else {
            const int c = (i * lanes + at) * N - before;
            uint2 m = inside(c, width);
            if constexpr (MASK) m.x &= on[i].x, m.y &= on[i].y;
            if (MASK || c < 0 || c + N > width) q[i].mask(m);
        }
    }
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
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
        const float d = shift(p[i].x, M), f = p[i].x == -INFINITY ? 0.0f : exp2f(d);
        S = fmaf(p[i].y, f, S);
        W = fmaf(fmaf(p[i].y, d, p[i].z), f, W);
    }
    S = warp_sum(S), W = warp_sum(W);
}

template <bool VEC, class T>
__device__ __forceinline__ void put(T* out, const T* e, int i, int at, int lanes, int width, int before, bool same) {
    constexpr int N = Chunk<T>::N;
    const int c = (i * lanes + at) * N - before;
    if (VEC || (same && c >= 0 && c + N <= width)) {
        if (c < width) put_chunk(out + c, e);
    } else {
#pragma unroll
        for (int k = 0; k < N; ++k)
            if (c + k >= 0 && c + k < width) out[c + k] = e[k];
    }
}

// Rows of up to 32 NV chunks: `lanes` threads of a warp a row (a power of two).
template <class T, bool MASK, bool ENTROPY, bool VEC, int NV>
__global__ void __launch_bounds__(256, VEC ? 4 : 2) k_policy_warp(wc_policy_loss_args a, int lanes, double* part) {
    constexpr int N = Chunk<T>::N;
    __shared__ double s[8];
    const int lane = threadIdx.x & 31, at = lane & (lanes - 1), per = 256 / lanes, width = (int)a.width;
    const int64_t stride = (int64_t)gridDim.x * per;
    double total = 0.0;
    RowIn next(a, (int64_t)blockIdx.x * per + threadIdx.x / lanes);
    for (int64_t t0 = (int64_t)blockIdx.x * per; t0 < a.rows; t0 += stride) {
        const int64_t t = t0 + threadIdx.x / lanes;
        const bool in = t < a.rows;
        const T* z = static_cast<const T*>(a.logits) + (in ? t : 0) * a.ld_logits;
        const uint8_t* legal = MASK ? a.legal + (in ? t : 0) * a.ld_legal : nullptr;
        const RowIn r = next;
        Chunk<T> q[NV];
        float za = -INFINITY;
        if (r.act >= 0 && (!MASK || legal[r.act])) za = to_f(z[r.act]);
        const int before = VEC ? 0 : (int)((reinterpret_cast<uintptr_t>(z) & 15) / sizeof(T));
        const int64_t row = in ? t : 0, rest = a.rows - 1 - row, ld = MASK ? min(a.ld_logits, a.ld_legal) : a.ld_logits;
        const bool edge = !VEC && (row * ld < 16 || rest * ld < 16);
        load_row<T, MASK, VEC, NV>(q, z, legal, r.act >= 0, at, lanes, width, before, edge);
        next = RowIn(a, t + stride);
        const bool live = za != -INFINITY;
        Largest<T> most;
#pragma unroll
        for (int i = 0; i < NV; ++i) most.add(q[i]);
        float m = most.get();
        for (int o = lanes >> 1; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
        const Pair f = twice(factor(live ? m : 0.0f)), c = twice(-scaled(live ? m : 0.0f));
        Pair sum = 0, mean = 0;  // (pairs of zeros)
#pragma unroll
        for (int i = 0; i < NV; ++i) add_chunk(q[i], f, c, sum, mean);
        float2 sw = make_float2(both(sum), both(mean));
        for (int o = lanes >> 1; o; o >>= 1) sw.x += __shfl_xor_sync(~0u, sw.x, o), sw.y += __shfl_xor_sync(~0u, sw.y, o);
        if (!in) continue;
        T* out = a.dlogits ? static_cast<T*>(a.dlogits) + t * a.ld_dlogits : nullptr;
        // the gradient's chunks are the logits' if they start at the same place of 16 bytes
        const bool same = (reinterpret_cast<uintptr_t>(out) & 15) == before * sizeof(T);
        if (live) {
            const Row row(a, r, m, sw.x, sw.y, za);
            if (at == 0) row.put(a, t), total += (double)(r.w * row.loss);
            if (!out) continue;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                alignas(16) T e[N];
                chunk_grad<T, ENTROPY>(q[i], row, e);
                put<VEC>(out, e, i, at, lanes, width, before, same);
            }
            if ((((r.act + before) / N) & (lanes - 1)) == at) out[r.act] = from_f<T>(row.grad<ENTROPY>(za) + row.g);
        } else {
            if (at == 0) put_void(a, t);
            alignas(16) T e[N];
#pragma unroll
            for (int k = 0; k < N; ++k) e[k] = from_f<T>(0.0f);
            if (out)
#pragma unroll
                for (int i = 0; i < NV; ++i) put<VEC>(out, e, i, at, lanes, width, before, same);
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

// Longer rows: one CTA, or the CTAs of a cluster, a row, each with a slice of
// it, which bulk copies bring into shared memory and which stays there until
// the gradient is written. A warp of its own starts the copies, joins the
// cluster's parts of a row and forms its loss (some thousand cycles in a chain)
// while the other warps, in the order of the CTA's rows, take the sums of row
// i + 1 and write the gradient of row i. (With that done by the first of the
// working warps, and barriers of the whole CTA, 8192 x 16384 in bf16 took 140 us
// for 129, 2048 x 131072 325 for 320.)
// 16 bytes into the shared memory of a CTA of the cluster (both addresses mapped to it), counted by its barrier. No
// fence: a cluster barrier's release would wait for the gradient's stores as well.
__device__ __forceinline__ void send(uint32_t to, float4 v, uint32_t bar) {
    asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v4.f32 [%0], {%1, %2, %3, %4}, [%5];" ::"r"(to), "f"(v.x),
                 "f"(v.y), "f"(v.z), "f"(v.w), "r"(bar)
                 : "memory");
}
__device__ __forceinline__ uint32_t of_rank(uint32_t addr, int rank) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
constexpr int MAX_SLICES = 4;
template <class T, bool MASK, int WARPS, int CTAS>
__global__ void __launch_bounds__(WARPS * 32 + 32, WARPS == 16 ? 2 : WARPS == 8 ? 4 : 6) k_policy_cluster(wc_policy_loss_args a, int slice, int slices, double* part, uint64_t wait_ns) {
    constexpr int N = Chunk<T>::N, THREADS = WARPS * 32;
    extern __shared__ __align__(128) uint8_t ring[];  // `slices` of the logits, then of the legal bytes
    __shared__ float4 parts[4][CTAS * WARPS];         // of every warp of the cluster, four (live) rows in turn
    __shared__ Row rows[2];                           // what was made of them, two in turn
    __shared__ float2 meta[MAX_SLICES];               // a slice's row: its action (-1: void) and the logit there
    __shared__ uint64_t full[MAX_SLICES], empty[MAX_SLICES], joined[4], ready[2];
    __shared__ int failed;
    cg::cluster_group cluster = cg::this_cluster();
    const int rank = CTAS > 1 ? (int)cluster.block_rank() : 0;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int first = rank * slice;
    const int64_t t0 = blockIdx.x / CTAS, step = gridDim.x / CTAS;
    // A row starts `before` entries into its first chunk, and its chunks are dealt to the CTAs: this one's are the entries
    // from first - before on, `width` of them (of which the row's first and last chunk may have fewer). Bulk copies take
    // whole chunks, with what lies there of the rows before and after; the matrix's first and last row, which have none,
    // are read where they are if they do not fill theirs.
    auto row_at = [&](int64_t t) { return static_cast<const T*>(a.logits) + t * a.ld_logits; };
    auto before = [&](int64_t t) { return (int)((reinterpret_cast<uintptr_t>(row_at(t)) & 15) / sizeof(T)); };
    auto width_of = [&](int b) { return min(slice, max(0, (int)a.width + b - first)); };
    auto in_place = [&](int64_t t) {
        if (t != 0 && t != a.rows - 1) return false;
        return before(t) != 0 || (a.width + before(t)) % N != 0 || (MASK && (((uintptr_t)(a.legal + t * a.ld_legal) & 15) != 0 || a.width % 16 != 0));
    };
    uint8_t* masks = ring + slices * slice * sizeof(T);
    auto arrive = [](uint64_t* bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(umma::smem_u32(bar)) : "memory"); };
    if (threadIdx.x == 0) {
        for (int i = 0; i < slices; ++i) umma::mbar_init(&full[i], 1), umma::mbar_init(&empty[i], WARPS);
        for (int i = 0; i < 4; ++i) umma::mbar_init(&joined[i], CTAS > 1 ? 1 : WARPS);
        for (int i = 0; i < 2; ++i) umma::mbar_init(&ready[i], 1);
        failed = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (CTAS > 1) cluster.sync();
    else __syncthreads();
    double total = 0.0;  // (CTAs by themselves)
    // A wait that runs out leaves NaN in the rows from here on. What a warp that gave up owes to others stays undone, so
    // that their waits run out too and none takes a place for free, or a row's parts for whole, that is not.
    bool bad = false;
    auto wait = [&](uint64_t* bar, int64_t use) {
        if (!bad && !wait_within(bar, (uint32_t)use & 1, wait_ns)) bad = true, failed = 1;
        bad = __any_sync(~0u, bad);  // (a warp's lanes go on together)
    };
    // the slice of a row, and how often it had others before
    struct Place {
        int slot = 0;
        uint32_t use = 0;
        __device__ __forceinline__ void next(int slices) {
            if (++slot == slices) slot = 0, ++use;
        }
    };
    if (warp == WARPS) {
        // Lane k has the scalars of the k-th of 32 rows, loaded 32 rows ahead of their use.
        struct Batch {
            RowIn in;
            float za;
        };
        auto load = [&](int64_t i) {
            const int64_t t = t0 + (i + lane) * step;
            Batch v{RowIn(a, t), -INFINITY};
            if (v.in.act >= 0 && (!MASK || a.legal[t * a.ld_legal + v.in.act])) v.za = to_f(row_at(t)[v.in.act]);
            return v;
        };
        Batch now = load(0), next = load(32);
        // the slice of the CTA's row i, of the batch now or next
        auto copy = [&](int64_t i, int slot, bool later) {
            const int from = (int)i & 31;
            const int act = __shfl_sync(~0u, later ? next.in.act : now.in.act, from);
            const float za = __shfl_sync(~0u, later ? next.za : now.za, from);
            const int64_t t = t0 + i * step;
            if (lane || t >= a.rows) return;
            const int b = before(t), width = width_of(b);
            const bool live = za != -INFINITY;
            meta[slot] = make_float2(__int_as_float(live ? act : -1), za);
            if (!live || !width || in_place(t)) {
                arrive(&full[slot]);
                return;
            }
            const uint32_t bytes = (width + N - 1) / N * 16;
            const uint8_t* on = MASK ? a.legal + t * a.ld_legal + max(0, first - b) : nullptr;
            const uint32_t skew = (uint32_t)((uintptr_t)on & 15), on_bytes = MASK ? (skew + width - (first ? 0 : b) + 15) / 16 * 16 : 0;
            umma::expect_tx(&full[slot], bytes + on_bytes);
            umma::bulk_g2s(ring + slot * slice * sizeof(T), row_at(t) - b + first, bytes, &full[slot]);
            if (MASK) umma::bulk_g2s(masks + slot * (slice + 32), on - skew, on_bytes, &full[slot]);
        };
        for (int i = 0; i < slices; ++i) copy(i, i, false);
        Place done;  // of the row before
        int64_t live = 0;
        for (int64_t i = 0, t = t0; t < a.rows; ++i, t += step) {
            const int at = (int)i & 31;
            if (at == 0 && i) now = next, next = load(i + 32);
            const float za = __shfl_sync(~0u, now.za, at);
            if (za != -INFINITY) {
                const int turn = (int)live & 3;
                RowIn in = now.in;
                in.w = __shfl_sync(~0u, in.w, at), in.old = __shfl_sync(~0u, in.old, at), in.A = __shfl_sync(~0u, in.A, at), in.r = __shfl_sync(~0u, in.r, at);
                if (CTAS > 1 && lane == 0 && !bad) umma::expect_tx(&joined[turn], CTAS * WARPS * 16);
                wait(&joined[turn], live >> 2);
                float M, S, W;
                join<(CTAS * WARPS + 31) / 32>(parts[turn], CTAS * WARPS, M, S, W);
                if (bad) S = __uint_as_float(0x7fffffffu);
                const Row row(a, in, M, S, W, za);
                if (lane == 0) {
                    if (!bad) rows[live & 1] = row, arrive(&ready[live & 1]);
                    if (rank == 0) row.put(a, t);
                    if (CTAS == 1) total += (double)(in.w * row.loss);
                }
                ++live;
            } else if (rank == 0 && lane == 0) {
                put_void(a, t);
            }
            // The slice of row i - 1 is free once its gradient is written, which is before the next row's parts are all
            // here: this wait holds nothing up.
            const int64_t ahead = i - 1 + slices;
            if (i && t + (slices - 1) * step < a.rows) {
                wait(&empty[done.slot], done.use);
                if (!bad) copy(ahead, done.slot, (ahead >> 5) != (i >> 5)), done.next(slices);
            }
            __syncwarp();
        }
        // the copies in flight land before the CTA leaves, also where no one waits for them any more
        const int64_t copied = min((a.rows - t0 + step - 1) / step, (int64_t)(done.use + 1) * slices + done.slot);
        if (lane == 0)
            for (int64_t i = max((int64_t)0, copied - slices); i < copied; ++i) umma::mbar_wait(&full[i % slices], (uint32_t)(i / slices) & 1, umma::DRAIN_NS);
    } else {
        int64_t live = 0;  // rows with parts sent
        int act0 = -1;
        float za0 = 0.0f;
        Place read, written;
        for (int64_t i = -1, t = t0 - step; t < a.rows; ++i, t += step) {
            const int64_t t1 = t + step;
            int act1 = -1;
            float za1 = 0.0f;
            if (t1 < a.rows) {
                const int slot = read.slot;
                wait(&full[slot], read.use);
                read.next(slices);
                const float2 about = meta[slot];
                act1 = bad ? -1 : __float_as_int(about.x), za1 = about.y;
                if (act1 >= 0) {
                    const int b = before(t1), width = width_of(b);
                    const uint32_t z = umma::smem_u32(ring) + (uint32_t)(slot * slice * sizeof(T));
                    const bool here = in_place(t1);
                    const uint8_t* on = MASK ? a.legal + t1 * a.ld_legal + max(0, first - b) : nullptr;
                    // legal byte of column col: base[skew + col]
                    const uint8_t* base = masks + slot * (slice + 32);
                    const int skew = (int)((uintptr_t)on & 15) - max(0, first - b);
                    const bool even = ((skew + first - b) & (N - 1)) == 0;  // a chunk's bytes are one word, or two
                    // First the maximum; a chunk whose entries do not all count goes back as what does.
                    const int from = b - first, last = (int)a.width + from - N;  // where chunks lie in the row
                    Largest<T> most;
                    auto some = [&](int at) {
                        const int col = at - from;
                        const bool whole = at >= from && at <= last;
                        Chunk<T> q;
                        if (here) {
                            alignas(16) T e[N];
#pragma unroll
                            for (int k = 0; k < N; ++k) {
                                e[k] = from_f<T>(-INFINITY);
                                if (col + k >= 0 && col + k < a.width && (!MASK || a.legal[t1 * a.ld_legal + col + k])) e[k] = row_at(t1)[col + k];
                            }
                            *reinterpret_cast<uint4*>(q.z) = *reinterpret_cast<const uint4*>(e);
                        } else {
                            q.read(z + at * sizeof(T));
                            uint2 m = make_uint2(0, 0);
                            if (!whole) {
                                for (int k = 0; k < N; ++k)
                                    if (col + k >= 0 && col + k < a.width && (!MASK || base[skew + col + k])) (k < 4 ? m.x : m.y) |= 1u << (8 * (k & 3));
                            } else if (MASK && even) {
                                if constexpr (N == 8) m = *reinterpret_cast<const uint2*>(base + skew + col);
                                else m.x = *reinterpret_cast<const uint32_t*>(base + skew + col);
                            } else if (MASK) {
                                const uint32_t* w = reinterpret_cast<const uint32_t*>(base + ((skew + col) & ~3));
                                const int by = 8 * ((skew + col) & 3);
                                m = make_uint2(__funnelshift_r(w[0], w[1], by), N == 8 ? __funnelshift_r(w[1], w[2], by) : 0u);
                            }
                            q.mask(m);
                        }
                        q.write(z + at * sizeof(T));
                        // ... before the copy that takes its place
                        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                        most.add(q);
                    };
                    if (MASK || here) {
                        for (int at = threadIdx.x * N; at < width; at += THREADS * N) some(at);
                    } else {
                        for (int at = threadIdx.x * N; at < width; at += THREADS * N) {
                            Chunk<T> q;
                            q.none();
                            if (at >= from && at <= last) q.read(z + at * sizeof(T));
                            else some(at);
                            most.add(q);
                        }
                    }
                    float m = most.get();
#pragma unroll
                    for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
                    if (m == -INFINITY) m = 0.0f;  // nothing here counts (or is a number): its sums are 0 (or NaN)
                    const Pair f = twice(factor(m)), c = twice(-scaled(m));
                    Pair sum = 0, mean = 0;
                    for (int at = threadIdx.x * N; at < width; at += THREADS * N) {
                        Chunk<T> q;
                        q.read(z + at * sizeof(T));
                        add_chunk(q, f, c, sum, mean);
                    }
                    const float2 v = make_float2(warp_sum(both(sum)), warp_sum(both(mean)));
                    const float4 mine = make_float4(v.x == 0.0f ? -INFINITY : m, v.x, v.y, 0.0f);
                    // Of four places in turn this one has been read everywhere: before this row a warp has written the
                    // gradient of the live row before last, for which every CTA's parts of it were joined; they were sent
                    // after the gradients of the live row two before that, for which each CTA had joined its parts.
                    const int turn = (int)live & 3;
                    float4* to = &parts[turn][rank * WARPS + warp];
                    if (CTAS == 1 && lane == 0) *to = mine, arrive(&joined[turn]);
                    if (CTAS > 1 && lane < CTAS) send(of_rank(umma::smem_u32(to), lane), mine, of_rank(umma::smem_u32(&joined[turn]), lane));
                    ++live;
                }
            }
            if (i >= 0) {
                const int64_t mine = live - 1 - (act1 >= 0);  // this row among the live ones
                if (act0 >= 0) wait(&ready[mine & 1], mine >> 1);
                const int slot = written.slot;
                if (a.dlogits) {
                    const int b = before(t), width = width_of(b);
                    const uint32_t z = umma::smem_u32(ring) + (uint32_t)(slot * slice * sizeof(T));
                    T* out = static_cast<T*>(a.dlogits) + t * a.ld_dlogits;
                    // the gradient's chunks are the logits' if they start at the same place of 16 bytes
                    const bool same = (reinterpret_cast<uintptr_t>(out) & 15) == b * sizeof(T);
                    const int from = b - first, last = (int)a.width + from - N;  // where chunks lie in the row
                    T* const o = out - from;
                    auto chunks = [&](auto&& make) {
                        for (int at = threadIdx.x * N; at < width; at += THREADS * N) {
                            Chunk<T> q;
                            q.read(z + at * sizeof(T));
                            alignas(16) T e[N];
                            make(q, e);
                            if (same && at >= from && at <= last) put_chunk(o + at, e);
                            else
#pragma unroll
                                for (int j = 0; j < N; ++j)
                                    if (at + j >= from && at + j < last + N) o[at + j] = e[j];
                        }
                    };
                    const Row r = rows[mine & 1];
                    if (act0 >= 0 && !bad) {
                        if (r.ce != 0.0f)
                            chunks([&](const Chunk<T>& q, T* e) { chunk_grad<T, true>(q, r, e); });
                        else
                            chunks([&](const Chunk<T>& q, T* e) { chunk_grad<T, false>(q, r, e); });
                        const int own = act0 + b - first;
                        if (own >= 0 && own < width && own / N % THREADS == (int)threadIdx.x) out[act0] = from_f<T>(r.grad<true>(za0) + r.g);
                    } else {
                        const T fill = from_f<T>(bad ? __uint_as_float(0x7fffffffu) : 0.0f);
                        chunks([&](const Chunk<T>&, T* e) {
#pragma unroll
                            for (int k = 0; k < N; ++k) e[k] = fill;
                        });
                    }
                }
                __syncwarp();
                if (lane == 0 && !bad) arrive(&empty[slot]);
                written.next(slices);
            }
            act0 = act1, za0 = za1;
        }
    }
    __syncthreads();
    if (CTAS == 1 && threadIdx.x == THREADS) part[blockIdx.x] = total;
    if (CTAS > 1) {
        cluster.sync();  // no CTA leaves while another may still write to it
        // Where this CTA's warp has not waited for all that was sent to it, the last of that may still be on its way, for less
        // than a few microseconds.
        if (failed)
            for (const uint64_t from = umma::now_ns(); umma::now_ns() - from < 100000;) {}
    }
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
        const RowIn r(a, t);
        float za = -INFINITY;
        if (r.act >= 0 && (!legal || legal[r.act])) za = to_f(z[r.act]);
        if (za == -INFINITY) {
            if (out)
                for (int64_t j = threadIdx.x; j < V; j += 512) out[j] = from_f<T>(0.0f);
            if (threadIdx.x == 0) put_void(a, t);
            continue;
        }
        // Eight entries at a time: their maximum moves the running one, then their powers are added up and the sum's share
        // to what there is. A thread has hundreds of entries, most of them small beside the sum: what rounding takes off them
        // is kept and added at the end (without it l was off by 1.3e-6 at 430000 entries with a deviation of 4).
        float m = -INFINITY, s = 0.0f, w = 0.0f, s_rest = 0.0f, w_rest = 0.0f;
        auto add_to = [](float& sum, float& rest, float v) {
            const float t = sum + v, had = t - v;
            rest += (sum - had) + (v - (t - had));
            sum = t;
        };
        for (int64_t j = threadIdx.x; j < V; j += 8 * 512) {
            float v[8], top = m;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const int64_t i = j + k * 512;
                v[k] = i < V && (!legal || legal[i]) ? to_f(z[i]) : -INFINITY;
                top = fmaxf(top, v[k]);
            }
            const float from = top == -INFINITY ? 0.0f : top, c = scaled(from), d = shift(m, from), f = exp2f(d);
            w = fmaf(s, d, w) * f, w_rest = fmaf(s_rest, d, w_rest) * f, s *= f, s_rest *= f, m = top;
            float ds = 0.0f, dw = 0.0f;
#pragma unroll
            for (int k = 0; k < 8; ++k) add_entry(v[k], factor(from), c, ds, dw);
            add_to(s, s_rest, ds), add_to(w, w_rest, dw);
        }
        s += s_rest, w += w_rest;
        float top = m;
#pragma unroll
        for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
        const float d = shift(m, top), f = exp2f(d);
        w = warp_sum(fmaf(s, d, w) * f), s = warp_sum(s * f);
        __syncthreads();  // the last row's parts have been read
        if (lane == 0) parts[warp] = make_float4(top, s, w, 0.0f);
        __syncthreads();
        float M, S, W;
        join<1>(parts, 16, M, S, W);
        const Row row(a, r, M, S, W, za);
        if (threadIdx.x == 0) row.put(a, t), total += (double)(r.w * row.loss);
        if (out)
            for (int64_t j = threadIdx.x; j < V; j += 512) {
                const float v = !legal || legal[j] ? to_f(z[j]) : -INFINITY;
                float d = row.grad<true>(v);
                if (j == r.act) d += row.g;
                out[j] = from_f<T>(d);
            }
    }
    if (threadIdx.x == 0) part[blockIdx.x] = total;
}

// a sum over the CTA's threads, in a fixed order
__device__ __forceinline__ double cta_sum(double v) {
    __shared__ double s[32];
    const int lane = threadIdx.x & 31;
    auto warp = [](double x) {
#pragma unroll
        for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(~0u, x, o);
        return x;
    };
    v = warp(v);
    if (lane == 0) s[threadIdx.x >> 5] = v;
    __syncthreads();
    return warp(lane < (int)blockDim.x / 32 ? s[lane] : 0.0);
}
// the CTAs' totals
__global__ void __launch_bounds__(1024) k_policy_total(const double* part, int n, float* loss) {
    double v = 0.0;
    for (int i = threadIdx.x; i < n; i += blockDim.x) v += part[i];
    v = cta_sum(v);
    if (threadIdx.x == 0) *loss = (float)v;
}
// Clusters of several CTAs have no totals: how many there are is the GPU's to say, and the loss would depend on it. CTA i
// sums up `run` rows' losses; a single one's total is the loss. (A void row's loss is 0, whatever its weight.)
__global__ void __launch_bounds__(1024) k_policy_row_total(const float* row_loss, const float* weights, int64_t rows, int64_t run, double* part, float* loss) {
    const int64_t first = blockIdx.x * run, last = min(first + run, rows);
    double v = 0.0;
#pragma unroll 8
    for (int64_t t = first + threadIdx.x; t < last; t += 1024) {
        const float l = row_loss[t], w = weights ? weights[t] : 1.0f;
        if (l != 0.0f) v += (double)(w * l);
    }
    v = cta_sum(v);
    if (threadIdx.x) return;
    if (gridDim.x == 1) *loss = (float)v;
    else part[blockIdx.x] = v;
}

constexpr int MOST_CTAS = 148 * 8;

constexpr size_t RING = 208 * 1024;  // of an SM's shared memory (the cluster's parts take 8 KB more of each CTA's)
// Slices are whole chunks of a row that may start up to N - 1 entries into its first
template <class T>
int64_t slice_of(const wc_policy_loss_args& a, int ctas) {
    return ((a.width + Chunk<T>::N - 1 + ctas - 1) / ctas + 15) / 16 * 16;
}
// ... and their bytes, with legal bytes' room for the 16s that they start and end in
template <class T, bool MASK>
int64_t slice_bytes(int64_t slice) {
    return slice * sizeof(T) + (MASK ? slice + 32 : 0);
}
// `sm`: CTAs of one SM. (The launchers answer how many CTAs left totals; 0: the rows are still to be added.)
template <class T, bool MASK, int WARPS, int CTAS>
int launch_cluster(const wc_policy_loss_args& a, int sm, double* part, cudaStream_t s) {
    const int slice = (int)slice_of<T>(a, CTAS);
    const int64_t bytes = slice_bytes<T, MASK>(slice);
    const int slices = (int)std::min<int64_t>(MAX_SLICES, (int64_t)RING / sm / bytes);
    const auto kernel = k_policy_cluster<T, MASK, WARPS, CTAS>;
    if (!wcdev::raise_smem_limit(reinterpret_cast<const void*>(kernel), RING)) return 0;
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim = {CTAS, 1, 1};
    cfg.blockDim = WARPS * 32 + 32, cfg.stream = s, cfg.attrs = &attr, cfg.numAttrs = 1, cfg.dynamicSmemBytes = (size_t)(slices * bytes);
    // As many clusters as are resident at a time: they do not fill the SMs of every GPC, and the ones left over would
    // start only when the others have ended (37 of 8 CTAs, of which 33 fit, took 560 us at 2048 x 131072 in bf16, 33
    // took 387).
    cfg.gridDim = CTAS * sm;
    int most = 0;
    if (CTAS == 1) most = 148 * sm;
    else if (cudaOccupancyMaxActiveClusters(&most, kernel, &cfg) != cudaSuccess || most < 1) most = 1;
    const int n = (int)std::min<int64_t>(most, a.rows);
    cfg.gridDim = n * CTAS;
    cudaLaunchKernelEx(&cfg, kernel, a, slice, slices, part, wait_limit());
    return CTAS == 1 ? n : 0;
}

template <class T, bool MASK, bool ENTROPY, bool VEC>
int launch_warp(const wc_policy_loss_args& a, double* part, cudaStream_t s) {
    const int64_t chunks = (a.width + (VEC ? 1 : 2) * (Chunk<T>::N - 1)) / Chunk<T>::N;
    // up to 4 chunks a lane (8 a lane and half the warps took 8% longer at 131072 x 512 in bf16)
    int lanes = 1;
    while (lanes < 32 && lanes * 4 < chunks) lanes *= 2;
    const int64_t per = 256 / lanes;
    const int n = (int)std::min<int64_t>(MOST_CTAS, (a.rows + per - 1) / per);
    const int nv = (int)((chunks + lanes - 1) / lanes);
    if (nv <= 1) k_policy_warp<T, MASK, ENTROPY, VEC, 1><<<n, 256, 0, s>>>(a, lanes, part);
    else if (nv == 2) k_policy_warp<T, MASK, ENTROPY, VEC, 2><<<n, 256, 0, s>>>(a, lanes, part);
    else if (nv == 3) k_policy_warp<T, MASK, ENTROPY, VEC, 3><<<n, 256, 0, s>>>(a, lanes, part);
    else k_policy_warp<T, MASK, ENTROPY, VEC, 4><<<n, 256, 0, s>>>(a, lanes, part);
    return n;
}

template <class T, bool MASK>
int launch_rows(const wc_policy_loss_args& a, double* part, cudaStream_t s) {
    constexpr int N = Chunk<T>::N;
    const auto fits = [&](const void* p, int64_t ld, size_t e, int to) { return ((uintptr_t)p & (to - 1)) == 0 && (ld * e) % to == 0; };
    const bool fit = a.width % N == 0 && fits(a.logits, a.ld_logits, sizeof(T), 16) && (!a.dlogits || fits(a.dlogits, a.ld_dlogits, sizeof(T), 16)) &&
                     (!a.legal || fits(a.legal, a.ld_legal, 1, 8));
    const bool is_short = (a.width + (fit ? 1 : 2) * (N - 1)) / N <= 32 * 4;
    if (is_short) {
        if (a.entropy_coef != 0.0f) return fit ? launch_warp<T, MASK, true, true>(a, part, s) : launch_warp<T, MASK, true, false>(a, part, s);
        return fit ? launch_warp<T, MASK, false, true>(a, part, s) : launch_warp<T, MASK, false, false>(a, part, s);
    }
    // The smallest CTA, then the smallest cluster, of which an SM's memory takes as many as its registers with three
    // slices each; of the longest rows one CTA, with two or more
    const auto fits_sm = [&](int ctas, int sm, int slices) { return slices * slice_bytes<T, MASK>(slice_of<T>(a, ctas)) <= (int64_t)RING / sm; };
    if (fits_sm(1, 6, 3)) return launch_cluster<T, MASK, 4, 1>(a, 6, part, s);
    if (fits_sm(1, 4, 3)) return launch_cluster<T, MASK, 8, 1>(a, 4, part, s);
    if (fits_sm(1, 2, 3)) return launch_cluster<T, MASK, 16, 1>(a, 2, part, s);
    if (fits_sm(2, 2, 3)) return launch_cluster<T, MASK, 16, 2>(a, 2, part, s);
    if (fits_sm(4, 2, 3)) return launch_cluster<T, MASK, 16, 4>(a, 2, part, s);
    if (fits_sm(8, 2, 3)) return launch_cluster<T, MASK, 16, 8>(a, 2, part, s);
    if (fits_sm(8, 1, 2)) return launch_cluster<T, MASK, 16, 8>(a, 1, part, s);
    const int n = (int)std::min<int64_t>(148 * 4, a.rows);
    k_policy_long<T><<<n, 512, 0, s>>>(a, part);
    return n;
}

template <class T>
int launch_type(const wc_policy_loss_args& a, double* part, cudaStream_t s) {
    return a.legal ? launch_rows<T, true>(a, part, s) : launch_rows<T, false>(a, part, s);
}

}  // namespace

uint64_t policy_loss_workspace(int64_t, int64_t) { return MOST_CTAS * sizeof(double); }

void launch_policy_loss(const wc_policy_loss_args& a, cudaStream_t s) {
    double* part = static_cast<double*>(a.workspace);
    int n = 0;
    if (a.rows) n = a.type == WC_F32   ? launch_type<float>(a, part, s)
                    : a.type == WC_F16 ? launch_type<__half>(a, part, s)
                                       : launch_type<__nv_bfloat16>(a, part, s);
    if (!n) {
        const int64_t run = std::max<int64_t>(32768, (a.rows + MOST_CTAS - 1) / MOST_CTAS);
        n = (int)std::max<int64_t>(1, (a.rows + run - 1) / run);
        k_policy_row_total<<<n, 1024, 0, s>>>(a.row_out, a.weights, a.rows, run, part, a.loss);
        if (n == 1) return;
    }
    k_policy_total<<<1, std::min(1024, std::max(32, (n + 31) / 32 * 32)), 0, s>>>(part, n, a.loss);
}

}  // namespace wctrain
