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
// and two out; four in and two out), read and written once. A thread has units
// of 8 columns: next to each other, 16 bytes of a 16-bit type at a time, where
// addresses and strides allow, else one column of each of 8 runs, so that the
// threads of a warp still read and write next to each other.
//   forward: a row in the registers of a part of a warp, or of a CTA; means and
//     deviations from the registers, in two passes.
//   backward, widths up to 256: a part of a warp a row, a unit a thread, which
//     also keeps that unit's sums over the rows (weights' and gate's).
//   backward, widths up to 4096: a CTA a row, a unit a thread; rows come to
//     shared memory by bulk copies some rows ahead where their addresses allow.
//   backward, wider: the sums of a CTA no longer fit its registers: the rows
//     first (dx, dh and two means a row), then the sums column by column, which
//     reads the inputs a second time.
//
// On a B200 16384 x 4096 in bf16 takes 100 to 112 us forward (4.8 TB/s and more of the
// 6.5 that a copy reaches: a CTA waits for its row's sums) and 240 us backward, 606208
// x 96 in f16 121 and 204 us (3.4 TB/s backward: 16 warps an SM that issue in half of
// the cycles, at 128 registers a thread, and 12 units for 16 lanes).
#include <algorithm>
#include <type_traits>

#include "colsum.cuh"
#include "kernels.h"
#include "umma.cuh"

namespace wctrain {

namespace {

struct Row {
    float pm, pr, nm, nr;
};

// The segments of a group joined: 32 columns of group blockIdx.y a CTA, the segments dealt to its warps and those joined in
// order. (With a thread a column, a chain of 2368 segments, the backward pass of one gate over 19184 x 25 took 174 us
// for 49.)
template <class T>
__global__ void __launch_bounds__(1024) k_gate_sum(const float* part, int segments, int64_t D, T* out) {
    __shared__ float s[32][33];
    const int64_t c = (int64_t)blockIdx.x * 32 + threadIdx.x, group = blockIdx.y;
    float v = 0.0f;
    if (c < D)
        for (int k = threadIdx.y; k < segments; k += blockDim.y) v += part[(group * segments + k) * D + c];
    s[threadIdx.y][threadIdx.x] = v;
    __syncthreads();
    if (threadIdx.y || c >= D) return;
    for (int j = 1; j < (int)blockDim.y; ++j) v += s[j][threadIdx.x];
    out[group * D + c] = from_f<T>(v);
}

// ---- units -------------------------------------------------------------------

// How a thread's 8 columns lie: next to each other; or one of each of 8 runs, the runs as long as the threads that share
// the row (of a warp or less), or 32 (a warp's 256 columns next to each other: offsets known to the compiler).
enum { VEC, LANES, RUNS };
// A thread's i-th unit of a row: `at` of `apart` threads.
template <class T, int LAY>
struct Cols {
    int D, at, apart;
    __device__ __forceinline__ int col(int i, int k) const {
        return LAY == VEC ? (i * apart + at) * 8 + k : LAY == RUNS ? (i * apart + (at & ~31)) * 8 + (at & 31) + k * 32 : (i * 8 + k) * apart + at;
    }
    __device__ __forceinline__ bool in(int i, int k) const { return col(i, LAY == VEC ? 0 : k) < D; }
    __device__ __forceinline__ bool any(int i) const { return col(i, 0) < D; }
};
template <class T, int LAY>
struct Unit {
    T e[8];
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int k = 0; k < 8; ++k) e[k] = from_f<T>(0.0f);
    }
    __device__ __forceinline__ void load(const T* row, const Cols<T, LAY>& c, int i) {
        const T* p = row + c.col(i, 0);
        const int left = c.D - c.col(i, 0), step = c.col(i, 1) - c.col(i, 0);
#pragma unroll
        for (int k = 0; k < 8; ++k) e[k] = k * step < left ? p[k * step] : from_f<T>(0.0f);
    }
    __device__ __forceinline__ void stream(const T* row, const Cols<T, LAY>& c, int i) { load(row, c, i); }
    __device__ __forceinline__ void get(float* v) const {
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = to_f(e[k]);
    }
    __device__ __forceinline__ static void put(T* row, const Cols<T, LAY>& c, int i, const float* v) {
        T* p = row + c.col(i, 0);
        const int left = c.D - c.col(i, 0), step = c.col(i, 1) - c.col(i, 0);
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (k * step < left) p[k * step] = from_f<T>(v[k]);
    }
};
template <class T>
struct Unit<T, VEC> {
    uint4 w[sizeof(T) / 2];
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) w[i] = make_uint4(0, 0, 0, 0);
    }
    __device__ __forceinline__ void load(const T* row, const Cols<T, VEC>& c, int i) {
        const T* p = row + c.col(i, 0);
#pragma unroll
        for (int j = 0; j < (int)sizeof(T) / 2; ++j) w[j] = reinterpret_cast<const uint4*>(p)[j];
    }
    __device__ __forceinline__ void stream(const T* row, const Cols<T, VEC>& c, int i) {
        const T* p = row + c.col(i, 0);
#pragma unroll
        for (int j = 0; j < (int)sizeof(T) / 2; ++j) w[j] = __ldcs(reinterpret_cast<const uint4*>(p) + j);
    }
    __device__ __forceinline__ void get(float* v) const {
        const uint32_t* u = reinterpret_cast<const uint32_t*>(w);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if constexpr (sizeof(T) == 4) v[2 * j] = __uint_as_float(u[2 * j]), v[2 * j + 1] = __uint_as_float(u[2 * j + 1]);
            else if constexpr (std::is_same<T, __nv_bfloat16>::value) v[2 * j] = __uint_as_float(u[j] << 16), v[2 * j + 1] = __uint_as_float(u[j] & 0xffff0000u);
            else {
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[j]));
                v[2 * j] = f.x, v[2 * j + 1] = f.y;
            }
        }
    }
    __device__ __forceinline__ static void put(T* row, const Cols<T, VEC>& c, int i, const float* v) {
        T* p = row + c.col(i, 0);
        alignas(16) uint32_t e[2 * sizeof(T)];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if constexpr (sizeof(T) == 4) e[2 * j] = __float_as_uint(v[2 * j]), e[2 * j + 1] = __float_as_uint(v[2 * j + 1]);
            else if constexpr (std::is_same<T, __nv_bfloat16>::value) *reinterpret_cast<__nv_bfloat162*>(&e[j]) = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
            else *reinterpret_cast<__half2*>(&e[j]) = __floats2half2_rn(v[2 * j], v[2 * j + 1]);
        }
#pragma unroll
        for (int j = 0; j < (int)sizeof(T) / 2; ++j) __stcs(reinterpret_cast<uint4*>(p) + j, reinterpret_cast<const uint4*>(e)[j]);
    }
};
// the same columns of a 32-bit vector
template <class T, int LAY>
__device__ __forceinline__ void load8(const float* p, const Cols<T, LAY>& c, int i, float* v) {
    if constexpr (LAY == VEC) {
        const float4 a = *reinterpret_cast<const float4*>(p + c.col(i, 0)), b = *reinterpret_cast<const float4*>(p + c.col(i, 0) + 4);
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    } else {
        const int left = c.D - c.col(i, 0), step = c.col(i, 1) - c.col(i, 0);
        p += c.col(i, 0);
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = k * step < left ? p[k * step] : 0.0f;
    }
}
template <class T, int LAY>
__device__ __forceinline__ void store8(float* p, const Cols<T, LAY>& c, int i, const float* v) {
    if constexpr (LAY == VEC) {
        *reinterpret_cast<float4*>(p + c.col(i, 0)) = make_float4(v[0], v[1], v[2], v[3]);
        *reinterpret_cast<float4*>(p + c.col(i, 0) + 4) = make_float4(v[4], v[5], v[6], v[7]);
    } else {
        const int left = c.D - c.col(i, 0), step = c.col(i, 1) - c.col(i, 0);
        p += c.col(i, 0);
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (k * step < left) p[k * step] = v[k];
    }
}
__device__ __forceinline__ void fill8(float* v, float x) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = x;
}
__device__ __forceinline__ void pairs(const float* f, Pair* v) {
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = umma::f2(f[2 * k], f[2 * k + 1]);
}
__device__ __forceinline__ void unpairs(const Pair* v, float* f) {
#pragma unroll
    for (int k = 0; k < 4; ++k) f[2 * k] = umma::f2_lo(v[k]), f[2 * k + 1] = umma::f2_hi(v[k]);
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
// NV units a thread.
template <class T, int LAY, int WARPS, int NV, int lanes = 32>
__global__ void __launch_bounds__(WARPS ? WARPS * 32 : 256, WARPS ? 32 / (WARPS ? WARPS : 1) : LAY == VEC ? 4 : 3) k_norm_units(wc_block_norm_args a) {
    __shared__ float2 s[2][32];
    Group<WARPS> group{s, lanes};
    const int D = (int)a.width;
    const Cols<T, LAY> cols{D, WARPS ? (int)threadIdx.x : (int)(threadIdx.x & (lanes - 1)), WARPS ? (int)blockDim.x : lanes};
    const int per = WARPS ? 1 : 256 / lanes, slot = WARPS ? 0 : (int)threadIdx.x / lanes;
    const int blocks = (D + 31) / 32;
    const float inv = 1.0f / (float)D;
    const bool layer = a.kind == WC_NORM_LAYER;
    // The next row's h and x are read from when this one's are used up, where that leaves registers: CTAs and 16-bit
    // types (16384 x 4096 in bf16 104 us for 119; parts of warps 127 for 119 at 606208 x 96, 32-bit types 108 for 100 at
    // 32768 x 1024).
    constexpr bool AHEAD = LAY == VEC && WARPS && sizeof(T) == 2;
    Unit<T, LAY> h[AHEAD ? NV : 1], x[NV];
    const int64_t step = (int64_t)gridDim.x * per;
    auto fetch = [&](int64_t t, int i, Unit<T, LAY>& to) {
        to.zero();
        if (t >= a.rows || !cols.any(i)) return;
        to.stream(static_cast<const T*>(a.h) + t * a.ld_h, cols, i);
        x[i].stream(static_cast<const T*>(a.x) + t * a.ld_x, cols, i);
    };
    auto fetch_ahead = [&](int64_t t) {
        if constexpr (AHEAD)
#pragma unroll
            for (int i = 0; i < NV; ++i) fetch(t, i, h[i]);
    };
    fetch_ahead((int64_t)blockIdx.x * per + slot);
    for (int64_t t0 = (int64_t)blockIdx.x * per; t0 < a.rows; t0 += step) {
        const int64_t t = t0 + slot;
        const bool in = t < a.rows;
        float v[NV][8];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if (!AHEAD) fetch(t, i, h[0]);
            h[AHEAD ? i : 0].get(v[i]);
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
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    if (cols.in(i, k)) q = fmaf(v[i][k] - mean, v[i][k] - mean, q);
            r = rsqrtf(group.sum(q) * inv + a.eps);
        };
        Row r{0.0f, 1.0f, 0.0f, 1.0f};
        if (a.post_weight) moments(r.pm, r.pr);
        const T* gate = a.gate && in ? static_cast<const T*>(a.gate) + t / a.rows_per_gate * D : nullptr;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if (!in || !cols.any(i)) continue;
            if (a.post_weight) {
                float w[8], b[8];
                load8(a.post_weight, cols, i, w);
                if (a.post_bias) load8(a.post_bias, cols, i, b);
                else fill8(b, 0.0f);
#pragma unroll
                for (int k = 0; k < 8; ++k) v[i][k] = fmaf((v[i][k] - r.pm) * r.pr, w[k], b[k]);
            }
            float xf[8];
            x[i].get(xf);
            if (gate) {
                Unit<T, LAY> gu;
                gu.load(gate, cols, i);
                float g[8];
                gu.get(g);
#pragma unroll
                for (int k = 0; k < 8; ++k) v[i][k] = fmaf(a.residual_scale, xf[k], g[k] * v[i][k]);
            } else {
#pragma unroll
                for (int k = 0; k < 8; ++k) v[i][k] = fmaf(a.residual_scale, xf[k], v[i][k]);
            }
            if (LAY != VEC)  // (whose columns past the width had weights of 0 but no x)
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    if (!cols.in(i, k)) v[i][k] = 0.0f;
            Unit<T, LAY>::put(static_cast<T*>(a.y) + t * a.ld_y, cols, i, v[i]);
        }
        fetch_ahead(t + step);
        if (a.pre_weight) {
            moments(r.nm, r.nr);
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                if (in && cols.any(i)) {
                    float w[8], b[8];
                    load8(a.pre_weight, cols, i, w);
                    if (a.pre_bias) load8(a.pre_bias, cols, i, b);
                    else fill8(b, 0.0f);
#pragma unroll
                    for (int k = 0; k < 8; ++k) v[i][k] = cols.in(i, k) ? fmaf((v[i][k] - r.nm) * r.nr, w[k], b[k]) : 0.0f;
                    if (a.n) Unit<T, LAY>::put(static_cast<T*>(a.n) + t * a.ld_n, cols, i, v[i]);
                }
                if (!a.n_q) continue;
                if constexpr (LAY == VEC) {  // 4 threads next to each other hold a block (lanes is at least 4 then)
                    uint32_t code;
                    const uint2 q = quantise8(v[i], &code);
                    const int c = cols.col(i, 0);
                    if (in && c < blocks * 32) {
                        *reinterpret_cast<uint2*>(a.n_q + t * blocks * 32 + c) = q;
                        if ((c & 31) == 0) a.n_scale[t * blocks + c / 32] = (uint8_t)code;
                    }
                } else {  // a warp does (lanes is 32 then)
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        const uint32_t code = act8_code(__uint_as_float(__reduce_max_sync(~0u, __float_as_uint(v[i][k]) & 0x7fffffffu)));
                        const int c = cols.col(i, k);
                        if (in && c < blocks * 32) {
                            a.n_q[t * blocks * 32 + c] = act8_whole(v[i][k], code);
                            if ((c & 31) == 0) a.n_scale[t * blocks + c / 32] = (uint8_t)code;
                        }
                    }
                }
            }
        }
        if (in && cols.at == 0) reinterpret_cast<float4*>(a.stats)[t] = make_float4(r.pm, r.pr, r.nm, r.nr);
    }
}

// ---- the backward pass -----------------------------------------------------------
// Rows come in items, a segment of a group of rows with the same gate. Worker w
// takes items w, w + workers, ...: it keeps the weights' sums over all of them
// and hands on the gate's sum of each.
struct Plan {
    int64_t R, groups, per, items;
    int width, segments, workers, lanes, parts;  // lanes of a warp a row (0: a CTA a row, -1: rows, then columns)
    Plan(const wc_block_norm_args& a) {
        width = (int)a.width;
        // (a gate for more rows than there are is one for all of them, however many it says)
        R = a.gate ? std::min(a.rows_per_gate, std::max<int64_t>(1, a.rows)) : a.rows;
        groups = a.rows ? (a.rows + R - 1) / R : 0;
        lanes = a.width > 4096 ? -1 : 0;
        if (a.width <= 256)
            for (lanes = 1; lanes * 8 < a.width;) lanes *= 2;
        const int64_t most = lanes > 0 ? 148 * 2 * 8 : lanes == 0 ? 148 * (512 / threads()) : 296;
        const int64_t longest = R < a.rows ? R : a.rows, want = groups ? (most + groups - 1) / groups : 1;
        const int64_t fit = (longest + 7) / 8;
        segments = (int)(fit < 1 ? 1 : fit < want ? fit : want);
        per = longest ? (longest + segments - 1) / segments : 1;
        items = groups * segments;
        workers = (int)(items < most ? items : most);
        parts = lanes > 0 ? (workers + 7) / 8 : workers;  // partial sums of the weights
    }
    int threads() const { return (width + 255) / 256 * 32; }  // of a CTA that has a row
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

// Arithmetic on pairs, each rounded as the scalar form: the backward pass has some 30 operations a column, which would
// bound it before the bytes do.
__device__ __forceinline__ void fill(Pair* v, float x) {
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = twice(x);
}

__device__ __forceinline__ void bulk_copy(uint32_t to, uint64_t from, uint32_t bytes, uint64_t* bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(to), "l"(from), "r"(bytes),
                 "r"(umma::smem_u32(bar))
                 : "memory");
}

// What a thread keeps of its unit: the parameters and their gradients' sums.
// Columns past the width have weights, gate and inputs of 0, and so add 0 to
// everything. Over the rows of an item the gate g is the same, so with A = g wp
// and B = g bp its rows need
//   y = c x + A hhat + B, dU wp = A dY, s1 = sum dY, s2 = sum dY hhat,
// and its end dg = wp s2 + bp s1, dwp += g s2, dbp += g s1. The last two wait
// in shared memory (`kept`: a thread's 16 numbers, a thread apart): with them in
// registers, and a sum a row for each of the three, 16384 x 4096 in bf16 took 330 us
// for 251. (The warp form still spills: 32 to 44 bytes in its aligned 16-bit
// instances, up to 280 where rows lie anywhere.)
struct Column {
    Pair A[4], B[4], wn[4];
    Pair s1[4], s2[4], dwn[4], dbn[4];
    float* kept;
    int apart;
    template <class T, int LAY>
    __device__ __forceinline__ static void param(const float* p, float otherwise, const Cols<T, LAY>& c, int i, Pair* to) {
        float v[8];
        fill8(v, 0.0f);
        if (c.any(i)) {
            if (p) load8(p, c, i, v);
            else
#pragma unroll
                for (int k = 0; k < 8; ++k) v[k] = c.in(i, k) ? otherwise : 0.0f;
        }
        pairs(v, to);
    }
    template <class T, int LAY>
    __device__ __forceinline__ static void gate(const wc_block_norm_args& a, int64_t group, const Cols<T, LAY>& c, int i, Pair* to) {
        if (!a.gate) {
            param(nullptr, 1.0f, c, i, to);
            return;
        }
        Unit<T, LAY> u;
        u.zero();
        if (c.any(i)) u.load(static_cast<const T*>(a.gate) + group * c.D, c, i);
        float v[8];
        u.get(v);
        pairs(v, to);
    }
    template <class T, int LAY>
    __device__ __forceinline__ void load(const wc_block_norm_args& a, const Cols<T, LAY>& c, int i, float* to, int threads) {
        kept = to, apart = threads;
        param(a.pre_weight, 0.0f, c, i, wn);
        fill(dwn, 0.0f), fill(dbn, 0.0f);
#pragma unroll
        for (int k = 0; k < 16; ++k) kept[k * apart] = 0.0f;
    }
    // an item begins
    template <class T, int LAY>
    __device__ __forceinline__ void begin(const wc_block_norm_args& a, int64_t group, const Cols<T, LAY>& c, int i) {
        Pair g[4];
        gate(a, group, c, i, g), param(a.post_weight, 1.0f, c, i, A), param(a.post_bias, 0.0f, c, i, B);
#pragma unroll
        for (int k = 0; k < 4; ++k) A[k] = mul(g[k], A[k]), B[k] = mul(g[k], B[k]);
        fill(s1, 0.0f), fill(s2, 0.0f);
    }
    // ... and ends, with the gate's gradient
    template <class T, int LAY>
    __device__ __forceinline__ void end(const wc_block_norm_args& a, int64_t group, const Cols<T, LAY>& c, int i, float* dg) {
        Pair g[4], w[4], b[4];
        gate(a, group, c, i, g), param(a.post_weight, 1.0f, c, i, w), param(a.post_bias, 0.0f, c, i, b);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const Pair d = fma(w[k], s2[k], mul(b[k], s1[k])), dw = mul(g[k], s2[k]), db = mul(g[k], s1[k]);
            dg[2 * k] = umma::f2_lo(d), dg[2 * k + 1] = umma::f2_hi(d);
            float* at = kept + 2 * k * apart;
            at[0] += umma::f2_lo(dw), at[apart] += umma::f2_hi(dw), at[8 * apart] += umma::f2_lo(db), at[9 * apart] += umma::f2_hi(db);
        }
    }
    // the sums over all items: dwp, dbp, dwn, dbn
    __device__ __forceinline__ void sums(int which, float* v) const {
        if (which < 2)
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = kept[(which * 8 + k) * apart];
        else unpairs(which == 2 ? dwn : dbn, v);
    }
    // A row's unit. get(i, v) reads its x, h, dy or dn (i = 0 .. 3; zeros past the width and for a gradient that is not
    // there), when it is needed: what is not held meanwhile leaves room for the sums. put(i, v) takes dx, then dh. `zero`
    // stands for what the pre norm gives where there is none.
    template <class G, class Get, class Put>
    __device__ __forceinline__ void row(const wc_block_norm_args& a, const float4& st, bool pre, float inv, float zero, G& group, Get&& get, Put&& put) {
        const bool layer = a.kind == WC_NORM_LAYER;
        Pair hh[4], yh[4], d[4];
        get(1, hh), get(0, yh);
        hats(a, st, hh, yh);
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
            const Pair a0 = twice(layer ? -m.x * inv : 0.0f), a1 = twice(-m.y * inv), nr = twice(st.w);
#pragma unroll
            for (int k = 0; k < 4; ++k) yh[k] = mul(nr, fma(yh[k], a1, add(d[k], a0)));
        } else {
            fill(yh, zero);
        }
        get(2, d);
        const Pair rs = twice(a.residual_scale);
#pragma unroll
        for (int k = 0; k < 4; ++k) yh[k] = add(d[k], yh[k]), d[k] = mul(rs, yh[k]);  // dY
        put(0, d);
        Pair c0 = 0, c1 = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            add_to(k, yh[k], hh[k]);
            yh[k] = mul(yh[k], A[k]);
            c0 = add(c0, yh[k]), c1 = fma(yh[k], hh[k], c1);
        }
        if (a.post_weight) {
            const float2 c = group.sum(make_float2(both(c0), both(c1)));
            const Pair a0 = twice(layer ? -c.x * inv : 0.0f), a1 = twice(-c.y * inv), pr = twice(st.y);
#pragma unroll
            for (int k = 0; k < 4; ++k) yh[k] = mul(pr, fma(hh[k], a1, add(yh[k], a0)));
        }
        put(1, yh);
    }
    // h and x to hhat and yhat
    __device__ __forceinline__ void hats(const wc_block_norm_args& a, const float4& st, Pair* hh, Pair* yh) const {
        const Pair pr = twice(st.y), pm = twice(-st.x), nr = twice(st.w), nm = twice(-st.z), rs = twice(a.residual_scale);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            hh[k] = mul(add(hh[k], pm), pr);
            yh[k] = mul(add(fma(hh[k], A[k], fma(rs, yh[k], B[k])), nm), nr);
        }
    }
    // the gate's and the post norm's sums
    __device__ __forceinline__ void add_to(int k, Pair dY, Pair hh) { s1[k] = add(s1[k], dY), s2[k] = fma(dY, hh, s2[k]); }
};

// A part of a warp a row; a warp is a worker.
template <class T, int LAY, int lanes>
__global__ void __launch_bounds__(256, 2) k_norm_backward_warp(wc_block_norm_args a, wc_block_norm_grads g, Items q,
                                                               float* gate_part, float* weight_part) {
    __shared__ float s[8][8][33], kept[16][256];
    const int D = (int)a.width, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int slots = 32 / lanes, slot = lane / lanes, worker = blockIdx.x * 8 + warp;
    const Cols<T, LAY> cols{D, lane & (lanes - 1), lanes};
    const bool any = cols.any(0), pre = a.pre_weight && g.dn;
    const float inv = 1.0f / (float)D;
    Group<0> group{nullptr, lanes};
    Column col;
    col.load(a, cols, 0, &kept[0][threadIdx.x], 256);
    for (int64_t i = worker; i < q.items; i += q.workers) {
        int64_t item_group, first, last;
        q.range(i, item_group, first, last);
        col.begin(a, item_group, cols, 0);
        Unit<T, LAY> u[4];  // x, h, dy, dn: the next row's from when dx is out
        float4 next = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        auto fetch = [&](int64_t t) {
#pragma unroll
            for (int k = 0; k < 4; ++k) u[k].zero();
            if (t >= last) return;
            next = reinterpret_cast<const float4*>(a.stats)[t];
            if (!any) return;
            u[0].stream(static_cast<const T*>(a.x) + t * a.ld_x, cols, 0);
            u[1].stream(static_cast<const T*>(a.h) + t * a.ld_h, cols, 0);
            if (g.dy) u[2].stream(static_cast<const T*>(g.dy) + t * g.ld_dy, cols, 0);
            if (g.dn) u[3].stream(static_cast<const T*>(g.dn) + t * g.ld_dn, cols, 0);
        };
        fetch(first + slot);
        for (int64_t t0 = first; t0 < last; t0 += slots) {
            const int64_t t = t0 + slot;
            const bool here = any && t < last;  // (a row past the last has gradients of 0: it adds 0 to every sum)
            const float4 st = next;
            col.row(a, st, pre, inv, 0.0f, group,
                    [&](int k, Pair* v) {
                        float f[8];
                        u[k].get(f);
                        pairs(f, v);
                    },
                    [&](int k, const Pair* v) {
                        float f[8];
                        unpairs(v, f);
                        if (k == 0 && here && g.dx) Unit<T, LAY>::put(static_cast<T*>(g.dx) + t * g.ld_dx, cols, 0, f);
                        if (k == 0) fetch(t + slots);
                        if (k == 1 && here && g.dh) Unit<T, LAY>::put(static_cast<T*>(g.dh) + t * g.ld_dh, cols, 0, f);
                    });
        }
        float dg[8];
        col.end(a, item_group, cols, 0, dg);
        if (g.dgate) {
#pragma unroll
            for (int k = 0; k < 8; ++k)
                for (int o = 16; o >= lanes; o >>= 1) dg[k] += __shfl_xor_sync(~0u, dg[k], o);
            if (slot == 0 && any) {
                if (q.segments == 1) Unit<T, LAY>::put(static_cast<T*>(g.dgate) + item_group * D, cols, 0, dg);
                else store8(gate_part + i * D, cols, 0, dg);
            }
        }
    }
    // the slots of a warp, then the warps
    auto flush = [&](int which) {
        float v[8];
        col.sums(which, v);
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            for (int o = 16; o >= lanes; o >>= 1) v[k] += __shfl_xor_sync(~0u, v[k], o);
            s[warp][k][lane] = v[k];
        }
        __syncthreads();
        const int k = warp;
        if (slot == 0 && cols.in(0, k)) {
            float t = 0.0f;
#pragma unroll
            for (int w = 0; w < 8; ++w) t += s[w][k][lane];
            weight_part[((int64_t)blockIdx.x * 4 + which) * D + cols.col(0, k)] = t;
        }
    };
    flush(0), flush(1), flush(2), flush(3);
}

// A CTA a row, one unit a thread; a CTA is a worker. Its rows in order come to
// shared memory by bulk copies: x, h, dy, dn and the statistics. A bulk copy
// moves whole 16-byte pieces: of rows that do not end on them (LAY != VEC) it
// takes the pieces they lie in, parts of the rows before and after; the
// matrices' first and last rows, which have none, are read where they are.
constexpr int MAX_RING = 8;
template <class T, int LAY>
__global__ void __launch_bounds__(512) k_norm_backward_cta(wc_block_norm_args a, wc_block_norm_grads g, Items q, int stages,
                                                           float* gate_part, float* weight_part, uint64_t wait_ns) {
    extern __shared__ __align__(128) uint8_t shared[];  // what Column keeps, then the ring
    uint8_t* const ring = shared + 64 * blockDim.x;
    __shared__ float2 s[2][32];
    __shared__ uint64_t full[MAX_RING];
    const int D = (int)a.width, row_bytes = D * (int)sizeof(T), piece = LAY == VEC ? row_bytes : (row_bytes + 15) / 16 * 16 + 16;
    const int stage_bytes = 4 * piece + 16;
    const Cols<T, LAY> cols{D, (int)threadIdx.x, (int)blockDim.x};
    const bool any = cols.any(0), pre = a.pre_weight && g.dn;
    const float inv = 1.0f / (float)D;
    Group<16> group{s, 32};
    Column col;
    col.load(a, cols, 0, reinterpret_cast<float*>(shared) + threadIdx.x, blockDim.x);
    if (threadIdx.x == 0) {
        for (int i = 0; i < stages; ++i) umma::mbar_init(&full[i], 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    auto row_of = [&](int k, int64_t t) -> const T* {
        return k == 0   ? static_cast<const T*>(a.x) + t * a.ld_x
               : k == 1 ? static_cast<const T*>(a.h) + t * a.ld_h
               : k == 2 ? (g.dy ? static_cast<const T*>(g.dy) + t * g.ld_dy : nullptr)
                        : (g.dn ? static_cast<const T*>(g.dn) + t * g.ld_dn : nullptr);
    };
    auto edge = [&](int64_t t) { return LAY != VEC && (t == 0 || t == a.rows - 1); };
    // The first warp walks ahead of the rows: lanes 0 to 3 copy x, h, dy and dn, lane 4 the statistics.
    const int array = threadIdx.x < 4 ? threadIdx.x : 0;
    const uint64_t base = reinterpret_cast<uint64_t>(row_of(array, 0));
    const int64_t pitch = (array == 0 ? a.ld_x : array == 1 ? a.ld_h : array == 2 ? g.ld_dy : g.ld_dn) * (int64_t)sizeof(T);
    int64_t copy_item = blockIdx.x, copy_row = 0, copy_last = 0, copy_group;
    int copy_slot = 0;
    uint32_t copied = 0;
    auto copy = [&] {
        while (copy_row >= copy_last) {
            if (copy_item >= q.items) return;
            q.range(copy_item, copy_group, copy_row, copy_last);
            copy_item += q.workers;
        }
        const uint64_t p = base + copy_row * pitch;
        const uint64_t from = threadIdx.x < 4 ? p & ~15ull : reinterpret_cast<uint64_t>(a.stats + copy_row * 4);
        const uint32_t bytes = threadIdx.x == 4 ? 16 : threadIdx.x > 4 || !base || edge(copy_row) ? 0 : (uint32_t)(((p + row_bytes + 15) & ~15ull) - from);
        const uint32_t total = __reduce_add_sync(~0u, bytes);
        if (threadIdx.x == 0) umma::expect_tx(&full[copy_slot], total);
        __syncwarp();
        if (bytes) bulk_copy(umma::smem_u32(ring + copy_slot * stage_bytes) + threadIdx.x * piece, from, bytes, &full[copy_slot]);
        copy_slot = copy_slot + 1 == stages ? 0 : copy_slot + 1;
        ++copy_row, ++copied;
    };
    if (threadIdx.x < 32)
        for (int i = 0; i + 1 < stages; ++i) copy();
    int slot = 0;
    uint32_t turns = 0;  // of the ring
    bool bad = false;
    for (int64_t i = blockIdx.x; i < q.items; i += q.workers) {
        int64_t item_group, first, last;
        q.range(i, item_group, first, last);
        col.begin(a, item_group, cols, 0);
        for (int64_t t = first; t < last; ++t) {
            // a copy that does not come leaves NaN from here on: hhat and yhat are none, nor is 0
            if (!bad && !wait_within(&full[slot], turns & 1, wait_ns)) bad = true;
            float4 st = *reinterpret_cast<const float4*>(ring + slot * stage_bytes + 4 * piece);
            const float zero = bad ? __uint_as_float(0x7fffffffu) : 0.0f;
            if (bad) st.y = st.w = zero;
            const bool here = !edge(t);
            // all have read the row before this one, whose stage takes another: with a post norm, before its last sum
            if (!a.post_weight) __syncthreads();
            if (threadIdx.x < 32 && __all_sync(~0u, !bad)) copy();
            col.row(a, st, pre, inv, zero, group,
                    [&](int k, Pair* v) {
                        Unit<T, LAY> u;
                        u.zero();
                        const T* p = row_of(k, t);
                        if (any && p) {
                            const T* copied = reinterpret_cast<const T*>(ring + slot * stage_bytes + k * piece + (reinterpret_cast<uintptr_t>(p) & 15));
                            if (here) u.load(copied, cols, 0);
                            else u.load(p, cols, 0);
                        }
                        float f[8];
                        u.get(f);
                        pairs(f, v);
                    },
                    [&](int k, const Pair* v) {
                        if (!any) return;
                        float f[8];
                        unpairs(v, f);
                        if (k == 0 && g.dx) Unit<T, LAY>::put(static_cast<T*>(g.dx) + t * g.ld_dx, cols, 0, f);
                        if (k == 1 && g.dh) Unit<T, LAY>::put(static_cast<T*>(g.dh) + t * g.ld_dh, cols, 0, f);
                    });
            if (++slot == stages) slot = 0, ++turns;
        }
        float dg[8];
        col.end(a, item_group, cols, 0, dg);
        if (g.dgate && any) {
            if (q.segments == 1) Unit<T, LAY>::put(static_cast<T*>(g.dgate) + item_group * D, cols, 0, dg);
            else store8(gate_part + i * D, cols, 0, dg);
        }
    }
    if (bad && threadIdx.x == 0)  // (the others' rows have all come where this thread's have)
        for (uint32_t i = copied > (uint32_t)stages ? copied - stages : 0; i < copied; ++i)
            umma::mbar_wait(&full[i % stages], (i / stages) & 1, umma::DRAIN_NS);
    if (bad) fill(col.dbn, __uint_as_float(0x7fffffffu));  // (a sum of dn alone)
    if (any) {
        float* to = weight_part + (int64_t)blockIdx.x * 4 * D;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            float v[8];
            col.sums(k, v);
            store8(to + k * D, cols, 0, v);
        }
    }
}

// Wide rows: a CTA a row, two units a thread; what it does is Column::row
// without the sums over rows.
template <class T, int LAY, int WARPS>
__global__ void __launch_bounds__(WARPS * 32) k_norm_backward_rows(wc_block_norm_args a, wc_block_norm_grads g, float2* means) {
    __shared__ float2 s[2][32];
    const int D = (int)a.width;
    const Cols<T, LAY> cols{D, (int)threadIdx.x, (int)blockDim.x};
    const bool layer = a.kind == WC_NORM_LAYER, pre = a.pre_weight && g.dn;
    const float inv = 1.0f / (float)D;
    Group<WARPS> group{s, 32};
    for (int64_t t = blockIdx.x; t < a.rows; t += gridDim.x) {
        const float4 st = reinterpret_cast<const float4*>(a.stats)[t];
        const T* gate = a.gate ? static_cast<const T*>(a.gate) + t / a.rows_per_gate * D : nullptr;
        auto get = [&](const void* p, int64_t ld, int i, float* v) {
            Unit<T, LAY> u;
            u.zero();
            if (p && cols.any(i)) u.load(static_cast<const T*>(p) + t * ld, cols, i);
            u.get(v);
        };
        float hh[2][8], d[2][8], yh[2][8];  // hhat; dY, then the gradient at the post norm's output times its weight; yhat
        float2 m = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            get(a.h, a.ld_h, i, hh[i]);
            get(a.x, a.ld_x, i, yh[i]);
            get(g.dn, g.ld_dn, i, d[i]);
            if (!cols.any(i)) continue;
            float w[8], b[8], ga[8];
            fill8(w, 1.0f), fill8(b, 0.0f), fill8(ga, 1.0f);
            if (a.post_weight) load8(a.post_weight, cols, i, w);
            if (a.post_bias) load8(a.post_bias, cols, i, b);
            if (gate) {
                Unit<T, LAY> u;
                u.load(gate, cols, i), u.get(ga);
            }
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                hh[i][k] = (hh[i][k] - st.x) * st.y;
                yh[i][k] = (fmaf(a.residual_scale, yh[i][k], ga[k] * fmaf(hh[i][k], w[k], b[k])) - st.z) * st.w;
            }
            if (pre) {
                load8(a.pre_weight, cols, i, w);
#pragma unroll
                for (int k = 0; k < 8; ++k) d[i][k] = cols.in(i, k) ? d[i][k] * w[k] : 0.0f, m.x += d[i][k], m.y = fmaf(d[i][k], yh[i][k], m.y);
            }
        }
        if (pre) {
            m = group.sum(m);
            m.x = layer ? m.x * inv : 0.0f, m.y *= inv;
        }
        if (threadIdx.x == 0) means[t] = m;
        float2 c = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            if (!cols.any(i)) continue;
            float dy[8], w[8];
            get(g.dy, g.ld_dy, i, dy);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                d[i][k] = dy[k] + (pre ? st.w * (d[i][k] - m.x - yh[i][k] * m.y) : 0.0f);
                dy[k] = a.residual_scale * d[i][k];
            }
            if (g.dx) Unit<T, LAY>::put(static_cast<T*>(g.dx) + t * g.ld_dx, cols, i, dy);
            if (gate) {
                Unit<T, LAY> u;
                u.load(gate, cols, i), u.get(w);
#pragma unroll
                for (int k = 0; k < 8; ++k) d[i][k] *= w[k];
            }
            if (a.post_weight) {
                load8(a.post_weight, cols, i, w);
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    d[i][k] = cols.in(i, k) ? d[i][k] * w[k] : 0.0f;
                    c.x += d[i][k], c.y = fmaf(d[i][k], hh[i][k], c.y);
                }
            }
        }
        if (a.post_weight) {
            c = group.sum(c);
            c.x = layer ? c.x * inv : 0.0f, c.y *= inv;
        }
        if (g.dh)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                if (!cols.any(i)) continue;
                if (a.post_weight)
#pragma unroll
                    for (int k = 0; k < 8; ++k) d[i][k] = st.y * (d[i][k] - c.x - hh[i][k] * c.y);
                Unit<T, LAY>::put(static_cast<T*>(g.dh) + t * g.ld_dh, cols, i, d[i]);
            }
    }
}

// ... and the sums: a warp has 256 columns and every eighth row of an item, the
// CTA's eight warps are joined at the end of one.
template <class T, int LAY>
__global__ void __launch_bounds__(256, 2) k_norm_backward_cols(wc_block_norm_args a, wc_block_norm_grads g, Items q, const float2* means,
                                                            float* gate_part, float* weight_part) {
    __shared__ float s[8][8][33], kept[16][256];
    const int D = (int)a.width, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    // the columns as one unit of `apart` threads' row, of which this CTA has 32
    const int all = gridDim.x * 32;
    const Cols<T, LAY> cols{D, (int)blockIdx.x * 32 + lane, all};
    const bool any = cols.any(0), pre = a.pre_weight && g.dn;
    Column col;
    col.load(a, cols, 0, &kept[0][threadIdx.x], 256);
    // v summed over the warps: thread (warp k, lane) gets column k of lane's unit
    auto over_warps = [&](const float* v) {
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 8; ++k) s[warp][k][lane] = v[k];
        __syncthreads();
        float t = 0.0f;
#pragma unroll
        for (int w = 0; w < 8; ++w) t += s[w][warp][lane];
        return t;
    };
    for (int64_t i = blockIdx.y; i < q.items; i += q.workers) {
        int64_t item_group, first, last;
        q.range(i, item_group, first, last);
        col.begin(a, item_group, cols, 0);
        for (int64_t t = first + warp; t < last; t += 8) {
            const float4 st = reinterpret_cast<const float4*>(a.stats)[t];
            const float2 m = means[t];
            Pair hh[4], yh[4], dn[4], dY[4];
            auto get = [&](const void* p, int64_t ld, Pair* v) {
                Unit<T, LAY> u;
                u.zero();
                if (p && any) u.stream(static_cast<const T*>(p) + t * ld, cols, 0);
                float f[8];
                u.get(f);
                pairs(f, v);
            };
            get(a.h, a.ld_h, hh), get(a.x, a.ld_x, yh), get(g.dn, g.ld_dn, dn), get(g.dy, g.ld_dy, dY);
            col.hats(a, st, hh, yh);
            const Pair a0 = twice(-m.x), a1 = twice(-m.y), nr = twice(st.w);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                if (pre) dY[k] = fma(nr, fma(yh[k], a1, fma(dn[k], col.wn[k], a0)), dY[k]);
                col.dwn[k] = fma(dn[k], yh[k], col.dwn[k]), col.dbn[k] = add(col.dbn[k], dn[k]);
                col.add_to(k, dY[k], hh[k]);
            }
        }
        float dg[8];
        col.end(a, item_group, cols, 0, dg);
        if (g.dgate) {
            const float v = over_warps(dg);
            if (cols.in(0, warp)) {
                if (q.segments == 1) static_cast<T*>(g.dgate)[item_group * D + cols.col(0, warp)] = from_f<T>(v);
                else gate_part[i * D + cols.col(0, warp)] = v;
            }
        }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        float sum[8];
        col.sums(k, sum);
        const float v = over_warps(sum);
        if (cols.in(0, warp)) weight_part[((int64_t)blockIdx.y * 4 + k) * D + cols.col(0, warp)] = v;
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

template <class T, bool UNITS>
void backward_as(const wc_block_norm_args& a, const wc_block_norm_grads& g, cudaStream_t s) {
    const Plan p(a);
    const int64_t D = a.width, e = sizeof(T);
    float* ws = static_cast<float*>(g.workspace);
    float2* means = reinterpret_cast<float2*>(ws);
    float *weights = ws + (a.rows + 1) / 2 * 4, *gates = weights + (int64_t)p.parts * 4 * D;  // both 16-byte aligned where D is a multiple of 4
    constexpr int WIDE = UNITS ? VEC : RUNS, NARROW = UNITS ? VEC : LANES;
    if (a.rows) {
        const Items q{p.items, p.per, p.R, a.rows, p.segments, p.workers};
        if (p.lanes > 0) {
            const auto kernel = p.lanes == 1   ? k_norm_backward_warp<T, NARROW, 1>
                                : p.lanes == 2 ? k_norm_backward_warp<T, NARROW, 2>
                                : p.lanes == 4 ? k_norm_backward_warp<T, NARROW, 4>
                                : p.lanes == 8 ? k_norm_backward_warp<T, NARROW, 8>
                                : p.lanes == 16 ? k_norm_backward_warp<T, NARROW, 16>
                                                : k_norm_backward_warp<T, NARROW, 32>;
            kernel<<<p.parts, 256, 0, s>>>(a, g, q, gates, weights);
        } else if (p.lanes == 0) {
            const int stage = (int)(4 * (UNITS ? D * e : (D * e + 15) / 16 * 16 + 16) + 16), threads = p.threads();
            const int stages = (int)std::min<int64_t>(MAX_RING, (200 * 1024 / (512 / threads) - 64 * threads) / stage);
            if (wcdev::raise_smem_limit(reinterpret_cast<const void*>(k_norm_backward_cta<T, WIDE>), 200 * 1024))
                k_norm_backward_cta<T, WIDE><<<p.workers, threads, (size_t)stages * stage + 64 * threads, s>>>(a, g, q, stages, gates, weights, wait_limit());
        } else {
            const unsigned threads = (unsigned)((D + 511) / 512 * 32);
            const unsigned n = (unsigned)std::min<int64_t>(a.rows, 148 * (1024 / threads));
            if (threads <= 512) k_norm_backward_rows<T, WIDE, 16><<<n, threads, 0, s>>>(a, g, means);
            else k_norm_backward_rows<T, WIDE, 32><<<n, threads, 0, s>>>(a, g, means);
            k_norm_backward_cols<T, WIDE><<<dim3((unsigned)((D + 255) / 256), p.workers), 256, 0, s>>>(a, g, q, means, gates, weights);
        }
        if (g.dgate && p.segments > 1)
            // (there are segments only where the groups are fewer than the workers)
            k_gate_sum<T><<<dim3((unsigned)((D + 31) / 32), (unsigned)p.groups), dim3(32, p.segments >= 16 ? 32 : 4), 0, s>>>(
                gates, p.segments, D, static_cast<T*>(g.dgate));
    }
    if (g.dpost_weight || g.dpost_bias || g.dpre_weight || g.dpre_bias)
        launch_colsum(weights, p.parts, 4 * D, D, 4, ColSums{{g.dpost_weight, g.dpost_bias, g.dpre_weight, g.dpre_bias}}, s);
}
template <class T>
void backward(const wc_block_norm_args& a, const wc_block_norm_grads& g, cudaStream_t s) {
    const size_t e = sizeof(T);
    const bool vec = units_ok(a) && unit_rows(g.dy, g.ld_dy, e) && unit_rows(g.dn, g.ld_dn, e) && unit_rows(g.dx, g.ld_dx, e) &&
                     unit_rows(g.dh, g.ld_dh, e) && unit_rows(g.dgate, a.width, e);
    if (vec) backward_as<T, true>(a, g, s);
    else backward_as<T, false>(a, g, s);
}

template <class T, bool UNITS>
void forward_as(const wc_block_norm_args& a, cudaStream_t s) {
    // units of a row, whole blocks of 32 columns where it is packed
    constexpr int WIDE = UNITS ? VEC : RUNS, NARROW = UNITS ? VEC : LANES;
    const int units = (int)(a.n_q ? (a.width + 31) / 32 * 4 : (a.width + 7) / 8);
    if (units <= 64) {
        // (where units are runs, a whole warp from 129 columns on)
        int lanes = UNITS ? (a.n_q ? 4 : 1) : a.n_q || a.width > 128 ? 32 : 1;
        while (lanes < 32 && lanes * 2 < units) lanes *= 2;
        const int64_t per = 256 / lanes;
        const unsigned n = (unsigned)std::min<int64_t>(148 * 16, (a.rows + per - 1) / per);
        const auto kernel = lanes == 32  ? (units <= 32 ? k_norm_units<T, NARROW, 0, 1, 32> : k_norm_units<T, NARROW, 0, 2, 32>)
                            : lanes == 16 ? k_norm_units<T, VEC, 0, 2, 16>
                            : lanes == 8  ? k_norm_units<T, NARROW, 0, 2, 8>
                            : lanes == 4  ? (units <= 4 ? k_norm_units<T, NARROW, 0, 1, 4> : k_norm_units<T, NARROW, 0, 2, 4>)
                            : lanes == 2  ? k_norm_units<T, NARROW, 0, 2, 2>
                            : units == 1  ? k_norm_units<T, NARROW, 0, 1, 1>
                                          : k_norm_units<T, NARROW, 0, 2, 1>;
        kernel<<<n, 256, 0, s>>>(a);
        return;
    }
    // two units a thread (one a thread was slower: 157 against 123 us at 16384 x 4096 in bf16)
    const int threads = (units + 63) / 64 * 32;
    const unsigned n = (unsigned)std::min<int64_t>(148 * std::max(1, 2048 / threads), a.rows);
    if (threads <= 128) k_norm_units<T, WIDE, 4, 2><<<n, threads, 0, s>>>(a);
    else if (threads <= 256) k_norm_units<T, WIDE, 8, 2><<<n, threads, 0, s>>>(a);
    else if (threads <= 512) k_norm_units<T, WIDE, 16, 2><<<n, threads, 0, s>>>(a);
    else k_norm_units<T, WIDE, 32, 2><<<n, threads, 0, s>>>(a);
}
template <class T>
void forward(const wc_block_norm_args& a, cudaStream_t s) {
    const size_t e = sizeof(T);
    if (!a.rows) return;
    if (units_ok(a) && unit_rows(a.y, a.ld_y, e) && unit_rows(a.n, a.ld_n, e)) forward_as<T, true>(a, s);
    else forward_as<T, false>(a, s);
}

}  // namespace

uint64_t block_norm_workspace(const wc_block_norm_args& a) { return Plan(a).floats(a) * sizeof(float) + 16; }

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
