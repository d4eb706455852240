// dw = x8^T dy with x8 kept in 8 bits, and db = the column sums of dy, on the
// tensor cores (tcgen05, f32 accumulators in TMEM).
//
// A stored value is a whole number times a power of two, so it is exact in
// bf16; dy is exact as the sum of 1 (bf16), 2 (f16) or 3 (f32) bf16 numbers,
// its parts. The products are therefore those of the 32-bit form, and only the
// f32 accumulation rounds. Parts of f16 and f32, and a bf16 dy whose rows TMA
// cannot address, are first laid out in the workspace by a kernel of their own.
//
// Both operands are summed over the rows, their slow axis, so both are MN-major
// in shared memory: a stage holds 64 rows, 64 columns of a row being one
// 128-byte swizzled line. A CTA's tile of dw is MT x 128 columns (of dy, the M
// of the product) by `bk` channels of x8 (its N, any multiple of 32: little is
// converted that is not used):
//   producers   (2 warps) x8's bytes and units, and dy, into shared memory
//   converters  (2 teams of 8 warps, a stage each in turn) x8 to bf16 in shared
//               memory; and the epilogue out of TMEM
//   issuer      (1 warp) the products
//   column sums (1 warp) db from the dy tiles in shared memory, as products
//               with ones
// The work is tiles x stages units dealt in equal runs to the CTAs; a tile
// that falls to several is joined from their partial results by a second
// kernel, in a fixed order.
//
// On a B200 8192 x 4096 x 4096 in bf16 takes 282 us in a burst, 330 when it goes on (0.97
// and 0.83 of the 1.63 PFLOP/s that a library product reaches: shared memory, which
// converted operands cross twice), 606208 x 192 x 96 86 to 88 us with db (2.7 of 6.5
// TB/s: conversion, and the column sums), 183 with dy in f16 and 294 in f32.
#include <cuda.h>

#include <algorithm>
#include <stdexcept>

#include "kernels.h"
#include "train.cuh"
#include "umma.cuh"

namespace wctrain {

namespace {

constexpr int BK = 64;           // rows of a stage
constexpr int RAW = BK * 64, GROUP = BK * 128;  // bytes of 64 columns of a stage, as bytes and as bf16
constexpr int UNIT_WORDS = 3, UNITS = BK * UNIT_WORDS * 4;  // a stage's units: up to 8 of a row, in whole words
constexpr int TEAM = 256, CONVERTERS = 2 * TEAM, THREADS = CONVERTERS + 128;
constexpr int MAX_STAGES = 8, MAX_CTAS = 148;
constexpr int RING = 230912;  // shared memory of the stages: 3 of the widest tile's operands, 3 of its dy, 2 of its x8
constexpr uint32_t TMEM_COLS = 512;

struct Plan {
    int mt, bk, ktiles, ntiles, ctas, joined, kept, whole, limit, parts, operands, dys, xs;
    int steps;              // stages of a tile
    int64_t units;          // tiles x steps, below 2^31
    int64_t split_ld;       // elements of a row of dy's parts in the workspace; 0: dy as it is
    __host__ __device__ int x_groups() const { return (bk + 63) / 64; }
    // a stage of each ring: x8 as bytes and its units, dy's parts, x8 as bf16
    __host__ __device__ int x_bytes() const { return x_groups() * RAW + UNITS; }
    __host__ __device__ int dy_bytes() const { return parts * mt * 2 * GROUP; }
    __host__ __device__ int operand_bytes() const { return x_groups() * GROUP; }
    // the CTA that a unit falls to
    __host__ __device__ int owner(int64_t u) const { return (int)(((u + 1) * ctas - 1) / units); }
    __host__ __device__ int ring_bytes() const { return operands * operand_bytes() + dys * dy_bytes() + xs * x_bytes(); }
};

struct Shared {
    uint64_t x_full[MAX_STAGES], x_empty[MAX_STAGES], dy_full[MAX_STAGES], dy_empty[MAX_STAGES];
    uint64_t op_full[MAX_STAGES], op_empty[MAX_STAGES], acc_full, acc_empty, drained;
    uint32_t tmem;
    int failed;
};

// A place in a ring of stages and the parity of its barriers
struct Place {
    int count, slot = 0;
    uint32_t phase = 0;
    __device__ Place(int n) : count(n) {}
    __device__ void next() {
        if (++slot == count) slot = 0, phase ^= 1;
    }
};

__device__ __forceinline__ uint64_t desc_mn(uint32_t saddr) {
    // MN-major, 128-byte swizzle: GROUP bytes to the next 64 columns (leading), 1024 to the next 8 rows (stride)
    uint64_t d = 0;
    d |= (uint64_t)((saddr >> 4) & 0x3FFFu);
    d |= (uint64_t)(GROUP >> 4) << 16;
    d |= (uint64_t)(1024u >> 4) << 32;
    d |= (uint64_t)1u << 46;
    d |= (uint64_t)2u << 61;
    return d;
}

__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
                 "l"(map), "r"(x), "r"(y), "r"(z), "r"(umma::smem_u32(bar))
                 : "memory");
}
// The product and the commit (umma.cuh) by one elected lane of a converged warp.
__device__ __forceinline__ void mma_one(uint32_t tmem_d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p, e;\n\t"
        "elect.sync _|e, 0xffffffff;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(tmem_d),
        "l"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
}
__device__ __forceinline__ void commit_one(uint64_t* bar) {
    asm volatile(
        "{\n\t.reg .pred e;\n\t"
        "elect.sync _|e, 0xffffffff;\n\t"
        "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}\n" ::"r"(umma::smem_u32(bar))
        : "memory");
}
__device__ __forceinline__ void arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(umma::smem_u32(bar)) : "memory");
}

// Bytes 0 and 2 of `w` as a pair of bf16 times `unit` (a bf16 pair). A byte's
// low seven bits are the mantissa of 128 + them; its sign bit, worth -128, is
// the exponent step from 128 to 256: (128 + low) - (128 or 256) is the byte.
__device__ __forceinline__ uint32_t even_bytes(uint32_t w, __nv_bfloat162 unit) {
    const uint32_t a = (w & 0x007f007fu) | 0x43004300u, b = (w & 0x00800080u) | 0x43004300u;
    const __nv_bfloat162 v = __hmul2(__hsub2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b)), unit);
    return *reinterpret_cast<const uint32_t*>(&v);
}
// 8 bytes to 8 bf16; of each four, the middle two change places (so do the tile's channels, see channel())
__device__ __forceinline__ uint4 eight_bytes(uint32_t x, uint32_t y, __nv_bfloat162 unit) {
    return make_uint4(even_bytes(x, unit), even_bytes(x >> 8, unit), even_bytes(y, unit), even_bytes(y >> 8, unit));
}
__device__ __forceinline__ constexpr int channel(int i) { return (i & ~3) | (i & 1) << 1 | (i >> 1 & 1); }

// Part `p` of v as bf16 and what is left for the next ones. An infinity or NaN goes whole into the first.
__device__ __forceinline__ float part_of(float& v) {
    const float hi = __bfloat162float(__float2bfloat16_rn(v));
    v = isfinite(hi) ? v - hi : 0.0f;
    return hi;
}

// dy's parts into the workspace: [parts][rows][ld], columns past the width zero.
template <class T, int P>
__global__ void __launch_bounds__(256) k_split(const T* __restrict__ dy, int64_t rows, int64_t n, int64_t ld_dy, bool vec,
                                               __nv_bfloat16* __restrict__ out, int64_t ld) {
    const int64_t chunks = ld / 8, total = rows * chunks;
    for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < total; i += gridDim.x * 256ll) {
        const int64_t t = i / chunks, c = (i - t * chunks) * 8;
        const T* from = dy + t * ld_dy + c;
        alignas(16) T e[8];
        if (vec && c + 8 <= n) {
#pragma unroll
            for (int k = 0; k < (int)sizeof(T) / 2; ++k) reinterpret_cast<uint4*>(e)[k] = reinterpret_cast<const uint4*>(from)[k];
        } else {
#pragma unroll
            for (int k = 0; k < 8; ++k) e[k] = c + k < n ? from[k] : from_f<T>(0.0f);
        }
        float v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = to_f(e[k]);
#pragma unroll
        for (int q = 0; q < P; ++q) {
            float h[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) h[k] = part_of(v[k]);
            *reinterpret_cast<uint4*>(out + (q * rows + t) * ld + c) = umma::pack_chunk(h);
        }
    }
}

// W channels of one column of dw, `ld` apart, stored or (32-bit results) added to what is there. The operand's
// channels lie in channel()'s order.
template <int W, class T>
__device__ __forceinline__ void put(T* p, int64_t ld, const float* v, int count, bool add) {
#pragma unroll
    for (int i = 0; i < W; i += 8) {
        float o[8] = {};
        if (sizeof(T) == 4 && add)
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (i + j < count) o[j] = to_f(p[j * ld]);
#pragma unroll
        for (int j = 0; j < 8; ++j, p += ld)
            if (i + j < count) *p = from_f<T>(o[j] + v[channel(i + j)]);
    }
}
// W consecutive f32 columns of this thread's TMEM lane
__device__ __forceinline__ void tmem_load(uint32_t at, float (&v)[32]) { umma::tmem_ld32(at, v); }
__device__ __forceinline__ void tmem_load(uint32_t at, float (&v)[16]) {
    uint32_t r[16];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(at));
    umma::tmem_wait_ld();
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}

// A run of stages of one tile that is summed in TMEM. The tensor core's f32
// accumulation drops the bits below the sum's last place, always towards zero:
// nothing while the products' bits still fit, up to 6e-8 of the result for each
// product of 16 rows (4 a stage) of a long sum. Values of one sign lose 1.8e-6
// in 40 stages, 4e-5 in 240, 4.7e-4 in 2048 (measured). A share therefore goes
// in runs, which are added up in global memory, each thread the values it wrote
// itself: at most RUN stages, and RUN_BF16 where the result is rounded to bf16
// (at most 6e-5, a 32nd of the least that its rounding can move a value by).
// Each run more is a tile written and read: 8192 x 4096 x 4096 takes 593 us in
// f16 for 523 in one run, in bf16 332 in runs of 64 for 282 in one of 128.
constexpr int RUN = 40, RUN_BF16 = 256;

// The units (a stage of a tile each) that fall to a CTA, in order. A share is
// what it has of one tile, cut into runs.
struct Walk {
    int u, end, s;            // unit, end of the CTA's, its stage
    int kt, nt;               // its tile: channels fastest
    int in_run;               // stages of the run before this one
    bool whole, head, begins; // the share is the whole tile; the CTA's first share; the share's first run
    __device__ explicit Walk(const Plan& p) {
        u = (int)(p.units * blockIdx.x / p.ctas), end = (int)(p.units * (blockIdx.x + 1) / p.ctas);
        const int tile = u / p.steps;
        s = u - tile * p.steps, nt = tile / p.ktiles, kt = tile - nt * p.ktiles;
        head = true;
        share(p);
    }
    __device__ void share(const Plan& p) { in_run = 0, begins = true, whole = s == 0 && end - u >= p.steps; }
    __device__ bool more() const { return u < end; }
    __device__ bool share_ends(const Plan& p) const { return u + 1 == end || s + 1 == p.steps; }
    __device__ bool run_ends(const Plan& p) const { return share_ends(p) || in_run + 1 == p.limit; }
    // the stages from this one to the end of its run, and past all of them
    __device__ int run_length(const Plan& p) const { return min(min(end - u, p.steps - s), p.limit - in_run); }
    __device__ void skip(const Plan& p, int n) {
        u += n - 1, s += n - 1, in_run += n - 1;
        next(p);
    }
    __device__ void next(const Plan& p) {
        ++u, ++in_run;
        if (++s == p.steps) {
            s = 0, head = false;
            if (++kt == p.ktiles) kt = 0, ++nt;
            share(p);
        } else if (in_run == p.limit) {
            in_run = 0, begins = false;
        }
    }
};

template <int P, int MT>
__global__ void __launch_bounds__(THREADS, 1)
    k_wgrad8(wc_act8_wgrad_args a, Plan p, const __grid_constant__ CUtensorMap map_q,
             const __grid_constant__ CUtensorMap map_dy, float* part, float* part_db, uint64_t wait_ns) {
    constexpr int GROUPS = 2 * MT;  // of 64 columns of dy
    extern __shared__ uint8_t raw[];
    __shared__ Shared sh;
    uint8_t* operands = raw + ((1024 - (umma::smem_u32(raw) & 1023)) & 1023);
    uint8_t* dys = operands + p.operands * p.operand_bytes();
    uint8_t* xs = dys + p.dys * p.dy_bytes();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int x_groups = p.x_groups();
    volatile int* failed = &sh.failed;

    if (threadIdx.x == 0) {
        for (int i = 0; i < MAX_STAGES; ++i) {
            umma::mbar_init(&sh.x_full[i], 1 + 32);  // the bytes, and each lane's share of the units
            umma::mbar_init(&sh.x_empty[i], TEAM / 32);
            umma::mbar_init(&sh.dy_full[i], 1);
            umma::mbar_init(&sh.dy_empty[i], 2);  // the issuer's commit, the column sums
            umma::mbar_init(&sh.op_full[i], TEAM / 32);
            umma::mbar_init(&sh.op_empty[i], 1);
        }
        umma::mbar_init(&sh.acc_full, 1);
        umma::mbar_init(&sh.acc_empty, CONVERTERS / 32);
        umma::mbar_init(&sh.drained, 1);
        sh.failed = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 0) umma::tmem_alloc(&sh.tmem, TMEM_COLS);
    umma::fence_before_sync();
    __syncthreads();
    umma::fence_after_sync();
    const uint32_t tmem = sh.tmem;
    Walk walk(p);
    Place x{p.xs}, dy{p.dys}, op{p.operands};
    // A wait that runs out makes every role give up: products and copies in flight are waited for, what the CTA had still
    // to write becomes NaN, and the tensor memory is released. What a role that gave up owes to others stays undone, so
    // that their waits run out too. wait_all: the same for a whole warp.
    auto wait = [&](uint64_t* bar, uint32_t parity) {
        if (sleep_on(bar, parity, wait_ns)) return true;
        if (!*failed && wait_ns > SLEEP_NS && umma::mbar_wait(bar, parity, wait_ns)) return true;
        *failed = 1;
        return false;
    };
    auto wait_all = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, wait(bar, parity)) != 0; };

    if (warp == 0) {  // ------------------------------------------- issuer
        // Little to compute between two products: that is what keeps the tensor core waiting. The warp stays together
        // and one lane issues, so that the operands are uniform; a stage's descriptors differ in the address field only.
        const uint32_t idesc = umma::idesc_bf16(128, p.bk) | (1u << 15) | (1u << 16);
        const uint64_t a_first = desc_mn(umma::smem_u32(dys)), b_first = desc_mn(umma::smem_u32(operands));
        const uint32_t a_step = p.dy_bytes() >> 4, b_step = p.operand_bytes() >> 4;
        uint32_t done = 0;
        bool ok = true;
        while (ok && walk.more()) {
            const int n = walk.run_length(p);
            if (done) ok = wait_all(&sh.acc_empty, (done - 1) & 1);
            for (int i = 0; ok && i < n; ++i) {
                // dy's copy is waited for here, not through the converters: the product reads it with no one between
                ok = wait_all(&sh.dy_full[dy.slot], dy.phase);
                ok = ok && wait_all(&sh.op_full[op.slot], op.phase);
                umma::fence_after_sync();
                if (ok) {
                    const uint64_t A = a_first + dy.slot * a_step, B = b_first + op.slot * b_step;
#pragma unroll
                    for (int m = 0; m < MT; ++m)
#pragma unroll
                        for (int q = 0; q < P; ++q)
#pragma unroll
                            for (int k = 0; k < BK / 16; ++k)
                                mma_one(tmem + (m * P + q) * p.bk, A + ((q * GROUPS + m * 2) * GROUP >> 4) + k * 128, B + k * 128,
                                        idesc, k ? 1 : i);
                    commit_one(&sh.op_empty[op.slot]);
                    commit_one(&sh.dy_empty[dy.slot]);
                }
                dy.next(), op.next();
            }
            if (ok) commit_one(&sh.acc_full), ++done;
            walk.skip(p, n);
        }
        // Every issued product has finished before TMEM is given back, also where no one waits for it any more. (On a barrier
        // of its own: acc_full would tell of a whole run.)
        commit_one(&sh.drained);
        umma::mbar_wait(&sh.drained, 0, umma::DRAIN_NS);
    } else if (warp == 1) {  // ----------------------------- dy's producer
        if (lane == 0) {
            const uint32_t ring = umma::smem_u32(dys);
            int it = 0;
            for (; walk.more(); walk.next(p), dy.next(), ++it) {
                if (it >= p.dys && !wait(&sh.dy_empty[dy.slot], dy.phase ^ 1)) break;
                const int n0 = walk.nt * (MT * 128);
                umma::expect_tx(&sh.dy_full[dy.slot], p.dy_bytes());
                uint32_t to = ring + dy.slot * p.dy_bytes();
#pragma unroll
                for (int q = 0; q < P; ++q)
#pragma unroll
                    for (int g = 0; g < GROUPS; ++g, to += GROUP)
                        tma_load(to, &map_dy, n0 + 64 * g, walk.s * BK, q, &sh.dy_full[dy.slot]);
            }
            // the copies in flight land before the CTA leaves, also where no one waits for them any more
            for (int i = it > p.dys ? it - p.dys : 0; i < it; ++i)
                umma::mbar_wait(&sh.dy_full[i % p.dys], (i / p.dys) & 1, umma::DRAIN_NS);
        }
        __syncwarp();
    } else if (warp == 2) {  // ----------------------------- x8's producer
        // The units' rows have any alignment: the words that hold a row's are copied, and read at its first one's offset. (So
        // are the up to 3 bytes around the matrix that share a word with it, and not used. Copying the last word in part
        // cost 8192 x 4096 x 4096 in bf16 291 us for 284.)
        const int64_t blocks = (a.k + 31) / 32;
        const uint32_t ring = umma::smem_u32(xs);
        int it = 0;
        for (; walk.more(); walk.next(p), x.next(), ++it) {
            if (it >= p.xs && !wait_all(&sh.x_empty[x.slot], x.phase ^ 1)) break;
            const uint32_t to = ring + x.slot * p.x_bytes();
            const int k0 = walk.kt * p.bk, t0 = walk.s * BK;
            if (lane == 0) {
                umma::expect_tx(&sh.x_full[x.slot], x_groups * RAW);
                for (int g = 0; g < x_groups; ++g) tma_load(to + g * RAW, &map_q, k0 + 64 * g, t0, 0, &sh.x_full[x.slot]);
            }
            const int count = (int)min((int64_t)(p.bk / 32), blocks - k0 / 32);
#pragma unroll
            for (int i = 0; i < BK / 32; ++i) {
                const int row = i * 32 + lane;
                if ((int64_t)t0 + row < a.rows) {
                    const uintptr_t from = reinterpret_cast<uintptr_t>(a.scale + ((int64_t)t0 + row) * blocks + k0 / 32);
                    const int words = (int)((from & 3) + count + 3) >> 2;
#pragma unroll
                    for (int w = 0; w < UNIT_WORDS; ++w)
                        if (w < words)
                            asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(to + x_groups * RAW + (w * BK + row) * 4),
                                         "l"((from & ~(uintptr_t)3) + 4 * w)
                                         : "memory");
                }
            }
            asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(umma::smem_u32(&sh.x_full[x.slot])) : "memory");
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        if (lane == 0)
            for (int i = it > p.xs ? it - p.xs : 0; i < it; ++i)
                umma::mbar_wait(&sh.x_full[i % p.xs], (i / p.xs) & 1, umma::DRAIN_NS);
        __syncwarp();
    } else if (warp == 3) {  // -------------------------------- column sums
        // Eight columns at a time as products with ones: 8 rows of 8 columns are a matrix fragment, and 4 products a stage
        // replace 64 additions a column (606208 x 192 x 96 takes 87 us, with additions it took 92; without db 68). Lanes
        // 4 j to 4 j + 3 keep the j-th eight of every 64 columns. The tiles of a column block take the stages in turn, so
        // that no CTA has more of this than another; a CTA keeps its sums until the column block ends.
        bool ok = true;
        float sum[4 * MT] = {};
        int turn = walk.s % p.ktiles;  // the tile whose stage this is
        for (; walk.more(); walk.next(p), dy.next()) {
            if (walk.s == 0) turn = 0;
            ok = ok && wait_all(&sh.dy_full[dy.slot], dy.phase);
            if (a.db && ok && walk.kt == (p.whole ? 0 : turn)) {
                const uint32_t B = umma::smem_u32(dys) + dy.slot * p.dy_bytes() + lane * 128;
                const int64_t left = a.n - (int64_t)walk.nt * (MT * 128);
#pragma unroll
                for (int h = 0; h < 2 * MT; ++h) {
                    if (h * 64 >= left) break;
#pragma unroll
                    for (int g = 0; g < 8; ++g) {
                        float d0 = 0.0f, d1 = 0.0f, x0 = 0.0f, x1 = 0.0f;  // (two rows of the result, all alike, are enough)
                        for (int q = 0; q < P; ++q) {
                            const uint32_t at = B + (q * GROUPS + h) * GROUP + ((g ^ (lane & 7)) << 4);
                            uint32_t b[8];
#pragma unroll
                            for (int r = 0; r < 2; ++r)
                                asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                                             : "=r"(b[4 * r]), "=r"(b[4 * r + 1]), "=r"(b[4 * r + 2]), "=r"(b[4 * r + 3])
                                             : "r"(at + r * 32 * 128));
#pragma unroll
                            for (int k = 0; k < 8; k += 2)
                                asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %4, %4, %4}, {%5, %6}, {%0, %1, "
                                    "%2, %3};"
                                    : "+f"(d0), "+f"(d1), "+f"(x0), "+f"(x1)
                                    : "r"(0x3f803f80u), "r"(b[k]), "r"(b[k + 1]));
                        }
                        if (lane >> 2 == g) sum[2 * h] += d0, sum[2 * h + 1] += d1;
                    }
                }
            }
            __syncwarp();
            if (ok && lane == 0) arrive(&sh.dy_empty[dy.slot]);
            if (++turn == p.ktiles) turn = 0;
            if (a.db && (walk.u + 1 == walk.end || (walk.s + 1 == p.steps && walk.kt + 1 == p.ktiles))) {
                if (!ok)
                    for (float& v : sum) v = __uint_as_float(0x7fffffffu);
                // the slot of (column block, CTA): their sum grows along the walk
                if (p.whole) {
                    const int64_t n = (int64_t)walk.nt * (MT * 128) + lane * 2;
#pragma unroll
                    for (int h = 0; h < 4 * MT; ++h)
                        if (walk.kt == 0 && n + h / 2 * 64 + (h & 1) < a.n) a.db[n + h / 2 * 64 + (h & 1)] = sum[h];
                    continue;
                }
                float* to = part_db + (int64_t)(walk.nt + blockIdx.x) * 256 + lane * 2;
#pragma unroll
                for (int h = 0; h < 2 * MT; ++h) *reinterpret_cast<float2*>(to + h * 64) = make_float2(sum[2 * h], sum[2 * h + 1]);
                for (float& v : sum) v = 0.0f;
            }
        }
    } else {  // -------------------------------------------------- converters
        const int team = (threadIdx.x - 128) / TEAM, tid = (threadIdx.x - 128) % TEAM, w = warp - 4;
        // A thread has one row of a stage and there 16 channels of every group of 64; 8 threads (two rows) then read 128
        // bytes in a row and store to 8 different chunks of a line.
        const int64_t blocks = (a.k + 31) / 32;
        const int ar = tid >> 2, ac = (tid & 3) * 2;
        const uint32_t raw_at = ar * 64 + ac * 8, lo_at = ar * 128 + ((ac ^ (ar & 7)) << 4), hi_at = ar * 128 + (((ac + 1) ^ (ar & 7)) << 4);
        // where a row's units start in their words, up to the stage's and the tile's share
        const uint32_t unit_row = (uint32_t)(reinterpret_cast<uintptr_t>(a.scale) + ar * blocks), unit_stage = (uint32_t)(BK * blocks);
        constexpr int X_GROUPS = 4;  // at most
        bool ok = true;
        uint32_t done = 0, it = 0;
        for (; walk.more(); walk.next(p), ++it, x.next(), op.next()) {
            if (ok && (int)(it & 1) == team) {
                ok = wait_all(&sh.x_full[x.slot], x.phase);
                const uint8_t* X = xs + x.slot * p.x_bytes() + raw_at;
                const uint32_t first = ((unit_row + walk.s * unit_stage + walk.kt * (p.bk / 32)) & 3) + (ac >> 2);
                const uint8_t* units = xs + x.slot * p.x_bytes() + x_groups * RAW + ar * 4;
                // Rows past the end come as bytes 0; their units are whatever the memory held, and have to be a number:
                // 0 times a finite one is 0. (A NaN block, code 255, is 0 times infinity.)
                const bool there = (int64_t)walk.s * BK + ar < a.rows;
                uint4 q[X_GROUPS];
                uint32_t code[X_GROUPS];
#pragma unroll
                for (int g = 0; g < X_GROUPS; ++g) {
                    if (g >= x_groups) break;
                    q[g] = *reinterpret_cast<const uint4*>(X + g * RAW);
                    code[g] = units[((first + 2 * g) >> 2) * (BK * 4) + ((first + 2 * g) & 3)];
                }
                if (it >= (uint32_t)p.operands) ok = ok && wait_all(&sh.op_empty[op.slot], op.phase ^ 1);
                uint8_t* A = operands + op.slot * p.operand_bytes();
#pragma unroll
                for (int g = 0; g < X_GROUPS; ++g) {
                    if (g >= x_groups) break;
                    const uint32_t uu = (there ? code[g] : 127u) * 0x00800080u;
                    const __nv_bfloat162 unit2 = *reinterpret_cast<const __nv_bfloat162*>(&uu);
                    *reinterpret_cast<uint4*>(A + g * GROUP + lo_at) = eight_bytes(q[g].x, q[g].y, unit2);
                    *reinterpret_cast<uint4*>(A + g * GROUP + hi_at) = eight_bytes(q[g].z, q[g].w, unit2);
                }
                umma::fence_async_smem();
                __syncwarp();
                if (ok && lane == 0) arrive(&sh.op_full[op.slot]), arrive(&sh.x_empty[x.slot]);
            }
            if (!walk.run_ends(p)) continue;
            // the tile out of TMEM: every fourth warp has the lanes of one quarter
            ok = ok && wait_all(&sh.acc_full, done & 1);
            umma::fence_after_sync();
            constexpr int W = P == 1 ? 32 : 16;  // channels at a time; a lane is a column of dw, 32 next to each other
            const int64_t k0 = (int64_t)walk.kt * p.bk;
            const int row = (warp & 3) * 32 + lane, runs = p.bk / W;
            for (int i = w >> 2; i < MT * runs; i += CONVERTERS / 128) {
                const int m = i / runs, c = i % runs * W;
                const int64_t n = (int64_t)walk.nt * (MT * 128) + m * 128 + row;
                float v[W];
                const uint32_t from = tmem + ((uint32_t)(warp & 3) * 32 << 16) + m * P * p.bk + c;
                tmem_load(from + (P - 1) * p.bk, v);  // the smallest part first
#pragma unroll
                for (int q = P - 2; q >= 0; --q) {
                    float y[W];
                    tmem_load(from + q * p.bk, y);
#pragma unroll
                    for (int e = 0; e < W; ++e) v[e] += y[e];
                }
                if (!ok)
                    for (float& e : v) e = __uint_as_float(0x7fffffffu);
                // A share that is not the whole tile is left to the second kernel, in the CTA's first or second place. A
                // 16-bit tile in several runs is summed up in the second (the CTA's last share comes after it), then rounded.
                const bool wide = a.out_type == WC_F32;
                float* kept = part + (((int64_t)(2 * blockIdx.x + (walk.head && !walk.whole ? 0 : 1)) * MT + m) * p.bk + c) * 128 + row;
                if (!wide && walk.whole && !walk.begins && walk.share_ends(p))
#pragma unroll
                    for (int e = 0; e < W; ++e) v[channel(e)] += kept[e * 128];
                if (!walk.whole || !(wide || walk.share_ends(p))) {
                    put<W>(kept, 128, v, W, !walk.begins);
                } else if (n < a.n) {
                    const int count = (int)min((int64_t)W, a.k - k0 - c);
                    const int64_t to = (k0 + c) * a.n + n;
                    if (a.out_type == WC_F32) put<W>(static_cast<float*>(a.dw) + to, a.n, v, count, !walk.begins);
                    else if (a.out_type == WC_F16) put<W>(static_cast<__half*>(a.dw) + to, a.n, v, count, false);
                    else put<W>(static_cast<__nv_bfloat16*>(a.dw) + to, a.n, v, count, false);
                }
            }
            umma::fence_before_sync();
            __syncwarp();
            if (ok && lane == 0) arrive(&sh.acc_empty);
            ++done;
        }
    }
    umma::fence_before_sync();
    __syncthreads();
    if (warp == 0) umma::tmem_dealloc(tmem, TMEM_COLS);
}

// The tiles that fall to several CTAs, at most one for each boundary between
// two CTAs: the CTAs' numbers, and the slot of the first one's partial result
// (the others' is their first, 2 c).
struct Split {
    int tile, slot;
    short c0, c1;
};
struct Splits {
    int n;
    Split at[MAX_CTAS];
    Splits(const Plan& p) : n(0) {
        auto start = [&](int64_t c) { return p.units * c / p.ctas; };
        for (int c = 0; c + 1 < p.ctas; ++c) {
            const int64_t cut = start(c + 1), tile = cut / p.steps, u0 = tile * p.steps;
            if (cut == u0) continue;                                                  // between two tiles
            if (n && at[n - 1].tile == tile) at[n - 1].c1 = (short)(c + 1);           // one more boundary of the same
            else at[n++] = Split{(int)tile, 2 * c + (start(c) >= u0 ? 0 : 1), (short)c, (short)(c + 1)};
        }
    }
};

// Joins the split tiles (one a blockIdx.y, then a column block of db each). A
// thread has 4 columns of a channel, or of db; with many CTAs to a tile they
// are dealt to blockDim.y threads and those joined in order.
constexpr int JOINERS = 256;
template <class T>
__global__ void __launch_bounds__(JOINERS) k_wgrad8_join(wc_act8_wgrad_args a, Plan p, const __grid_constant__ Splits splits,
                                                         const float* part, const float* part_db) {
    __shared__ float4 s[JOINERS];
    const int i = blockIdx.x * blockDim.x + threadIdx.x, cols = p.mt * 128;
    const bool bias = (int)blockIdx.y >= splits.n;
    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    auto add = [&](const float* from) {
        const float4 w = *reinterpret_cast<const float4*>(from);
        v.x += w.x, v.y += w.y, v.z += w.z, v.w += w.w;
    };
    int64_t k = 0, n;
    bool in;
    if (bias) {
        const int nt = blockIdx.y - splits.n;
        const int64_t per = (int64_t)p.ktiles * p.steps;
        n = (int64_t)nt * cols + i * 4;
        in = i < cols / 4 && n < a.n;
        if (in) {
            const int c0 = p.owner(nt * per), c1 = p.owner((nt + 1) * per - 1);
            for (int j = c0 + (int)threadIdx.y; j <= c1; j += blockDim.y)
                add(part_db + ((int64_t)(nt + j) * 64 + i) * 4);
        }
    } else {
        const Split& cut = splits.at[blockIdx.y];
        const int m = i / (p.bk * 32), c = i / 32 % p.bk;
        k = (int64_t)(cut.tile % p.ktiles) * p.bk + c, n = (int64_t)(cut.tile / p.ktiles) * cols + m * 128 + i % 32 * 4;
        in = i < p.bk * cols / 4 && n < a.n && k < a.k;
        if (in)
#pragma unroll 4
            for (int j = cut.c0 + (int)threadIdx.y; j <= cut.c1; j += blockDim.y)
                add(part + ((int64_t)(j == cut.c0 ? cut.slot : 2 * j) * p.bk * cols + i * 4));
    }
    if (blockDim.y > 1) {
        s[threadIdx.y * blockDim.x + threadIdx.x] = v;
        __syncthreads();
        if (threadIdx.y) return;
        for (int j = 1; j < (int)blockDim.y; ++j) {
            const float4 w = s[j * blockDim.x + threadIdx.x];
            v.x += w.x, v.y += w.y, v.z += w.z, v.w += w.w;
        }
    }
    if (!in) return;
    const float e[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if (n + j >= a.n) break;
        if (bias) a.db[n + j] = e[j];
        else static_cast<T*>(a.dw)[k * a.n + n + j] = from_f<T>(e[j]);
    }
}

Plan plan_of(const wc_act8_wgrad_args& a) {
    Plan p{};
    p.parts = a.type == WC_F32 ? 3 : a.type == WC_F16 ? 2 : 1;
    const bool as_is = p.parts == 1 && ((uintptr_t)a.dy & 15) == 0 && (a.ld_dy * 2) % 16 == 0;
    p.split_ld = as_is ? 0 : (a.n + 7) / 8 * 8;
    p.steps = (int)((a.rows + BK - 1) / BK);
    // TMEM holds 512 columns: MT x parts x bk sums
    p.mt = p.parts == 1 && a.n > 128 ? 2 : 1;
    const int64_t widest = p.parts == 3 ? 160 : 256, kt = (a.k + widest - 1) / widest;
    p.bk = (int)(((a.k + kt - 1) / kt + 31) / 32 * 32);
    p.ktiles = (int)((a.k + p.bk - 1) / p.bk);
    p.ntiles = (int)((a.n + p.mt * 128 - 1) / (p.mt * 128));
    p.units = (int64_t)p.ktiles * p.ntiles * p.steps;
    // Short sums take a CTA a tile: it has no partial results, and the second kernel is not launched (which takes as long
    // as some three stages)
    const int64_t tiles = (int64_t)p.ktiles * p.ntiles;
    p.whole = p.steps <= 4 && tiles <= MAX_CTAS;
    p.ctas = (int)std::max<int64_t>(1, p.whole ? tiles : std::min<int64_t>(MAX_CTAS, p.steps == 1 ? p.units : (p.units + 1) / 2));
    p.joined = p.steps > 1 && (p.units % p.ctas != 0 || (p.units / p.ctas) % p.steps != 0);
    p.limit = a.out_type == WC_BF16 ? RUN_BF16 : RUN;
    p.kept = p.joined || (a.out_type != WC_F32 && p.steps > p.limit);
    // Converters work a stage or two ahead of the products; what is left holds copies in flight, of dy and x8 in turn.
    // x8's ring has an even number of places, so that a place is always the same team's. With an odd one a team that is
    // ahead could take the barrier's phase before last for the one it waits for, when the copy between the two (the
    // other team's) is late: it would convert what is not there yet and free a place that is still in use.
    p.operands = 3, p.xs = 2, p.dys = 2;
    for (bool grew = true; grew;) {
        grew = false;
        const auto grow = [&](int& n, int by) {
            if (n + by > MAX_STAGES) return;
            n += by;
            if (p.ring_bytes() <= RING) grew = true;
            else n -= by;
        };
        grow(p.dys, 1), grow(p.dys, 1), grow(p.xs, 2);
    }
    return p;
}

uint64_t parts_bytes(const wc_act8_wgrad_args& a, const Plan& p) {
    return ((uint64_t)p.parts * a.rows * p.split_ld * 2 + 255) / 256 * 256;
}

using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                            const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                            CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
Encode encoder() {
    static const Encode fn = [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult st;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &st) != cudaSuccess ||
            st != cudaDriverEntryPointSuccess)
            throw std::runtime_error("cuTensorMapEncodeTiled is not available");
        return reinterpret_cast<Encode>(f);
    }();
    return fn;
}

// `planes` row-major matrices as boxes of 64 columns x 64 rows, zeros outside
CUtensorMap map_of(const void* base, CUtensorMapDataType type, int64_t width, int64_t rows, int planes, int64_t row_bytes,
                   CUtensorMapSwizzle swizzle) {
    CUtensorMap m;
    const cuuint64_t dims[3] = {(cuuint64_t)width, (cuuint64_t)rows, (cuuint64_t)planes};
    const cuuint64_t strides[2] = {(cuuint64_t)row_bytes, (cuuint64_t)(row_bytes * rows)};
    const cuuint32_t box[3] = {64, BK, 1}, step[3] = {1, 1, 1};
    if (encoder()(&m, type, 3, const_cast<void*>(base), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
        throw std::runtime_error("cuTensorMapEncodeTiled refused a tensor map");
    return m;
}

template <int P, class T>
void launch_split(const wc_act8_wgrad_args& a, const Plan& p, __nv_bfloat16* to, cudaStream_t s) {
    const bool vec = ((uintptr_t)a.dy & 15) == 0 && (a.ld_dy * sizeof(T)) % 16 == 0;
    const int64_t blocks = (a.rows * (p.split_ld / 8) + 255) / 256;
    k_split<T, P><<<(unsigned)std::min<int64_t>(blocks, 148 * 16), 256, 0, s>>>(static_cast<const T*>(a.dy), a.rows, a.n, a.ld_dy,
                                                                              vec, to, p.split_ld);
}

template <int P, int MT>
void launch_tile(const wc_act8_wgrad_args& a, const Plan& p, const __nv_bfloat16* split, float* part, float* part_db, cudaStream_t s) {
    const int64_t pitch = (a.k + 31) / 32 * 32;
    const CUtensorMap q = map_of(a.q, CU_TENSOR_MAP_DATA_TYPE_UINT8, pitch, a.rows, 1, pitch, CU_TENSOR_MAP_SWIZZLE_NONE);
    const CUtensorMap dy = p.split_ld
        ? map_of(split, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, a.n, a.rows, P, p.split_ld * 2, CU_TENSOR_MAP_SWIZZLE_128B)
        : map_of(a.dy, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, a.n, a.rows, 1, a.ld_dy * 2, CU_TENSOR_MAP_SWIZZLE_128B);
    const size_t smem = (size_t)p.ring_bytes() + 1024;
    if (!wcdev::raise_smem_limit(reinterpret_cast<const void*>(k_wgrad8<P, MT>), RING + 1024)) return;
    k_wgrad8<P, MT><<<p.ctas, THREADS, smem, s>>>(a, p, q, dy, part, part_db, wait_limit());
}

template <class T>
void launch_join(const wc_act8_wgrad_args& a, const Plan& p, const float* part, const float* part_db, cudaStream_t s) {
    const Splits splits(p);
    int sharers = 0;
    for (int i = 0; i < splits.n; ++i) sharers = std::max(sharers, splits.at[i].c1 - splits.at[i].c0 + 1);
    const int ny = sharers >= 8 ? 32 : 1;
    const dim3 block(JOINERS / ny, ny);
    const int wide = splits.n ? p.bk * p.mt * 32 : p.mt * 32;  // threads that sum up a tile, or db alone
    const dim3 grid((wide + block.x - 1) / block.x, splits.n + (a.db ? p.ntiles : 0));
    k_wgrad8_join<T><<<grid, block, 0, s>>>(a, p, splits, part, part_db);
}

}  // namespace

uint64_t wgrad8_workspace(const wc_act8_wgrad_args& a) {
    if (!a.n || !a.rows) return 0;
    const Plan p = plan_of(a);
    return parts_bytes(a, p) + (uint64_t)(p.ntiles + p.ctas) * 1024 + (p.kept ? (uint64_t)2 * p.ctas * p.mt * 128 * p.bk * sizeof(float) : 0);
}

void launch_wgrad8(const wc_act8_wgrad_args& a, cudaStream_t s) {
    if (!a.rows) {  // empty sums
        cudaMemsetAsync(a.dw, 0, (size_t)a.k * a.n * (a.out_type == WC_F32 ? 4 : 2), s);
        if (a.db) cudaMemsetAsync(a.db, 0, (size_t)a.n * 4, s);
        return;
    }
    const Plan p = plan_of(a);
    __nv_bfloat16* split = static_cast<__nv_bfloat16*>(a.workspace);
    float* part_db = reinterpret_cast<float*>(static_cast<uint8_t*>(a.workspace) + parts_bytes(a, p));
    float* part = part_db + (int64_t)(p.ntiles + p.ctas) * 256;
    if (p.parts == 3) launch_split<3, float>(a, p, split, s);
    else if (p.parts == 2) launch_split<2, __half>(a, p, split, s);
    else if (p.split_ld) launch_split<1, __nv_bfloat16>(a, p, split, s);
    const auto launch = p.parts == 3 ? launch_tile<3, 1> : p.parts == 2 ? launch_tile<2, 1> : p.mt == 2 ? launch_tile<1, 2> : launch_tile<1, 1>;
    launch(a, p, split, part, part_db, s);
    if (!p.joined && (!a.db || p.whole)) return;
    if (a.out_type == WC_F32) launch_join<float>(a, p, part, part_db, s);
    else if (a.out_type == WC_F16) launch_join<__half>(a, p, part, part_db, s);
    else launch_join<__nv_bfloat16>(a, p, part, part_db, s);
}

}  // namespace wctrain
