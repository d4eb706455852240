// dw = x8^T dy with x8 kept in 8 bits, and db = the column sums of dy, on the
// tensor cores (tcgen05, f32 accumulators in TMEM).
//
// A stored value is a whole number times a power of two, so it is exact in
// bf16; dy is exact as the sum of `parts` bf16 numbers (1 for bf16, 2 for f16,
// 3 for f32). The products are therefore those of the 32-bit form, and only
// the f32 accumulation rounds.
//
// Both operands are summed over the rows, their slow axis, so both are MN-major
// in shared memory: a stage holds 64 rows, 64 columns of a row being one
// 128-byte swizzled line. Per CTA, `mt` 128-row tiles of dw (channels of x8)
// by `bn` columns:
//   producer    (1 warp) the bytes of x8, and dy, by TMA
//   converters  (2 teams of 8 warps, a stage each in turn) x8 to bf16 in shared
//               memory; dy too where TMA cannot take it (parts > 1 or an
//               unaligned dy); and the epilogue out of TMEM
//   issuer      (1 warp) the products
//   column sums (2 warps) db from the dy tiles in shared memory
// The work is tiles x stages units dealt in equal runs to the CTAs; a tile
// that falls to several is joined from their partial results by a second
// kernel, in a fixed order.
#include <cuda.h>

#include <algorithm>
#include <stdexcept>

#include "colsum.cuh"
#include "kernels.h"
#include "umma.cuh"

namespace wctrain {

namespace {

constexpr int BK = 64;           // rows of a stage
constexpr int RAW = BK * 64, GROUP = BK * 128;  // bytes of 64 columns of a stage, as bytes and as bf16
constexpr int TEAM = 256, CONVERTERS = 2 * TEAM, THREADS = CONVERTERS + 128;
constexpr int MAX_STAGES = 8, MAX_CTAS = 148;
constexpr int RING = 220 * 1024;  // shared memory of the stages
constexpr uint32_t TMEM_COLS = 512;

// How dy reaches shared memory: by TMA, or through the converters.
enum { TMA, BF16, F16, F32 };
__host__ __device__ constexpr int parts_of(int mode) { return mode == F32 ? 3 : mode == F16 ? 2 : 1; }
__host__ __device__ constexpr int widest(int mode) { return mode == TMA ? 256 : mode == F32 ? 64 : 128; }

struct Plan {
    int mt, bn, ktiles, ntiles, ctas, joined, limit, mode, operands, inputs;
    int steps;              // stages of a tile
    int64_t units;          // tiles x steps, below 2^31
    __host__ __device__ int groups() const { return (bn + 63) / 64; }
    __host__ __device__ int dy_bytes() const { return parts_of(mode) * groups() * GROUP; }
    // a stage of what TMA brings (x8 as bytes, dy) and of what the converters write (x8 as bf16, dy's parts)
    __host__ __device__ int input_bytes() const { return mt * 2 * RAW + (mode == TMA ? dy_bytes() : 0); }
    __host__ __device__ int operand_bytes() const { return mt * 2 * GROUP + (mode == TMA ? 0 : dy_bytes()); }
};

struct Shared {
    uint64_t in_full[MAX_STAGES], in_empty[MAX_STAGES], op_full[MAX_STAGES], op_empty[MAX_STAGES], acc_full, acc_empty;
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

__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap* map, int x, int y, uint64_t* bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
                 "l"(map), "r"(x), "r"(y), "r"(umma::smem_u32(bar))
                 : "memory");
}
// One test that may sleep for up to 100 us: a warp that polls instead takes issue slots and shared-memory cycles from
// the warps it waits for.
__device__ __forceinline__ bool mbar_sleep(uint64_t* bar, uint32_t parity) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}\n"
        : "=r"(done)
        : "r"(umma::smem_u32(bar)), "r"(parity), "r"(100000u)
        : "memory");
    return done != 0;
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
// 8 bytes to 8 bf16; of each four, the middle two change places (the rows of the tile do, see channel())
__device__ __forceinline__ uint4 eight_bytes(uint32_t x, uint32_t y, __nv_bfloat162 unit) {
    return make_uint4(even_bytes(x, unit), even_bytes(x >> 8, unit), even_bytes(y, unit), even_bytes(y >> 8, unit));
}
__device__ __forceinline__ int channel(int row) { return (row & ~3) | (row & 1) << 1 | (row >> 1 & 1); }

// Part `p` of v as bf16 and what is left for the next ones. An infinity or NaN goes whole into the first.
__device__ __forceinline__ float part_of(float& v) {
    const float hi = __bfloat162float(__float2bfloat16_rn(v));
    v = isfinite(hi) ? v - hi : 0.0f;
    return hi;
}

// 8 values of a row as they lie in memory; past the width they are 0
template <class T>
struct Eight {
    uint4 w[sizeof(T) / 2];
    __device__ __forceinline__ void load(const T* p, int64_t n, int64_t width, bool vec) {
        if (vec && n + 8 <= width) {
#pragma unroll
            for (int i = 0; i < (int)sizeof(T) / 2; ++i) w[i] = reinterpret_cast<const uint4*>(p + n)[i];
        } else {
            alignas(16) T e[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) e[i] = n + i < width ? p[n + i] : from_f<T>(0.0f);
#pragma unroll
            for (int i = 0; i < (int)sizeof(T) / 2; ++i) w[i] = reinterpret_cast<const uint4*>(e)[i];
        }
    }
    __device__ __forceinline__ void get(float* v) const {
        alignas(16) T e[8];
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) reinterpret_cast<uint4*>(e)[i] = w[i];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = to_f(e[i]);
    }
};

// W columns of one row of dw: stored, or what is there added to them
template <int W, class T>
__device__ __forceinline__ void store_run(T* p, const float* v, int count, bool vec) {
    if (vec && count >= W) {
        constexpr int E = 16 / sizeof(T);
#pragma unroll
        for (int i = 0; i < W / E; ++i) {
            alignas(16) T e[E];
#pragma unroll
            for (int j = 0; j < E; ++j) e[j] = from_f<T>(v[i * E + j]);
            reinterpret_cast<uint4*>(p)[i] = *reinterpret_cast<const uint4*>(e);
        }
    } else {
#pragma unroll
        for (int i = 0; i < W; ++i)
            if (i < count) p[i] = from_f<T>(v[i]);
    }
}
template <int W>
__device__ __forceinline__ void add_run(float* v, const float* p, int count, bool vec) {
    if (vec && count >= W) {
#pragma unroll
        for (int i = 0; i < W / 4; ++i) {
            const float4 w = reinterpret_cast<const float4*>(p)[i];
            v[4 * i] += w.x, v[4 * i + 1] += w.y, v[4 * i + 2] += w.z, v[4 * i + 3] += w.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < W; ++i)
            if (i < count) v[i] += p[i];
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
// accumulation drops the bits below the sum's last place, about 4e-9 of the
// result for each product of 16 rows, always towards zero; a 32-bit dw
// therefore takes runs of at most RUN stages (below 8e-7) and adds them up in
// global memory, each thread the values it wrote itself. For a 16-bit dw a
// whole segment is one run.
constexpr int RUN = 40;

// The units (a stage of a tile each) that fall to a CTA, in order. A share is
// what it has of one tile, cut into runs.
struct Walk {
    int u, end, tile, s;      // unit, end of the CTA's, their tile and stage
    int in_run;               // stages of the run before this one
    bool whole, head, begins; // the share is the whole tile; the CTA's first share; the share's first run
    __device__ explicit Walk(const Plan& p) {
        u = (int)(p.units * blockIdx.x / p.ctas), end = (int)(p.units * (blockIdx.x + 1) / p.ctas);
        tile = u / p.steps, s = u - tile * p.steps;
        head = true;
        share(p);
    }
    __device__ void share(const Plan& p) { in_run = 0, begins = true, whole = s == 0 && end - u >= p.steps; }
    __device__ bool more() const { return u < end; }
    __device__ bool share_ends(const Plan& p) const { return u + 1 == end || s + 1 == p.steps; }
    __device__ bool run_ends(const Plan& p) const { return share_ends(p) || in_run + 1 == p.limit; }
    __device__ void next(const Plan& p) {
        ++u, ++in_run;
        if (++s == p.steps) s = 0, ++tile, head = false, share(p);
        else if (in_run == p.limit) in_run = 0, begins = false;
    }
};

template <int MODE, int MT, class T>
__global__ void __launch_bounds__(THREADS, 1)
    k_wgrad8(wc_act8_wgrad_args a, Plan p, const __grid_constant__ CUtensorMap map_q,
             const __grid_constant__ CUtensorMap map_dy, float* part, float* part_db) {
    constexpr int P = parts_of(MODE), GROUPS = 2 * MT;
    extern __shared__ uint8_t raw[];
    __shared__ Shared sh;
    uint8_t* operands = raw + ((1024 - (umma::smem_u32(raw) & 1023)) & 1023);
    uint8_t* inputs = operands + p.operands * p.operand_bytes();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int groups = p.groups();
    volatile int* failed = &sh.failed;

    if (threadIdx.x == 0) {
        for (int i = 0; i < p.inputs; ++i) {
            umma::mbar_init(&sh.in_full[i], 1);
            umma::mbar_init(&sh.in_empty[i], TEAM / 32 + (MODE == TMA ? 3 : 0));
        }
        for (int i = 0; i < p.operands; ++i) {
            umma::mbar_init(&sh.op_full[i], TEAM / 32);
            umma::mbar_init(&sh.op_empty[i], MODE == TMA ? 1 : 3);
        }
        umma::mbar_init(&sh.acc_full, 1);
        umma::mbar_init(&sh.acc_empty, CONVERTERS / 32);
        sh.failed = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 0) umma::tmem_alloc(&sh.tmem, TMEM_COLS);
    umma::fence_before_sync();
    __syncthreads();
    umma::fence_after_sync();
    const uint32_t tmem = sh.tmem;
    Walk walk(p);
    Place in{p.inputs}, op{p.operands};
    // A wait that runs out (umma.cuh) makes every role give up: products and copies in flight are waited for, what
    // the CTA had still to write becomes NaN, and the tensor memory is released. wait_all: the same for a whole warp.
    auto wait = [&](uint64_t* bar, uint32_t parity) {
        if (mbar_sleep(bar, parity)) return true;
        if (!*failed && umma::mbar_wait(bar, parity)) return true;
        *failed = 1;
        return false;
    };
    auto wait_all = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, wait(bar, parity)) != 0; };

    if (warp == 0) {  // ------------------------------------------- issuer
        // One thread, and little for it to compute: its instructions between two products are what keeps the tensor
        // core waiting when the tiles are small. Descriptors differ from their stage's only in the address field.
        if (lane == 0) {
            const uint32_t idesc = umma::idesc_bf16(128, p.bn) | (1u << 15) | (1u << 16);
            const uint64_t a_first = desc_mn(umma::smem_u32(operands)), b_first = desc_mn(umma::smem_u32(inputs) + GROUPS * RAW);
            const uint32_t a_step = p.operand_bytes() >> 4, b_step = p.input_bytes() >> 4, q_step = (groups * GROUP) >> 4;
            uint32_t done = 0;
            bool ok = true;
            for (; walk.more(); walk.next(p), in.next(), op.next()) {
                if (walk.in_run == 0 && done && !(ok = wait(&sh.acc_empty, (done - 1) & 1))) break;
                if (MODE == TMA && !(ok = wait(&sh.in_full[in.slot], in.phase))) break;
                if (!(ok = wait(&sh.op_full[op.slot], op.phase))) break;
                umma::fence_after_sync();
                const uint64_t A = a_first + op.slot * a_step;
                const uint64_t B = MODE == TMA ? b_first + in.slot * b_step : A + (GROUPS * GROUP >> 4);
#pragma unroll
                for (int m = 0; m < MT; ++m)
#pragma unroll
                    for (int q = 0; q < P; ++q) {
                        const uint32_t to = tmem + (m * P + q) * p.bn;
                        const uint64_t Am = A + (m * 2 * GROUP >> 4), Bq = B + q * q_step;
                        umma::mma16(to, Am, Bq, idesc, walk.in_run);
#pragma unroll
                        for (int k = 1; k < BK / 16; ++k) umma::mma16(to, Am + k * 128, Bq + k * 128, idesc, 1);
                    }
                umma::commit(&sh.op_empty[op.slot]);
                if (MODE == TMA) umma::commit(&sh.in_empty[in.slot]);
                if (walk.run_ends(p)) umma::commit(&sh.acc_full), ++done;
            }
            // every issued product has finished before TMEM is given back
            if (!ok) {
                umma::commit(&sh.acc_full);
                umma::mbar_wait(&sh.acc_full, done & 1, umma::DRAIN_NS);
            }
        }
        __syncwarp();
    } else if (warp == 1) {  // ------------------------------------ producer
        if (lane == 0) {
            bool ok = true;
            uint32_t it = 0;
            for (; walk.more(); walk.next(p), in.next(), ++it) {
                if (it >= (uint32_t)p.inputs && !(ok = wait(&sh.in_empty[in.slot], in.phase ^ 1))) break;
                const int k0 = walk.tile % p.ktiles * (MT * 128), n0 = walk.tile / p.ktiles * p.bn, t0 = walk.s * BK;
                umma::expect_tx(&sh.in_full[in.slot], p.input_bytes());
                const uint32_t to = umma::smem_u32(inputs + in.slot * p.input_bytes());
                for (int g = 0; g < GROUPS; ++g) tma_load(to + g * RAW, &map_q, k0 + 64 * g, t0, &sh.in_full[in.slot]);
                if (MODE == TMA)
                    for (int g = 0; g < groups; ++g)
                        tma_load(to + GROUPS * RAW + g * GROUP, &map_dy, n0 + 64 * g, t0, &sh.in_full[in.slot]);
            }
            if (!ok)  // the copies in flight land before the CTA leaves
                for (uint32_t i = it > (uint32_t)p.inputs ? it - p.inputs : 0; i < it; ++i)
                    umma::mbar_wait(&sh.in_full[i % p.inputs], (i / p.inputs) & 1, umma::DRAIN_NS);
        }
        __syncwarp();
    } else if (warp < 4) {  // --------------------------------- column sums
        const int c = 4 * (threadIdx.x - 64);  // this thread's four columns
        bool ok = true;
        float sum[4] = {};
        for (; walk.more(); walk.next(p), in.next(), op.next()) {
            const bool mine = a.db && walk.tile % p.ktiles == 0 && c < p.bn;
            if (walk.begins && walk.in_run == 0)
                for (float& v : sum) v = 0.0f;
            ok = ok && (MODE == TMA ? wait_all(&sh.in_full[in.slot], in.phase) : wait_all(&sh.op_full[op.slot], op.phase));
            if (mine && ok) {
                const uint8_t* B = MODE == TMA ? inputs + in.slot * p.input_bytes() + GROUPS * RAW
                                               : operands + op.slot * p.operand_bytes() + GROUPS * GROUP;
                float x[4] = {};
                for (int q = 0; q < P; ++q) {
                    const uint8_t* G = B + (q * groups + (c >> 6)) * GROUP + (c & 4) * 2;
#pragma unroll 16
                    for (int t = 0; t < BK; ++t) {
                        const uint2 w = *reinterpret_cast<const uint2*>(G + t * 128 + ((((c & 63) >> 3) ^ (t & 7)) << 4));
                        x[0] += umma::Op16<false>::lo(w.x), x[1] += umma::Op16<false>::hi(w.x);
                        x[2] += umma::Op16<false>::lo(w.y), x[3] += umma::Op16<false>::hi(w.y);
                    }
                }
#pragma unroll
                for (int h = 0; h < 4; ++h) sum[h] += x[h];
            }
            __syncwarp();
            if (ok && lane == 0) arrive(MODE == TMA ? &sh.in_empty[in.slot] : &sh.op_empty[op.slot]);
            if (mine && walk.share_ends(p)) {
                const int64_t n0 = (int64_t)(walk.tile / p.ktiles) * p.bn;
#pragma unroll
                for (int h = 0; h < 4; ++h) {
                    if (c + h >= p.bn) continue;
                    const float v = ok ? sum[h] : __uint_as_float(0x7fffffffu);
                    if (!walk.whole) part_db[(2 * blockIdx.x + (walk.head ? 0 : 1)) * (int64_t)p.bn + c + h] = v;
                    else if (n0 + c + h < a.n) a.db[n0 + c + h] = v;
                }
            }
        }
    } else {  // -------------------------------------------------- converters
        const int team = (threadIdx.x - 128) / TEAM, tid = (threadIdx.x - 128) % TEAM, w = warp - 4;
        // x8: a thread has one row of a stage and there 16 channels of every group of 64; 8 threads (two rows) then read
        // 128 bytes in a row and store to 8 different chunks of a line. dy (where it does not come by TMA): chunks of 8
        // columns, all of a thread's at the same columns. What comes through registers is fetched one stage ahead.
        constexpr int B_PER = MODE == TMA ? 1 : BK * widest(MODE) / 8 / TEAM;
        const int64_t blocks = (a.k + 31) / 32;
        const int ar = tid >> 2, ac = (tid & 3) * 2;
        const uint32_t raw_at = ar * 64 + ac * 8, lo_at = ar * 128 + ((ac ^ (ar & 7)) << 4), hi_at = ar * 128 + (((ac + 1) ^ (ar & 7)) << 4);
        const int b_bits = groups > 1 ? 4 : 3, bt = tid >> b_bits, bg = tid & ((1 << b_bits) - 1), b_step = TEAM >> b_bits;
        const bool vec_dy = ((uintptr_t)a.dy & 15) == 0 && (a.ld_dy * sizeof(T)) % 16 == 0;
        uint32_t code[GROUPS];
        Eight<T> held[MODE == TMA ? 1 : B_PER];
        // the stage to fetch: this team's next
        int fetch_u = walk.u, fetch_s = walk.s, fetch_tile = walk.tile;
        const uint8_t* units = nullptr;  // this thread's units in the tile to fetch from
        int here = 0;                    // how many of its groups have channels there
        int64_t fn = 0;                  // its first column of dy
        auto aim = [&] {
            const int64_t b = (int64_t)(fetch_tile % p.ktiles) * (MT * 4) + (ac >> 2);
            units = a.scale + ar * blocks + b;
            here = (int)min((int64_t)GROUPS, (blocks - b + 1) / 2);
            fn = (int64_t)(fetch_tile / p.ktiles) * p.bn + bg * 8;
        };
        auto advance = [&](int by) {
            fetch_u += by, fetch_s += by;
            if (fetch_s >= p.steps) {
                while (fetch_s >= p.steps) fetch_s -= p.steps, ++fetch_tile;
                aim();
            }
        };
        aim();
        advance(team);
        auto fetch = [&] {
            if (fetch_u >= walk.end) return;
            const int64_t t0 = (int64_t)fetch_s * BK;
            const int rows = (int)min((int64_t)BK, a.rows - t0);
#pragma unroll
            for (int g = 0; g < GROUPS; ++g) code[g] = g < here && ar < rows ? units[t0 * blocks + g * 2] : 127u;
            if constexpr (MODE != TMA) {
                const T* dy = static_cast<const T*>(a.dy) + (t0 + bt) * a.ld_dy;
#pragma unroll
                for (int i = 0; i < B_PER; ++i) {
                    if (bt + i * b_step < rows) held[i].load(dy + i * b_step * a.ld_dy, fn, a.n, vec_dy);
                    else held[i] = Eight<T>{};
                }
            }
            advance(2);
        };
        fetch();
        bool ok = true;
        uint32_t done = 0, it = 0;
        for (; walk.more(); walk.next(p), ++it, in.next(), op.next()) {
            if (ok && op.slot == team) {
                ok = wait_all(&sh.in_full[in.slot], in.phase);
                const uint8_t* X = inputs + in.slot * p.input_bytes() + raw_at;
                uint4 q[GROUPS];
#pragma unroll
                for (int g = 0; g < GROUPS; ++g) q[g] = *reinterpret_cast<const uint4*>(X + g * RAW);
                if (it >= (uint32_t)p.operands) ok = ok && wait_all(&sh.op_empty[op.slot], op.phase ^ 1);
                uint8_t* A = operands + op.slot * p.operand_bytes();
#pragma unroll
                for (int g = 0; g < GROUPS; ++g) {
                    const uint32_t uu = code[g] * 0x00800080u;  // a NaN block (code 255, bytes 0) is 0 times infinity
                    const __nv_bfloat162 unit2 = *reinterpret_cast<const __nv_bfloat162*>(&uu);
                    *reinterpret_cast<uint4*>(A + g * GROUP + lo_at) = eight_bytes(q[g].x, q[g].y, unit2);
                    *reinterpret_cast<uint4*>(A + g * GROUP + hi_at) = eight_bytes(q[g].z, q[g].w, unit2);
                }
                if constexpr (MODE != TMA) {
                    uint8_t* B = A + GROUPS * GROUP + (bg >> 3) * GROUP;
#pragma unroll
                    for (int i = 0; i < B_PER; ++i) {
                        const int t = bt + i * b_step;
                        if (t >= BK) break;
                        float left[8];
                        held[i].get(left);
#pragma unroll
                        for (int q = 0; q < P; ++q) {
                            float h[8];
#pragma unroll
                            for (int k = 0; k < 8; ++k) h[k] = part_of(left[k]);
                            *reinterpret_cast<uint4*>(B + q * groups * GROUP + t * 128 + (((bg & 7) ^ (t & 7)) << 4)) = umma::pack_chunk(h);
                        }
                    }
                }
                umma::fence_async_smem();
                __syncwarp();
                if (ok && lane == 0) arrive(&sh.op_full[op.slot]), arrive(&sh.in_empty[in.slot]);
                fetch();
            }
            if (!walk.run_ends(p)) continue;
            // the tile out of TMEM: every fourth warp has the lanes of one quarter
            ok = ok && wait_all(&sh.acc_full, done & 1);
            umma::fence_after_sync();
            const int64_t k0 = (int64_t)(walk.tile % p.ktiles) * (MT * 128), n0 = (int64_t)(walk.tile / p.ktiles) * p.bn;
            constexpr int W = P == 1 ? 32 : 16;  // columns at a time
            const int row = (w & 3) * 32 + lane, runs = p.bn / W;
            for (int i = w >> 2; i < MT * runs; i += CONVERTERS / 128) {
                const int m = i / runs, c = i % runs * W;
                float x[W];
                const uint32_t from = tmem + ((uint32_t)(w & 3) * 32 << 16) + m * P * p.bn + c;
                tmem_load(from + (P - 1) * p.bn, x);  // the smallest part first
#pragma unroll
                for (int q = P - 2; q >= 0; --q) {
                    float y[W];
                    tmem_load(from + q * p.bn, y);
#pragma unroll
                    for (int e = 0; e < W; ++e) x[e] += y[e];
                }
                if (!ok)
                    for (float& e : x) e = __uint_as_float(0x7fffffffu);
                const int64_t k = k0 + m * 128 + channel(row), n = n0 + c;
                if (!walk.whole) {
                    float* to = part + ((2 * blockIdx.x + (walk.head ? 0 : 1)) * (int64_t)MT * 128 + m * 128 + channel(row)) * p.bn + c;
                    if (!walk.begins) add_run<W>(x, to, W, true);
                    store_run<W>(to, x, W, true);
                } else if (k < a.k && n < a.n) {
                    const int count = (int)min((int64_t)W, a.n - n);
                    const int64_t to = k * a.n + n;
                    const bool vec = ((uintptr_t)a.dw & 15) == 0 && a.n % 8 == 0;
                    if (a.out_type == WC_F32) {
                        if (!walk.begins) add_run<W>(x, static_cast<float*>(a.dw) + to, count, vec);
                        store_run<W>(static_cast<float*>(a.dw) + to, x, count, vec);
                    } else if (a.out_type == WC_F16) {
                        store_run<W>(static_cast<__half*>(a.dw) + to, x, count, vec);
                    } else {
                        store_run<W>(static_cast<__nv_bfloat16*>(a.dw) + to, x, count, vec);
                    }
                }
            }
            umma::fence_before_sync();
            __syncwarp();
            if (lane == 0) arrive(&sh.acc_empty);
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

// Joins the split tiles (one a blockIdx.y). A thread has 4 columns of a row
// (row mt * 128 is db); with many CTAs to a tile they are dealt to blockDim.y
// threads and those joined in order.
constexpr int JOINERS = 256;
template <class T>
__global__ void __launch_bounds__(JOINERS) k_wgrad8_join(wc_act8_wgrad_args a, Plan p, const __grid_constant__ Splits splits,
                                                         const float* part, const float* part_db) {
    __shared__ float4 s[JOINERS];
    const Split& cut = splits.at[blockIdx.y];
    const int tile = cut.tile, c0 = cut.c0, c1 = cut.c1;
    const int rows = p.mt * 128, runs = p.bn / 4;
    const int i = blockIdx.x * blockDim.x + threadIdx.x, r = i / runs, c = i % runs * 4;
    const int64_t k0 = tile % p.ktiles * rows, n0 = tile / p.ktiles * p.bn, n = n0 + c;
    const bool bias = r == rows;
    const bool in = r <= rows && n < a.n && (bias ? a.db && tile % p.ktiles == 0 : k0 + r < a.k);
    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (in)
#pragma unroll 4
        for (int j = c0 + (int)threadIdx.y; j <= c1; j += blockDim.y) {
            const int64_t slot = j == c0 ? cut.slot : 2 * j;
            const float4 w = *reinterpret_cast<const float4*>(bias ? part_db + slot * p.bn + c : part + (slot * rows + r) * p.bn + c);
            v.x += w.x, v.y += w.y, v.z += w.z, v.w += w.w;
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
        else static_cast<T*>(a.dw)[(k0 + r) * a.n + n + j] = from_f<T>(e[j]);
    }
}

int mode_of(const wc_act8_wgrad_args& a) {
    if (a.type == WC_F32) return F32;
    if (a.type == WC_F16) return F16;
    return ((uintptr_t)a.dy & 15) == 0 && (a.ld_dy * 2) % 16 == 0 ? TMA : BF16;
}

Plan plan_of(const wc_act8_wgrad_args& a, int mode) {
    Plan p{};
    const int64_t k = a.k;
    p.steps = (int)((a.rows + BK - 1) / BK);
    p.mt = k > 128 ? 2 : 1;
    int64_t nt = (a.n + widest(mode) - 1) / widest(mode);
    p.bn = (int)(((a.n + nt - 1) / nt + 31) / 32 * 32);
    p.ktiles = (int)((k + p.mt * 128 - 1) / (p.mt * 128));
    p.ntiles = (int)((a.n + p.bn - 1) / p.bn);
    p.units = (int64_t)p.ktiles * p.ntiles * p.steps;
    p.ctas = (int)std::max<int64_t>(1, std::min<int64_t>(MAX_CTAS, p.steps == 1 ? p.units : (p.units + 1) / 2));
    p.joined = p.steps > 1 && (p.units % p.ctas != 0 || (p.units / p.ctas) % p.steps != 0);
    p.limit = a.out_type == WC_F32 ? RUN : 1 << 30;
    p.mode = mode;
    // a stage of operands for each team of converters; the rest of the memory holds inputs in flight
    p.operands = CONVERTERS / TEAM;
    p.inputs = std::min(MAX_STAGES, (RING - p.operands * p.operand_bytes()) / p.input_bytes());
    return p;
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

// A row-major matrix as boxes of 64 columns x 64 rows, zeros outside
CUtensorMap map_of(const void* base, CUtensorMapDataType type, int64_t width, int64_t rows, int64_t row_bytes, CUtensorMapSwizzle swizzle) {
    CUtensorMap m;
    const cuuint64_t dims[2] = {(cuuint64_t)width, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)row_bytes};
    const cuuint32_t box[2] = {64, BK}, step[2] = {1, 1};
    if (encoder()(&m, type, 2, const_cast<void*>(base), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
        throw std::runtime_error("cuTensorMapEncodeTiled refused a tensor map");
    return m;
}

template <int MODE, int MT, class T>
void launch_tile(const wc_act8_wgrad_args& a, const Plan& p, float* part, float* part_db, cudaStream_t s) {
    const int64_t pitch = (a.k + 31) / 32 * 32;
    const CUtensorMap q = map_of(a.q, CU_TENSOR_MAP_DATA_TYPE_UINT8, pitch, a.rows, pitch, CU_TENSOR_MAP_SWIZZLE_NONE);
    CUtensorMap dy{};
    if (MODE == TMA)
        dy = map_of(a.dy, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, a.n, a.rows, a.ld_dy * 2, CU_TENSOR_MAP_SWIZZLE_128B);
    const size_t smem = (size_t)p.operands * p.operand_bytes() + (size_t)p.inputs * p.input_bytes() + 1024;
    if (!wcdev::raise_smem_limit(reinterpret_cast<const void*>(k_wgrad8<MODE, MT, T>), RING + 1024)) return;
    k_wgrad8<MODE, MT, T><<<p.ctas, THREADS, smem, s>>>(a, p, q, dy, part, part_db);
}
template <int MODE, class T>
void launch_mode(const wc_act8_wgrad_args& a, const Plan& p, float* part, float* part_db, cudaStream_t s) {
    if (p.mt == 2) launch_tile<MODE, 2, T>(a, p, part, part_db, s);
    else launch_tile<MODE, 1, T>(a, p, part, part_db, s);
}

template <class T>
void launch_join(const wc_act8_wgrad_args& a, const Plan& p, const float* part, const float* part_db, cudaStream_t s) {
    const Splits splits(p);
    int sharers = 0;
    for (int i = 0; i < splits.n; ++i) sharers = std::max(sharers, splits.at[i].c1 - splits.at[i].c0 + 1);
    const int ny = sharers >= 8 ? 32 : 1;
    const dim3 block(JOINERS / ny, ny), grid(((p.mt * 128 + 1) * (p.bn / 4) + block.x - 1) / block.x, splits.n);
    k_wgrad8_join<T><<<grid, block, 0, s>>>(a, p, splits, part, part_db);
}

}  // namespace

uint64_t wgrad8_workspace(const wc_act8_wgrad_args& a) {
    if (!a.n || !a.rows) return 0;
    uint64_t most = 0;
    const Plan p = plan_of(a, mode_of(a));
    if (p.joined) most = (uint64_t)2 * p.ctas * (p.mt * 128 + 1) * p.bn * sizeof(float);
    return most;
}

void launch_wgrad8(const wc_act8_wgrad_args& a, cudaStream_t s) {
    if (!a.rows) {  // empty sums
        cudaMemsetAsync(a.dw, 0, (size_t)a.k * a.n * (a.out_type == WC_F32 ? 4 : 2), s);
        if (a.db) cudaMemsetAsync(a.db, 0, (size_t)a.n * 4, s);
        return;
    }
    const int mode = mode_of(a);
    const Plan p = plan_of(a, mode);
    float* part = static_cast<float*>(a.workspace);
    float* part_db = part + (int64_t)2 * p.ctas * p.mt * 128 * p.bn;
    if (mode == TMA) launch_mode<TMA, __nv_bfloat16>(a, p, part, part_db, s);
    else if (mode == BF16) launch_mode<BF16, __nv_bfloat16>(a, p, part, part_db, s);
    else if (mode == F16) launch_mode<F16, __half>(a, p, part, part_db, s);
    else launch_mode<F32, float>(a, p, part, part_db, s);
    if (!p.joined) return;
    if (a.out_type == WC_F32) launch_join<float>(a, p, part, part_db, s);
    else if (a.out_type == WC_F16) launch_join<__half>(a, p, part, part_db, s);
    else launch_join<__nv_bfloat16>(a, p, part, part_db, s);
}

}  // namespace wctrain
