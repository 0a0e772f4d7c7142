// Products with decoded weights: linear and grouped_linear.
//
//     out[i][j] = act(sum_k x[i][k] w[j][k] + bias[j]) * gate[i][j] + residual[i][j]
//
// linear is grouped_linear with one expert that owns every row.  Weights are
// dense matrices of x's type or INT4 payloads laid out by
// hct_b200_int4_weight_pack (the layout is described below).
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <type_traits>

#include "common.cuh"
#include "per_device.cuh"
#include "timeouts.cuh"

namespace hct {
namespace {

constexpr uint32_t MAX_EXPERTS = 1024;
constexpr uint64_t DIM_LIMIT = 1ull << 31;

// ---- packed INT4 weights ------------------------------------------------------
//
// A packed matrix is a sequence of blocks [ceil(rows / 128)][ceil(cols / 64)],
// each 128 rows x 64 columns (two scale blocks per row), 4608 contiguous
// bytes, so that one bulk copy brings everything a K step of a tile needs:
//   nibbles  [2 scale blocks][128 rows][16 bytes]
//   scales   [2 scale blocks][8][16] f16, that of row r at [r % 8][r / 8]
// A row's 16 bytes are what a dequantising thread takes, and the 4-byte words
// of 8 consecutive rows are what a warp's mma fragment takes (the lane of row
// r % 8 needs the scales of rows r % 8 + 8 i: 32 bytes in a row).
// Each 32-bit word holds the 8 values k = 8 c .. 8 c + 7 of its scale block,
// value 2 j in bits 4 j .. 4 j + 3 and value 2 j + 1 in bits 16 + 4 j .., so
// that (word >> 4 j) & 0x000f000f is the pair (2 j, 2 j + 1) in two 16-bit
// halves.  Rows and scale blocks past the matrix hold zero scales.
constexpr uint32_t PK_ROWS = 128, PK_COLS = 64;
constexpr uint32_t PK_NIB = PK_ROWS * PK_COLS / 2;       // 4096
constexpr uint32_t PK_BYTES = PK_NIB + PK_ROWS * 2 * 2;  // 4608

__host__ __device__ inline uint64_t pk_kblocks(uint64_t cols) { return (cols + PK_COLS - 1) / PK_COLS; }
__host__ __device__ inline uint32_t pk_scale_at(uint32_t row) { return row % 8 * 16 + row / 8; }
inline uint64_t pk_bytes(uint64_t rows, uint64_t cols) {
    return (rows + PK_ROWS - 1) / PK_ROWS * pk_kblocks(cols) * PK_BYTES;
}

// One thread per (row, scale block) of the padded matrix: 16 nibble bytes and
// a scale in, a permuted 16-byte word and the scale out.
__global__ void int4_weight_pack_kernel(const uint8_t *__restrict__ data, uint64_t rows,
                                        uint64_t cols, uint8_t *__restrict__ out, uint64_t tasks) {
    const uint64_t kb = pk_kblocks(cols);
    const uint64_t groups = cols / 32;
    const uint8_t *nib = data + rows * groups * 2;
    for (uint64_t t = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x; t < tasks;
         t += (uint64_t)gridDim.x * blockDim.x) {
        // block (row tile, k block), then scale block g, then row: the order of the output
        const uint64_t blk = t / (2 * PK_ROWS);
        const uint32_t in = (uint32_t)(t % (2 * PK_ROWS)), g = in / PK_ROWS, r = in % PK_ROWS;
        const uint64_t row = blk / kb * PK_ROWS + r, group = blk % kb * 2 + g;
        uint32_t w[4] = {0, 0, 0, 0};
        uint16_t scale = 0;
        if (row < rows && group < groups) {
            const uint64_t b = row * groups + group;
            scale = (uint16_t)(data[2 * b] | (data[2 * b + 1] << 8));
#pragma unroll
            for (int c = 0; c < 4; c++) {
                uint32_t v = 0;
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const uint32_t byte = nib[16 * b + 4 * c + j];
                    v |= (byte & 15u) << (4 * j) | (byte >> 4) << (16 + 4 * j);
                }
                w[c] = v;
            }
        }
        uint8_t *o = out + blk * PK_BYTES;
        *reinterpret_cast<uint4 *>(o + in * 16) = make_uint4(w[0], w[1], w[2], w[3]);
        *reinterpret_cast<uint16_t *>(o + PK_NIB + (g * PK_ROWS + pk_scale_at(r)) * 2) = scale;
    }
}

// Division by a number known on the host, of values below 2^31: a product and a
// shift in place of the 35 dependent instructions of a division.
struct Divisor {
    uint32_t d, mul, shift;
    Divisor() = default;
    explicit Divisor(uint32_t n) : d(n), shift(0) {
        while (shift < 31 && (1ull << shift) < n) shift++;
        mul = (uint32_t)(((1ull << 32) * ((1ull << shift) - n)) / n + 1);
    }
    __device__ __forceinline__ uint32_t of(uint32_t v) const { return (__umulhi(v, mul) + v) >> shift; }
};

// ---- what every kernel is given -------------------------------------------------

struct LinParams {
    const void *x, *w, *bias, *gate, *res, *offsets;
    void *out;
    uint64_t w_stride;
    uint32_t ldx, ldw, ldgate, ldres, ldo;  // at most 2^30
    uint32_t M, N, K, E;
    int off64;  // offsets are int64 (else int32)
    int bias_f32, act, odt;
    int vec_gate, vec_res, vec_out;  // rows start on 16-byte boundaries
};

// The groups, in shared memory: off[e] .. off[e + 1] are the rows of expert e,
// first[e] is the number of row tiles of the experts before it (first[E] their
// total) and per[e] the rows of each of its tiles: dealt out evenly, in whole
// multiples of 16 up to `tile.d`.  Offsets are clamped to [0, M] and to the
// largest before them, so that groups never overlap; without offsets the one
// expert owns every row.  Called by one whole warp.
struct Groups {
    uint32_t *first, *off, *per;
    __device__ __forceinline__ Groups(uint32_t *at, uint32_t E) : first(at), off(at + E + 1), per(off + E + 1) {}
};
constexpr uint32_t groups_bytes(uint32_t E) { return (3 * E + 2) * 4; }

__device__ __forceinline__ void scan_groups(const LinParams &p, const Divisor &tile, const Groups &g) {
    const uint32_t lane = threadIdx.x & 31u;
    uint32_t most = 0;  // largest offset so far
    for (uint32_t i0 = 0; i0 <= p.E; i0 += 32) {
        const uint32_t i = i0 + lane;
        int64_t v = 0;
        if (i <= p.E) {
            if (!p.offsets) v = i ? p.M : 0;
            else if (p.off64) v = reinterpret_cast<const int64_t *>(p.offsets)[i];
            else v = reinterpret_cast<const int32_t *>(p.offsets)[i];
        }
        uint32_t o = v < 0 ? 0u : v > (int64_t)p.M ? p.M : (uint32_t)v;
        o = max(o, most);
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const uint32_t w = __shfl_up_sync(0xffffffffu, o, d);
            if (lane >= (uint32_t)d) o = max(o, w);
        }
        if (i <= p.E) g.off[i] = o;
        most = __shfl_sync(0xffffffffu, o, 31);
    }
    __syncwarp();
    uint32_t base = 0;
    for (uint32_t e0 = 0; e0 < p.E; e0 += 32) {
        const uint32_t e = e0 + lane;
        const uint32_t m = e < p.E ? g.off[e + 1] - g.off[e] : 0;
        const uint32_t c = tile.of(m + tile.d - 1);
        uint32_t sum = c;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const uint32_t w = __shfl_up_sync(0xffffffffu, sum, d);
            if (lane >= (uint32_t)d) sum += w;
        }
        if (e < p.E) {
            g.first[e] = base + sum - c;
            g.per[e] = c > 1 ? ((m + c - 1) / c + 15) / 16 * 16 : m;
        }
        base += __shfl_sync(0xffffffffu, sum, 31);
    }
    if (lane == 0) g.first[p.E] = base;
    __syncwarp();
}

// The expert that owns tile t: the last e with first[e] <= t.
__device__ __forceinline__ uint32_t expert_of(const uint32_t *first, uint32_t E, uint32_t t) {
    uint32_t lo = 0, hi = E - 1;
    while (lo < hi) {
        const uint32_t mid = (lo + hi + 1) / 2;
        if (first[mid] <= t) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// These kernels are launched while the one before them on the stream may still
// run (programmatic serialisation): a kernel sets itself up and waits for
// everything before it, in every thread, before it touches global memory; and
// it says when the kernel after it may start doing the same.  One thread of a CTA
// says so for the CTA, so it is the one that has allocated TMEM: a next kernel of
// another library that fits beside it on an SM could else take the TMEM first and
// wait for this kernel, which waits for the TMEM.  The stream kernel does not say
// so: early CTAs of the next kernel take the room that its clusters need (1 x 4096 x
// 4096 in a row: 7.1 us against 6.8).
__device__ __forceinline__ void after_previous_kernel() {
    asm volatile("griddepcontrol.wait;" ::: "memory");
}
__device__ __forceinline__ void let_next_kernel_start() {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

__device__ __forceinline__ float h2f(uint16_t v) { return __half2float(__ushort_as_half(v)); }
__device__ __forceinline__ float bf2f(uint16_t v) { return __uint_as_float((uint32_t)v << 16); }
template <bool BF>
__device__ __forceinline__ float from16(uint16_t v) {
    return BF ? bf2f(v) : h2f(v);
}

template <class T>
__device__ __forceinline__ uint32_t bits_of(T v) {
    return *reinterpret_cast<uint32_t *>(&v);
}

// z / (1 + 2^(-t log2 e)): the hardware's ex2 and reciprocal, a few 2^-23 of the
// value, as the rest of the f32 epilogue.
__device__ __forceinline__ float times_sigmoid(float z, float minus_t_log2e) {
    float e, r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(minus_t_log2e));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));
    return z * r;
}
__device__ __forceinline__ float activate(float z, int act) {
    constexpr float LOG2E = 1.44269504088896341f;
    switch (act) {
        case HCT_B200_ACT_RELU: return z < 0.0f ? 0.0f : z;
        case HCT_B200_ACT_SILU: return times_sigmoid(z, -LOG2E * z);
        case HCT_B200_ACT_GELU: return 0.5f * z * (1.0f + erff(z * 0.70710678118654752f));
        case HCT_B200_ACT_GELU_TANH:  // (1 + tanh(t)) / 2 = 1 / (1 + e^-2t)
            return times_sigmoid(
                z, z * fmaf(-0.0713548162726f * LOG2E, z * z, -1.59576912160573071f * LOG2E));
        default: return z;
    }
}

template <bool BF>
__device__ __forceinline__ float bias_of(const LinParams &p, uint32_t e, uint32_t n) {
    if (!p.bias) return 0.0f;
    const uint64_t i = (uint64_t)e * p.N + n;
    return p.bias_f32 ? reinterpret_cast<const float *>(p.bias)[i]
                      : from16<BF>(reinterpret_cast<const uint16_t *>(p.bias)[i]);
}

__device__ uint32_t g_linear_timeouts;  // bounded waits that have expired, never cleared

// ---- tensor-core kernel ---------------------------------------------------------
//
// A tile is 128 output features x up to BN rows of x, computed transposed:
// the weights are the M side of the tcgen05 contraction (A, 128 rows, K-major)
// and the rows of x its N side (B), so that one token costs an instruction of
// width 16 instead of an almost empty 128-row tile, and INT4 weights are
// dequantised straight into the A operand.  The instruction's N is the tile's
// own row count rounded up to 16.
//
//   warp 0      TMA producer: x tiles (and dense weight tiles) into a ring of
//               K steps of 64, packed INT4 blocks into a ring of their own
//   warp 1      TMEM allocation; one thread issues the MMAs.  Up to 128 rows the
//               issuing (450 to 600 clocks a K step: a wait, four MMAs, a commit)
//               takes longer than the MMAs (256), so warps 1 and 2 issue every
//               other K step each (the even and the odd slots of the ring), into
//               accumulators of their own
//   warps 4-11  epilogue, two sets of four warps that take every other 16 rows:
//               accumulators (TMEM lanes = features) through shared memory into
//               runs of 8 features, so that outputs, gate and residual move in
//               16-byte pieces of a row
//   warps 12-23 INT4: three groups of 128 threads dequantise every third K step,
//               a thread per weight row, into the 128B-swizzled A tile.  Dense
//               rows that TMA cannot fetch (unaligned starts, odd strides): they
//               copy both operands by loads of 4 or of 2 bytes
//
// PAIR: where whole tiles of rows keep every SM busy, two CTAs share one tile of
// 256 features (cta_group::2): each holds the weights of its 128 features and
// half of the rows, so that a K step moves 32 KB instead of 48 KB from L2 to
// each SM for the same MMAs.  The first CTA's MMA warp issues for both.
//
// With at least one tile per SM the kernel is persistent (grid = SMs) and the
// accumulators are double-buffered, so a tile's epilogue runs under the next
// tile's MMAs.  With fewer, the K range of a tile is split over a cluster of
// CTAs: each pushes the rows that another finishes into that one's shared memory
// by bulk copies (196 x 1792 x 1664: 9.4 us; reading them there with
// ld.shared::cluster, 6 to 8 bytes a clock, took 17.6), and a row's parts are added
// in rank order: no workspace, no atomics, the same bits every time.
//
// F32 outputs (PRECISE) accumulate at most SECTION K steps in TMEM and add the
// sections in registers with rounding; INT4 weights are then two A operands,
// the rounded weight and what the rounding left, each with accumulators of its
// own.  Where a value of x is infinite, the rounded weights alone give the sum
// that the weights would (a weight is 0 where its rounding is), and the sum of
// what was left, with infinity times 0 or infinities of both signs, is dropped.
//
// A wait on a slot's parity is sound only for one that cannot be two passes
// behind.  The producers and issuers meet every pass of a slot in order.  The
// three dequantising or loading groups take the steps of a slot by turns: the
// packed ring has a multiple of 3 slots, so that a slot is always one group's;
// a slot of the operand ring is one group's too where there are two issuers (6
// slots), and with one issuer, whose MMAs complete in order, the step before
// in the group has already seen every step up to its own less (slots + 3).
//
// Every wait is bounded; an expired one is counted in g_linear_timeouts, the CTA's
// roles leave their loops, its copies and MMAs are drained (bounded) and TMEM
// is freed.
constexpr int BK = 64;  // 128 bytes of a row: one swizzle row
constexpr int A_BYTES = 128 * BK * 2;
constexpr int MAX_STAGES = 8, MAX_RAW = 16;
constexpr int SECTION = 4;  // 256 products to an accumulator: at most 16 truncated sums
constexpr uint32_t SMEM_LIMIT = 232448;  // 227 KB
constexpr uint32_t SMEM_MIN = 120 * 1024;  // one CTA per SM: TMEM is never waited for
constexpr uint32_t RASTER = 8;
constexpr uint32_t EPI_BYTES = 2 * 16 * 128 * 4;  // staging of the two epilogue sets

struct UmmaParams {
    LinParams p;
    uint32_t bn;      // rows per tile at most
    uint32_t xbox;    // rows per TMA box of x (a multiple of 8)
    uint32_t stages, raw_stages;
    uint32_t tmem_cols, tmem_stride;
    uint32_t split;   // CTAs per cluster, each a part of K
    uint32_t issuers; // warps that issue MMAs, each with its own accumulators
    Divisor tile, nt, band;  // by bn, by feature tiles, by RASTER x feature tiles
};

struct Ctl {
    uint64_t xfull[MAX_STAGES], afull[MAX_STAGES], empty[MAX_STAGES];
    uint64_t rfull[MAX_RAW], rempty[MAX_RAW];
    uint64_t tfull[2], tempty[2], drain, parts;
    uint32_t tmem_base;
    uint32_t note[12];  // of the other CTA's dequantising warps (note_at)
    int abort, issued, raw_issued;
};

__device__ __forceinline__ uint32_t smem_u32(const void *p) {
    return (uint32_t)__cvta_generic_to_shared(p);
}
__device__ __forceinline__ uint64_t globaltimer() {
    uint64_t t;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
    return t;
}
__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_expect_tx(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes)
                 : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
// Arrival on the barrier at the same place in CTA `rank` of the cluster, released
// to the cluster: its waiters see what was done before it.  It takes about 1000
// clocks.
__device__ __forceinline__ void mbar_arrive_at(uint32_t bar, uint32_t rank) {
    asm volatile(
        "{\n\t.reg .b32 a;\n\t"
        "mapa.shared::cluster.u32 a, %0, %1;\n\t"
        "mbarrier.arrive.release.cluster.shared::cluster.b64 _, [a];\n\t}" ::"r"(bar),
        "r"(rank)
        : "memory");
}
// The same in a K loop, to a barrier that expects 4 bytes of it: an asynchronous
// store of a word that nobody reads, whose completion on the barrier is a release at
// cluster scope too and which the thread does not wait for.  (2048 x 14336 x 4096
// INT4 with SiLU and gate: 194 us; arrivals as above, sent on by one warp 312, by two
// 231; arrivals released to their own CTA only, which order nothing for the waiter,
// 191.)
__device__ __forceinline__ void note_at(uint32_t word, uint32_t bar) {
    asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.b32 [%0], %1, [%2];" ::"r"(
                     word),
                 "r"(0), "r"(bar)
                 : "memory");
}
__device__ __forceinline__ uint32_t map_to(uint32_t addr, uint32_t rank) {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(addr), "r"(rank));
    return a;
}
// Acquires at cluster scope: arrivals may come from the other CTA of a pair.
__device__ __forceinline__ bool mbar_try_wait(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    return ok != 0;
}
// Bounded wait (2 s): false when the phase did not complete in time or the CTA
// has given up meanwhile.  The clock is read only once the wait is a long one.
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, const int *abort) {
    uint64_t t0 = 0;
    for (uint32_t i = 1; i < (1u << 30); ++i) {
        if (mbar_try_wait(bar, parity)) return true;
        if ((i & 255u) == 0) {
            if (*(const volatile int *)abort) return false;
            const uint64_t t = globaltimer();
            if (t0 == 0) t0 = t;
            else if (t - t0 > 2000000000ull) return false;
        }
    }
    return false;
}
// The same by a whole warp: true when every lane's phase completed.
__device__ __forceinline__ bool mbar_wait_warp(uint32_t bar, uint32_t parity, const int *abort) {
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort));
}
// Whether every one of the 128 threads of an epilogue set says ok, so that all of
// them go on to its barriers or none does.
__device__ __forceinline__ bool set_agrees(uint32_t set, bool ok) {
    uint32_t all;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.u32 p, %1, 0;\n\t"
        "barrier.cta.red.and.pred q, %2, 128, p;\n\t"
        "selp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(all)
        : "r"((uint32_t)ok), "r"(set + 1)
        : "memory");
    return all != 0;
}
__device__ __forceinline__ bool elect_one() {
    uint32_t e;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "elect.sync _|p, 0xffffffff;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(e));
    return e != 0;
}

// A position in a ring of slots: the slot and the parity of its current pass.
struct Ring {
    uint32_t slot, pass, size;
    __device__ __forceinline__ explicit Ring(uint32_t n, uint32_t at = 0) : slot(at), pass(0), size(n) {}
    __device__ __forceinline__ void step(uint32_t by = 1) {  // by <= size
        slot += by;
        if (slot >= size) {
            slot -= size;
            pass ^= 1u;
        }
    }
};
// PAIR: the barrier may be the other CTA's.
template <bool PAIR>
__device__ __forceinline__ void tma_2d(uint32_t dst, const CUtensorMap *map, uint32_t bar, int x,
                                       int y) {
    if (PAIR)
        asm volatile(
            "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
            " [%0], [%1, {%3, %4}], [%2];" ::"r"(dst),
            "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y)
            : "memory");
    else
        asm volatile(
            "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes"
            " [%0], [%1, {%3, %4}], [%2];" ::"r"(dst),
            "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y)
            : "memory");
}
template <bool PAIR>
__device__ __forceinline__ void tma_3d(uint32_t dst, const CUtensorMap *map, uint32_t bar, int x,
                                       int y, int z) {
    if (PAIR)
        asm volatile(
            "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
            " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
            "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y), "r"(z)
            : "memory");
    else
        asm volatile(
            "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes"
            " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
            "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y), "r"(z)
            : "memory");
}
__device__ __forceinline__ void bulk_load(uint32_t dst, const void *src, uint32_t bytes,
                                          uint32_t bar) {
    asm volatile(
        "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
            dst),
        "l"(src), "r"(bytes), "r"(bar)
        : "memory");
}
// K-major, 128B swizzle: rows of 128 bytes, 8-row groups 1024 bytes apart.
__device__ __forceinline__ uint64_t umma_desc(uint32_t saddr) {
    return (uint64_t)((saddr & 0x3FFFFu) >> 4) | (1ull << 16) | (64ull << 32) | (1ull << 46) |
           (2ull << 61);
}
// A value that is the same in every lane, in a form that lets the compiler keep
// it (and the addresses and descriptors made of it) in uniform registers.
__device__ __forceinline__ uint32_t uniform(uint32_t v) { return __shfl_sync(0xffffffffu, v, 0); }

template <bool PAIR>
__device__ __forceinline__ void umma(uint32_t tmem_d, uint64_t da, uint64_t db, uint32_t idesc,
                                     uint32_t accumulate) {
    if (PAIR)
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
            "l"(da), "l"(db), "r"(idesc), "r"(accumulate)
            : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
            "l"(da), "l"(db), "r"(idesc), "r"(accumulate)
            : "memory");
}
// Arrives, once the MMAs issued before have completed, on the barrier at this
// place: of both CTAs of a pair.
template <bool PAIR>
__device__ __forceinline__ void umma_commit(uint32_t bar) {
    if (PAIR)
        asm volatile(
            "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64"
            " [%0], %1;" ::"r"(bar),
            "h"((uint16_t)3)
            : "memory");
    else
        asm volatile(
            "tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar)
            : "memory");
}
template <bool PAIR>
__device__ __forceinline__ void tmem_alloc(uint32_t to, uint32_t cols) {
    if (PAIR) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(to),
                     "r"(cols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(to),
                     "r"(cols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
}
template <bool PAIR>
__device__ __forceinline__ void tmem_free(uint32_t base, uint32_t cols) {
    if (PAIR)
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(cols)
                     : "memory");
    else
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(cols)
                     : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
          "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]),
          "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_barrier() {
    asm volatile("barrier.cluster.arrive.release;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
}
// The last barrier of a cluster: no CTA ends while another may still read its
// memory.  Nothing is published, so the arrival need not wait for the outputs'
// stores.
__device__ __forceinline__ void cluster_leave() {
    asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory");
    asm volatile("barrier.cluster.wait;" ::: "memory");
}
// One bulk copy from this CTA's shared memory to another's, and to its barrier.
__device__ __forceinline__ void push(uint32_t to, uint32_t from, uint32_t bytes, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.shared::cluster.shared::cta.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
            to),
        "r"(from), "r"(bytes), "r"(bar)
        : "memory");
}

// One tile: expert, its rows [m0, m0 + rows) and first feature n0.
struct Tile {
    uint32_t e, m0, rows, n0;
};
template <uint32_t FEATURES>
__device__ __forceinline__ Tile tile_at(const UmmaParams &u, const Groups &g, uint32_t t) {
    Tile r;
    r.e = u.p.E > 1 ? expert_of(g.first, u.p.E, u.nt.of(t)) : 0;
    const uint32_t lo = g.off[r.e], hi = g.off[r.e + 1], per = g.per[r.e], first = g.first[r.e];
    // bands of RASTER row tiles; within one, the row tiles of a feature tile run
    // next to each other, so that the tiles in flight share x and w in L2
    const uint32_t q = t - first * u.nt.d, band = u.band.of(q), in = q - band * u.band.d;
    const uint32_t width = min(RASTER, g.first[r.e + 1] - first - band * RASTER);
    const uint32_t ft = width == RASTER ? in / RASTER : width == 1 ? in : in / width;
    r.n0 = ft * FEATURES;
    r.m0 = lo + (band * RASTER + in - ft * width) * per;
    r.rows = min(per, hi - r.m0);
    return r;
}

// Eight INT4 values times their scale as four pairs of x's type, and for
// PRECISE what the rounding of each left.  Without PRECISE the rounding stays in the
// result of a 16-bit output, as it does when a weight is decoded to x's type: in
// bf16 2.4e-3 of the norm against 1.7e-3 with the output rounded alone.  Two operands
// for every output would double the MMAs.
//
// (word >> 4 j) & 0x000f000f are the nibbles of the pair (2 j, 2 j + 1); or'ed
// into the mantissa of 1024 (fp16) or 128 (bf16) they are 1024 + n or 128 + n
// exactly, and n - 8 after an exact subtraction (fp16 has room for 1024 + 16 n
// too, which saves the shift of every other pair).  fp16: one multiplication by
// the scale, rounded once.  bf16: the f16 scale (11 bits) is hi + lo, two
// bf16 values; (n - 8) lo has at most 6 bits, so fma(n - 8, hi, (n - 8) lo)
// rounds the exact product once.
//
// fp16 and PRECISE: a weight is 8 h + l with h = (n - 8) / 8 s rounded, which is in
// range for every finite scale, and l = 8 ((n - 8) / 8 s - h), which has at most 5
// bits and no bit below 2^-24: exact.  To keep every step of l in range too, it is
// 8 fma((n - 8) / 8, s, -h) for scales of 2^-8 and more, and fma((n - 8) / 8, 8 s,
// -8 h) for smaller ones.  h takes a scale of 2^-21 in the place of smaller ones, so
// that it is 0 only where the weight is.
template <bool BF, bool PRECISE>
struct Scale;
template <>
struct Scale<false, false> {
    __half2 s;
    __device__ __forceinline__ explicit Scale(uint16_t b) : s(__half2half2(__ushort_as_half(b))) {}
};
template <>
struct Scale<false, true> {
    __half2 h, s, minus, times;  // l = times fma(n, s, minus h)
    bool finite;
    __device__ __forceinline__ explicit Scale(uint16_t b) {
        const uint16_t mag = b & 0x7fffu, sign = b & 0x8000u;
        finite = mag < 0x7c00u;
        h = __half2half2(__ushort_as_half(mag != 0 && mag < 8 ? (uint16_t)(sign | 8) : b));
        const bool large = mag >= 0x1c00u;  // 2^-8
        s = __half2half2(__ushort_as_half(b));
        if (!large) s = __hmul2(s, __float2half2_rn(8.0f));
        minus = __float2half2_rn(large ? -1.0f : -8.0f);
        times = __float2half2_rn(large ? 8.0f : 1.0f);
    }
};
template <bool PRECISE>
struct Scale<true, PRECISE> {
    __nv_bfloat162 hi, lo;
    bool finite;
    __device__ __forceinline__ explicit Scale(uint16_t b) {
        const float f = h2f(b);
        const __nv_bfloat16 h = __float2bfloat16_rn(f);
        finite = (b & 0x7c00u) != 0x7c00u;
        hi = __bfloat162bfloat162(h);
        lo = __bfloat162bfloat162(__float2bfloat16_rn(finite ? f - __bfloat162float(h) : 0.0f));
    }
};
// odd pairs stay where they are: 1024 + 16 n, whose sixteenth less 72 is n - 8
__device__ __forceinline__ __half2 fp16_pair(uint32_t w, int j) {
    uint32_t b = (j & 1 ? (w >> (8 * (j / 2))) & 0x00f000f0u : (w >> (8 * (j / 2))) & 0x000f000fu) |
                 0x64006400u;
    return *reinterpret_cast<__half2 *>(&b);
}
__device__ __forceinline__ void dequant8(uint32_t w, const Scale<false, false> &s, uint32_t (&v)[4],
                                         uint32_t (&)[4]) {
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const __half2 m = fp16_pair(w, j);
        const __half2 n = j & 1 ? __hfma2(m, __float2half2_rn(0.0625f), __float2half2_rn(-72.0f))
                                : __hsub2(m, __float2half2_rn(1032.0f));
        v[j] = bits_of(__hmul2(n, s.s));
    }
}
__device__ __forceinline__ void dequant8(uint32_t w, const Scale<false, true> &s, uint32_t (&v)[4],
                                         uint32_t (&l)[4]) {
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const __half2 m = fp16_pair(w, j);  // 1024 + n or 1024 + 16 n; here to (n - 8) / 8, exactly
        const __half2 n = j & 1 ? __hfma2(m, __float2half2_rn(0.0078125f), __float2half2_rn(-9.0f))
                                : __hfma2(m, __float2half2_rn(0.125f), __float2half2_rn(-129.0f));
        const __half2 h = __hmul2(n, s.h);
        v[j] = bits_of(h);
        l[j] = s.finite ? bits_of(__hmul2(__hfma2(n, s.s, __hmul2(h, s.minus)), s.times)) : 0u;
    }
}
template <bool PRECISE>
__device__ __forceinline__ void dequant8(uint32_t w, const Scale<true, PRECISE> &s, uint32_t (&v)[4],
                                         uint32_t (&l)[4]) {
#pragma unroll
    for (int j = 0; j < 4; j++) {
        uint32_t b = ((w >> (4 * j)) & 0x000f000fu) | 0x43004300u;
        const __nv_bfloat162 n =
            __hsub2(*reinterpret_cast<__nv_bfloat162 *>(&b), __float2bfloat162_rn(136.0f));
        const __nv_bfloat162 c = __hmul2(n, s.lo);
        const __nv_bfloat162 h = __hfma2(n, s.hi, c);
        v[j] = bits_of(h);
        if (PRECISE) l[j] = s.finite ? bits_of(__hadd2(__hfma2(n, s.hi, __hneg2(h)), c)) : 0u;
    }
}

template <int ACT, int W>
__device__ __forceinline__ void activate_all(float (&z)[W]) {
#pragma unroll
    for (int j = 0; j < W; j++) z[j] = activate(z[j], ACT);
}

// What an epilogue writes: F32, one of the 16-bit types, or any.
enum { OUT_F32 = 0, OUT_16 = 1, OUT_ANY = 2 };
template <int OUT>
__device__ __forceinline__ bool writes_f32(const LinParams &p) {
    return OUT == OUT_F32 || (OUT == OUT_ANY && p.odt == HCT_B200_F32);
}

template <bool BF>
__device__ __forceinline__ float2 unpack2(uint32_t v) {
    if (BF) return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
    return __half22float2(*reinterpret_cast<const __half2 *>(&v));
}

// 8 consecutive 16-bit values, `live` of which exist; one load where aligned.
__device__ __forceinline__ void load8(const uint16_t *q, bool vec, uint32_t live, uint32_t (&v)[4]) {
    if (vec && live >= 8) {
        const uint4 w = *reinterpret_cast<const uint4 *>(q);
        v[0] = w.x, v[1] = w.y, v[2] = w.z, v[3] = w.w;
    } else {
#pragma unroll
        for (int j = 0; j < 4; j++) {
            v[j] = 2 * j < (int)live ? q[2 * j] : 0u;
            if (2 * j + 1 < (int)live) v[j] |= (uint32_t)q[2 * j + 1] << 16;
        }
    }
}

// The operands of 8 consecutive features n .. n + 7 of row m: the gate in g, the
// residual in r (8 16-bit values in r[0..3], or 8 floats).
struct Operands {
    uint32_t g[4], r[8];
};
template <int OUT>
__device__ __forceinline__ void load_operands(const LinParams &p, uint32_t m, uint32_t n,
                                              Operands &o) {
    const uint32_t live = p.N - n;
    if (p.gate)
        load8(reinterpret_cast<const uint16_t *>(p.gate) + (uint64_t)m * p.ldgate + n, p.vec_gate, live,
              o.g);
    if (p.res) {
        const uint64_t at = (uint64_t)m * p.ldres + n;
        if (writes_f32<OUT>(p)) {
            const uint32_t *q = reinterpret_cast<const uint32_t *>(p.res) + at;
            if (p.vec_res && live >= 8) {
                const uint4 a = reinterpret_cast<const uint4 *>(q)[0];
                const uint4 b = reinterpret_cast<const uint4 *>(q)[1];
                o.r[0] = a.x, o.r[1] = a.y, o.r[2] = a.z, o.r[3] = a.w;
                o.r[4] = b.x, o.r[5] = b.y, o.r[6] = b.z, o.r[7] = b.w;
            } else {
#pragma unroll
                for (int j = 0; j < 8; j++) o.r[j] = j < (int)live ? q[j] : 0u;
            }
        } else {
            uint32_t v[4];
            load8(reinterpret_cast<const uint16_t *>(p.res) + at, p.vec_res, live, v);
#pragma unroll
            for (int j = 0; j < 4; j++) o.r[j] = v[j];
        }
    }
}

// 8 sums (bias included) of row m, features n .. n + 7, to outputs.
template <bool BF, int OUT>
__device__ __forceinline__ void finish8(const LinParams &p, float (&z)[8], const Operands &o,
                                        uint32_t m, uint32_t n) {
    switch (p.act) {
        case HCT_B200_ACT_RELU: activate_all<HCT_B200_ACT_RELU>(z); break;
        case HCT_B200_ACT_SILU: activate_all<HCT_B200_ACT_SILU>(z); break;
        case HCT_B200_ACT_GELU: activate_all<HCT_B200_ACT_GELU>(z); break;
        case HCT_B200_ACT_GELU_TANH: activate_all<HCT_B200_ACT_GELU_TANH>(z); break;
        default: break;
    }
    if (p.gate) {
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const float2 g = unpack2<BF>(o.g[j]);
            z[2 * j] *= g.x, z[2 * j + 1] *= g.y;
        }
    }
    const uint32_t live = p.N - n;
    const bool whole = p.vec_out && live >= 8;
    const uint64_t at = (uint64_t)m * p.ldo + n;
    if (writes_f32<OUT>(p)) {
        if (p.res) {
#pragma unroll
            for (int j = 0; j < 8; j++) z[j] += __uint_as_float(o.r[j]);
        }
        float *q = reinterpret_cast<float *>(p.out) + at;
        if (whole) {
            reinterpret_cast<float4 *>(q)[0] = make_float4(z[0], z[1], z[2], z[3]);
            reinterpret_cast<float4 *>(q)[1] = make_float4(z[4], z[5], z[6], z[7]);
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (j < (int)live) q[j] = z[j];
        }
    } else {
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            float a = z[2 * j], b = z[2 * j + 1];
            if (p.odt == HCT_B200_F16) {
                if (p.res) {
                    const float2 r = unpack2<false>(o.r[j]);
                    a += r.x, b += r.y;
                }
                w[j] = bits_of(__floats2half2_rn(a, b));
            } else {
                if (p.res) {
                    const float2 r = unpack2<true>(o.r[j]);
                    a += r.x, b += r.y;
                }
                w[j] = bits_of(__floats2bfloat162_rn(a, b));
            }
        }
        uint16_t *q = reinterpret_cast<uint16_t *>(p.out) + at;
        if (whole) {
            *reinterpret_cast<uint4 *>(q) = make_uint4(w[0], w[1], w[2], w[3]);
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (j < (int)live) q[j] = (uint16_t)(w[j / 2] >> (16 * (j & 1)));
        }
    }
}

// Sixteen rows m .. m + 15 (count of them live) of a tile's 128 features, a
// feature per thread of the set in z: through the set's shared memory (16 x
// 128 floats) to its threads by rows, each 2 rows x 8 features n .. n + 7.
template <bool BF, int OUT>
__device__ __forceinline__ void finish_rows(const LinParams &p, const float (&z)[16], float *stage,
                                            uint32_t set, uint32_t id, const float (&bias)[8],
                                            uint32_t m, uint32_t count, uint32_t n) {
    Operands o[2];
    const uint32_t j0 = id / 16;
    const bool live = n < p.N;
#pragma unroll
    for (int i = 0; i < 2; i++)
        if (live && j0 + 8 * i < count) load_operands<OUT>(p, m + j0 + 8 * i, n, o[i]);
    asm volatile("bar.sync %0, 128;" ::"r"(set + 1) : "memory");  // the last rows have been read
#pragma unroll
    for (int j = 0; j < 16; j++) stage[j * 128 + id] = z[j];
    asm volatile("bar.sync %0, 128;" ::"r"(set + 1) : "memory");
#pragma unroll
    for (int i = 0; i < 2; i++) {
        if (!live || j0 + 8 * i >= count) continue;
        const float4 *q = reinterpret_cast<const float4 *>(stage + (j0 + 8 * i) * 128 + id % 16 * 8);
        const float4 a = q[0], b = q[1];
        float v[8] = {a.x + bias[0], a.y + bias[1], a.z + bias[2], a.w + bias[3],
                      b.x + bias[4], b.y + bias[5], b.z + bias[6], b.w + bias[7]};
        finish8<BF, OUT>(p, v, o[i], m + j0 + 8 * i, n);
    }
}

template <bool BF>
__device__ __forceinline__ void load_bias8(const LinParams &p, uint32_t e, uint32_t n,
                                           float (&bias)[8]) {
#pragma unroll
    for (int j = 0; j < 8; j++) bias[j] = n + j < p.N ? bias_of<BF>(p, e, n + j) : 0.0f;
}

__device__ __forceinline__ void prefetch_l2(const void *q) {
    asm volatile("prefetch.global.L2 [%0];" ::"l"(q));
}

// Where the operands come from: dense matrices by TMA, packed INT4 weights (x by
// TMA), or dense matrices of any stride and alignment, copied by warps, whose loads
// are 4 bytes wide where every row starts on 4 bytes and K is even, else 2.
enum { FORM_DENSE = 0, FORM_INT4 = 1, FORM_ANY = 2, FORM_WORDS = 3 };
constexpr int umma_threads(int form) { return form == FORM_DENSE ? 384 : 768; }
// rows per tile at most: a thread of the epilogue keeps half of them as f32 sums where PRECISE
__host__ __device__ constexpr uint32_t max_rows(int form, bool precise) {
    return precise ? (form == FORM_DENSE ? 128 : 64) : 256;
}

template <int FORM, bool BF, bool PRECISE, bool PAIR>
__global__ void __launch_bounds__(umma_threads(FORM), 1)
    linear_umma_kernel(const __grid_constant__ CUtensorMap tmX,
                       const __grid_constant__ CUtensorMap tmW, const __grid_constant__ UmmaParams u) {
    constexpr bool INT4 = FORM == FORM_INT4, WORDS = FORM == FORM_WORDS, ANY = WORDS || FORM == FORM_ANY,
                   TMA_W = FORM == FORM_DENSE;
    constexpr uint32_t A_PARTS = INT4 && PRECISE ? 2 : 1;
    constexpr float A_UNIT = INT4 && PRECISE && !BF ? 8.0f : 1.0f;  // of the first operand (dequant8)
    constexpr uint32_t GROUPS = 3;  // of dequantising or loading warps
    constexpr uint32_t FEATURES = PAIR ? 256 : 128, CTAS = PAIR ? 2 : 1;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    const LinParams &p = u.p;
    const uint32_t stages = u.stages, stage_bytes = A_PARTS * A_BYTES + u.bn / CTAS * 128;
    uint8_t *raw = smem + (size_t)stages * stage_bytes;
    uint8_t *epi = raw + (size_t)u.raw_stages * PK_BYTES;
    Ctl *ctl = reinterpret_cast<Ctl *>(epi + EPI_BYTES);
    const Groups groups(reinterpret_cast<uint32_t *>(ctl + 1), p.E);
    const uint32_t warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31u;

    if (warp == 0) {
        if (lane < MAX_STAGES) {
            mbar_init(smem_u32(&ctl->xfull[lane]), 1);
            mbar_init(smem_u32(&ctl->afull[lane]), 4);  // a group's warps
            mbar_init(smem_u32(&ctl->empty[lane]), 1);
        }
        if (INT4 && lane < MAX_RAW) {
            mbar_init(smem_u32(&ctl->rfull[lane]), 1);
            mbar_init(smem_u32(&ctl->rempty[lane]), 4);
        }
        if (lane < 2) {
            mbar_init(smem_u32(&ctl->tfull[lane]), u.issuers);
            // the epilogue's warps, and for a pair's leader the other CTA's
            mbar_init(smem_u32(&ctl->tempty[lane]), PAIR && !(blockIdx.x & 1u) ? 9 : 8);
        }
        if (lane == 0) {
            mbar_init(smem_u32(&ctl->drain), u.issuers);
            mbar_init(smem_u32(&ctl->parts), 1);
            ctl->abort = 0;
            ctl->issued = 0;
            ctl->raw_issued = 0;
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 1) {
        tmem_alloc<PAIR>(smem_u32(&ctl->tmem_base), u.tmem_cols);
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        let_next_kernel_start();
    }
    after_previous_kernel();
    if (warp == 2) scan_groups(p, u.tile, groups);
    __syncthreads();
    if (PAIR) cluster_barrier();  // the other CTA's barriers are set up too
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = uniform(ctl->tmem_base);
    const auto aborted = [&] { return *(volatile int *)&ctl->abort != 0; };
    const auto give_up = [&] {
        atomicAdd(&g_linear_timeouts, 1u);
        atomicExch(&ctl->abort, 1);
    };

    const uint32_t tiles = uniform(groups.first[p.E]) * u.nt.d;
    // clusters are consecutive CTAs: the parts of a K range, or a pair
    const uint32_t rank = u.split > 1 ? blockIdx.x % u.split : 0, side = PAIR ? blockIdx.x & 1u : 0u;
    const uint32_t t0 = PAIR ? blockIdx.x / 2 : u.split > 1 ? blockIdx.x / u.split : blockIdx.x;
    const uint32_t step = PAIR ? gridDim.x / 2 : gridDim.x;  // a split has one tile per cluster
    const uint32_t kbs = max((p.K + BK - 1) / BK, 1u);
    uint32_t kb0 = 0, kb1 = kbs;
    if (u.split > 1) {  // below 2^25 x 8
        kb0 = kbs * rank / u.split;
        kb1 = kbs * (rank + 1) / u.split;
    }
    const uint32_t sect = PRECISE ? SECTION * u.issuers : kb1 - kb0;  // K steps per accumulation

    // The producers and the MMA warp run whole (their addresses and descriptors
    // are warp-uniform); one elected lane issues.
    if (!ANY && warp == 0) {
        Ring at(stages);
        uint32_t issued = 0;
        bool ok = true;
        for (uint32_t t = t0; ok && t < tiles; t += step) {
            const Tile c = tile_at<FEATURES>(u, groups, t);
            // each CTA of a pair holds its 128 features and half of the tile's rows,
            // and both copies complete on the leader's barrier
            const uint32_t held = (c.rows + 15) / 16 * 16 / CTAS;
            const uint32_t boxes = (held + u.xbox - 1) / u.xbox;
            const uint32_t bytes = (boxes * u.xbox * 128 + (TMA_W ? A_BYTES : 0)) * CTAS;
            const int m0 = (int)(c.m0 + side * held), n0 = (int)(c.n0 + side * 128);
            for (uint32_t kb = kb0; kb < kb1; kb++, at.step()) {
                ok = mbar_wait_warp(smem_u32(&ctl->empty[at.slot]), at.pass ^ 1u, &ctl->abort);
                if (!ok) break;
                if (elect_one()) {
                    const uint32_t sa = smem_u32(smem + (size_t)at.slot * stage_bytes);
                    const uint32_t sb = sa + A_PARTS * A_BYTES;
                    uint32_t fb = smem_u32(&ctl->xfull[at.slot]);
                    if (side == 0) mbar_expect_tx(fb, bytes);
                    if (PAIR) fb = map_to(fb, 0);
                    if (TMA_W) tma_3d<PAIR>(sa, &tmW, fb, (int)(kb * BK), n0, (int)c.e);
                    for (uint32_t b = 0; b < boxes; b++)
                        tma_2d<PAIR>(sb + b * u.xbox * 128, &tmX, fb, (int)(kb * BK),
                                     m0 + (int)(b * u.xbox));
                }
                __syncwarp();
                issued++;
            }
        }
        if (lane == 0) ctl->issued = (int)issued;
        if (!ok) give_up();
    } else if (PAIR && warp == 1 && side == 1) {
        // tells the leader, which issues for both CTAs, of each accumulator that has
        // been read here, but for the last two, which it does not wait for: nothing is on
        // its way when it ends.  (The epilogue's warps would wait for their outputs'
        // stores: 2048 x 14336 x 4096 dense 171 us for 167)
        Ring acc(2);
        for (uint32_t t = t0; t + 2 * step < tiles; t += step, acc.step()) {
            if (!mbar_wait_warp(smem_u32(&ctl->tempty[acc.slot]), acc.pass, &ctl->abort)) {
                give_up();
                break;
            }
            if (lane == 0) mbar_arrive_at(smem_u32(&ctl->tempty[acc.slot]), 0);
            __syncwarp();
        }
    } else if (warp == 1 || (warp == 2 && u.issuers == 2)) {
        // D = F32, A = B = x's type, both K-major, M = FEATURES; N follows the tile
        const uint32_t idesc0 =
            (1u << 4) | (BF ? (1u << 7) | (1u << 10) : 0u) | ((FEATURES / 16) << 24);
        // INT4: half of the lanes wait for the x tile, half for the weights; the upper
        // half of the warp for the second of two K steps
        const uint32_t full = smem_u32(ANY || (INT4 && (lane & 8u)) ? ctl->afull : ctl->xfull);
        // INT4: two steps to a wait where that leaves the ring three to be filled
        // meanwhile.  The issuing warp shares its scheduler with three dequantising
        // ones; 2048 x 14336 x 4096 with SiLU and gate takes 190 us for 213.  Dense
        // operands, which come in order from one producer, lost by it (170 us for 168)
        const bool pairs = INT4 && u.issuers == 1 && stages >= 5;
        const uint32_t me = warp - 1, every = u.issuers - 1;  // slots: me modulo u.issuers
        Ring at(stages), acc(2);
        bool ok = true;
        for (uint32_t t = t0; side == 0 && ok && t < tiles; t += step) {
            const Tile c = tile_at<FEATURES>(u, groups, t);
            const uint32_t idesc = uniform(idesc0 | ((c.rows + 15) / 16 * 2) << 17);
            for (uint32_t kb = kb0; ok && kb < kb1; acc.step()) {
                const uint32_t end = min(kb + sect, kb1);
                bool fresh = true;  // nothing accumulated yet
                ok = mbar_wait_warp(smem_u32(&ctl->tempty[acc.slot]), acc.pass ^ 1u, &ctl->abort);
                if (!ok) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const uint32_t d = tmem + (acc.slot * u.issuers * A_PARTS + me) * u.tmem_stride;
                while (kb < end) {
                    if ((at.slot & every) != me) {
                        kb++, at.step();
                        continue;
                    }
                    const Ring here = at;
                    const bool two = pairs && kb + 1 < end;
                    kb++, at.step();
                    const bool later = two && lane >= 16;
                    ok = mbar_wait_warp(full + (later ? at.slot : here.slot) * 8,
                                        later ? at.pass : here.pass, &ctl->abort);
                    if (!ok) break;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const auto issue = [&](uint32_t slot, bool more) {
                        const uint32_t sa = smem_u32(smem) + slot * stage_bytes;
                        const uint64_t da = umma_desc(sa), db = umma_desc(sa + A_PARTS * A_BYTES);
#pragma unroll
                        for (uint32_t a = 0; a < A_PARTS; a++)
#pragma unroll
                            for (uint32_t k = 0; k < BK / 16; k++)
                                umma<PAIR>(d + a * u.tmem_stride, da + a * (A_BYTES >> 4) + 2 * k, db + 2 * k,
                                           idesc, more || k);
                        umma_commit<PAIR>(smem_u32(&ctl->empty[slot]));
                    };
                    if (elect_one()) {
                        issue(here.slot, !fresh);
                        if (two) issue(at.slot, true);
                    }
                    __syncwarp();
                    fresh = false;
                    if (two) kb++, at.step();
                }
                if (ok && elect_one()) umma_commit<PAIR>(smem_u32(&ctl->tfull[acc.slot]));
                __syncwarp();
            }
        }
        if (!ok) give_up();
        // completes once every MMA above has, in both CTAs
        if (side == 0 && elect_one()) umma_commit<PAIR>(smem_u32(&ctl->drain));
        __syncwarp();
    } else if (INT4 && warp == 3) {
        const uint32_t nt = (p.N + 127) / 128;
        Ring at(u.raw_stages);
        uint32_t issued = 0;
        bool ok = true;
        for (uint32_t t = t0; ok && t < tiles; t += step) {
            const Tile c = tile_at<FEATURES>(u, groups, t);
            // a pair's second half may lie past the last features: any block will do there
            const uint64_t block = (uint64_t)c.e * nt + min(c.n0 / 128 + side, nt - 1);
            const uint8_t *src = reinterpret_cast<const uint8_t *>(p.w) + (block * kbs + kb0) * PK_BYTES;
            for (uint32_t kb = kb0; kb < kb1; kb++, at.step(), src += PK_BYTES) {
                ok = mbar_wait_warp(smem_u32(&ctl->rempty[at.slot]), at.pass ^ 1u, &ctl->abort);
                if (!ok) break;
                if (elect_one()) {
                    const uint32_t fb = smem_u32(&ctl->rfull[at.slot]);
                    mbar_expect_tx(fb, PK_BYTES);
                    bulk_load(smem_u32(raw + (size_t)at.slot * PK_BYTES), src, PK_BYTES, fb);
                }
                __syncwarp();
                issued++;
            }
        }
        if (lane == 0) ctl->raw_issued = (int)issued;
        if (!ok) give_up();
    } else if (INT4 && warp >= 12) {
        // this group's K steps of all the CTA's tiles, one after another
        const uint32_t group = (warp - 12) >> 2, row = threadIdx.x & 127u;
        const uint64_t steps = t0 < tiles ? (uint64_t)((tiles - t0 - 1) / step + 1) * (kb1 - kb0) : 0;
        Ring in(u.raw_stages, group), to(stages, group);
        const uint32_t mine = row * 128 + ((row & 7u) << 4);  // chunk c of my row: ^ (c << 4)
        for (uint64_t it = group; it < steps; it += GROUPS, in.step(GROUPS), to.step(GROUPS)) {
            if (!mbar_wait_warp(smem_u32(&ctl->rfull[in.slot]), in.pass, &ctl->abort)) {
                give_up();
                break;
            }
            const uint8_t *src = raw + (size_t)in.slot * PK_BYTES;
            uint4 q[2];
            uint16_t sc[2];
#pragma unroll
            for (int g = 0; g < 2; g++) {
                q[g] = *reinterpret_cast<const uint4 *>(src + (g * 128 + row) * 16);
                sc[g] = *reinterpret_cast<const uint16_t *>(src + PK_NIB + (g * 128 + pk_scale_at(row)) * 2);
            }
            if (!mbar_wait_warp(smem_u32(&ctl->empty[to.slot]), to.pass ^ 1u, &ctl->abort)) {
                give_up();
                break;
            }
            uint8_t *a = smem + (size_t)to.slot * stage_bytes;
#pragma unroll
            for (int g = 0; g < 2; g++) {
                const Scale<BF, PRECISE> scale(sc[g]);
                const uint32_t w[4] = {q[g].x, q[g].y, q[g].z, q[g].w};
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    uint32_t v[4], l[4];
                    dequant8(w[c], scale, v, l);
                    uint8_t *o = a + (mine ^ ((g * 4 + c) << 4));
                    *reinterpret_cast<uint4 *>(o) = make_uint4(v[0], v[1], v[2], v[3]);
                    if (PRECISE)
                        *reinterpret_cast<uint4 *>(o + A_BYTES) = make_uint4(l[0], l[1], l[2], l[3]);
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) {
                // a pair's leader issues for both CTAs: each of its warps expects the note
                // of the other CTA's
                const uint32_t bar = smem_u32(&ctl->afull[to.slot]);
                if (!PAIR) mbar_arrive(bar);
                else if (side == 0) mbar_expect_tx(bar, 4);
                else note_at(map_to(smem_u32(&ctl->note[warp - 12]), 0), map_to(bar, 0));
                mbar_arrive(smem_u32(&ctl->rempty[in.slot]));
            }
        }
    } else if (ANY && warp >= 12) {
        // this group's K steps: a warp copies 32 rows of w and a quarter of the rows of
        // x, a row at a time, two values per lane
        const uint32_t group = (warp - 12) >> 2, part = (warp - 12) & 3u, col = lane * 2;
        Ring to(stages, group);
        uint32_t turn = group;  // K steps until the group's next
        bool ok = true;
        for (uint32_t t = t0; ok && t < tiles; t += step) {
            const Tile c = tile_at<FEATURES>(u, groups, t);
            const uint16_t *w = reinterpret_cast<const uint16_t *>(p.w) + c.e * p.w_stride;
            const uint16_t *x = reinterpret_cast<const uint16_t *>(p.x);
            const uint32_t xrows = (c.rows + 15) / 16 * 16, quarter = xrows / 4;
            for (uint32_t kb = kb0; kb < kb1; kb++) {
                if (turn) {
                    turn--;
                    continue;
                }
                turn = GROUPS - 1;
                ok = mbar_wait_warp(smem_u32(&ctl->empty[to.slot]), to.pass ^ 1u, &ctl->abort);
                if (!ok) break;
                uint8_t *a = smem + (size_t)to.slot * stage_bytes;
                const uint32_t k = kb * BK + col;
                const auto copy = [&](const uint16_t *src, uint64_t ld, uint32_t row0, uint32_t live,
                                      uint32_t r0, uint32_t count, uint8_t *dst) {
                    const uint16_t *q = src + (uint64_t)(row0 + r0) * ld + k;
                    constexpr uint32_t N = WORDS ? 16 : 8;  // 16 loads in flight
                    for (uint32_t i = 0; i < count; i += N, q += N * ld) {
                        uint32_t v[N];
                        uint16_t hi[N];
#pragma unroll
                        for (uint32_t j = 0; j < N; j++) {
                            const bool there = i + j < count && r0 + i + j < live;
                            if (WORDS) {
                                v[j] = there && k < p.K ? *reinterpret_cast<const uint32_t *>(q + j * ld) : 0;
                            } else {
                                v[j] = there && k < p.K ? q[j * ld] : 0;
                                hi[j] = there && k + 1 < p.K ? q[j * ld + 1] : 0;
                            }
                        }
#pragma unroll
                        for (uint32_t j = 0; j < N; j++) {
                            const uint32_t r = r0 + i + j;
                            if (i + j < count)
                                *reinterpret_cast<uint32_t *>(dst + r * 128 +
                                                              (((lane >> 2) ^ (r & 7u)) << 4) +
                                                              (lane & 3u) * 4) =
                                    WORDS ? v[j] : v[j] | (uint32_t)hi[j] << 16;
                        }
                    }
                };
                // the group's next K step on its way to L2 meanwhile
                if (kb + GROUPS < kb1) {
                    const uint32_t next = (kb + GROUPS) * BK, row = c.n0 + part * 32 + lane;
                    if (row < p.N) prefetch_l2(w + (uint64_t)row * p.ldw + next);
                    for (uint32_t r = part * quarter + lane; r < min((part + 1) * quarter, c.rows); r += 32)
                        prefetch_l2(x + (uint64_t)(c.m0 + r) * p.ldx + next);
                }
                copy(w, p.ldw, c.n0, p.N - c.n0, part * 32, 32, a);
                copy(x, p.ldx, c.m0, c.rows, part * quarter, quarter, a + A_BYTES);
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&ctl->afull[to.slot]));
                to.step(GROUPS);
            }
        }
        if (!ok) give_up();
    } else if (warp >= 4 && warp < 12) {
        constexpr int CHUNKS = max_rows(FORM, PRECISE) / 32;  // of 16 rows, per set
        const uint32_t set = (warp - 4) >> 2, q = warp & 3u, id = q * 32 + lane;
        float *part = reinterpret_cast<float *>(smem);  // split: [rows of x][128 features]
        float *stage = reinterpret_cast<float *>(epi + set * (EPI_BYTES / 2));
        Ring acc(2);
        uint32_t steps = 0;  // K steps of the sections before
        bool ok = true;
        for (uint32_t t = t0; ok && t < tiles; t += step) {
            const Tile c = tile_at<FEATURES>(u, groups, t);
            const uint32_t n = c.n0 + side * 128 + id % 16 * 8;
            float bias[8];
            if (u.split == 1) load_bias8<BF>(p, c.e, n, bias);
            float sum[PRECISE ? CHUNKS : 1][16];
            if (PRECISE) {
#pragma unroll
                for (int i = 0; i < (PRECISE ? CHUNKS : 1); i++)
#pragma unroll
                    for (int j = 0; j < 16; j++) sum[i][j] = 0.0f;
            }
            for (uint32_t kb = kb0; kb < kb1; kb += sect, acc.step()) {
                ok = mbar_wait_warp(smem_u32(&ctl->tfull[acc.slot]), acc.pass, &ctl->abort);
                if (!PRECISE) ok = set_agrees(set, ok);
                if (!ok) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                // a section of one K step is in the accumulators of that step's issuer
                const bool two = u.issuers == 2 && kb + 1 < kb1;
                const uint32_t lone = two ? 0 : steps & (u.issuers - 1);
                const uint32_t ta = tmem + (acc.slot * u.issuers * A_PARTS + lone) * u.tmem_stride +
                                    ((q * 32) << 16);
                steps += min(sect, kb1 - kb);
                if (PRECISE) {
#pragma unroll
                    for (int i = 0; i < (PRECISE ? CHUNKS : 1); i++) {
                        const uint32_t j0 = (2 * i + set) * 16;
                        if (j0 >= c.rows) continue;
                        uint32_t v[16];
                        __syncwarp();
                        tmem_ld16(ta + j0, v);
#pragma unroll
                        for (int j = 0; j < 16; j++) sum[i][j] += A_UNIT * __uint_as_float(v[j]);
                        if (two || A_PARTS == 2) {
                            tmem_ld16(ta + u.tmem_stride + j0, v);
#pragma unroll
                            for (int j = 0; j < 16; j++) {
                                const float f = __uint_as_float(v[j]);
                                sum[i][j] += A_PARTS == 1 || fabsf(f) < INFINITY ? f : 0.0f;
                            }
                        }
                    }
                } else {
                    for (uint32_t j0 = set * 16; j0 < c.rows; j0 += 32) {
                        uint32_t v[16];
                        float z[16];
                        __syncwarp();
                        tmem_ld16(ta + j0, v);
#pragma unroll
                        for (int j = 0; j < 16; j++) z[j] = __uint_as_float(v[j]);
                        if (two) {
                            tmem_ld16(ta + u.tmem_stride + j0, v);
#pragma unroll
                            for (int j = 0; j < 16; j++) z[j] += __uint_as_float(v[j]);
                        }
                        if (u.split > 1) {
#pragma unroll
                            for (int j = 0; j < 16; j++) part[(j0 + j) * 128 + id] = z[j];
                        } else {
                            finish_rows<BF, OUT_16>(p, z, stage, set, id, bias, c.m0 + j0,
                                                   c.rows - j0, n);
                        }
                    }
                }
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&ctl->tempty[acc.slot]));
            }
            if (PRECISE) ok = set_agrees(set, ok);
            if (PRECISE && ok) {
#pragma unroll
                for (int i = 0; i < (PRECISE ? CHUNKS : 1); i++) {
                    const uint32_t j0 = (2 * i + set) * 16;
                    if (j0 >= c.rows) continue;
                    if (u.split > 1) {
#pragma unroll
                        for (int j = 0; j < 16; j++) part[(j0 + j) * 128 + id] = sum[i][j];
                    } else {
                        finish_rows<BF, OUT_F32>(p, sum[i], stage, set, id, bias, c.m0 + j0, c.rows - j0, n);
                    }
                }
            }
        }
        if (!ok) give_up();
    }

    if (!PAIR && u.split > 1) {
        // one tile per cluster: each CTA finishes its share of the tile's rows, adding the
        // CTAs' parts in rank order.  A CTA pushes every other one its rows by one bulk
        // copy.  The barriers and the wait are reached on every path
        constexpr int OUT = PRECISE ? OUT_F32 : OUT_16;
        Tile c{};
        uint32_t j = 0, j0 = 0, j1 = 0, n = 0;
        float bias[8];
        Operands o;
        const uint32_t slot = (u.bn + u.split - 1) / u.split * 512;  // bytes that a CTA receives of one other
        uint8_t *recv = smem + u.bn * 512;
        if (t0 < tiles) {
            c = tile_at<FEATURES>(u, groups, t0);
            n = c.n0 + threadIdx.x % 16 * 8;
            j0 = c.rows * rank / u.split;
            j1 = c.rows * (rank + 1) / u.split;
            j = j0 + threadIdx.x / 16;
            if (j < j1 && n < p.N) {
                load_bias8<BF>(p, c.e, n, bias);
                load_operands<OUT>(p, c.m0 + j, n, o);
            }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // the parts, for the copies
        __syncwarp();
        cluster_barrier();  // every CTA's ring is free to receive
        if (warp == 0 && lane < u.split && t0 < tiles) {
            // lane r: the rows of CTA r
            const uint32_t r0 = c.rows * lane / u.split, rows = c.rows * (lane + 1) / u.split - r0;
            if (lane == rank) {
                if (rows) mbar_expect_tx(smem_u32(&ctl->parts), rows * 512 * (u.split - 1));
            } else if (rows) {
                push(map_to(smem_u32(recv + (rank - (rank > lane)) * slot), lane), smem_u32(smem + r0 * 512), rows * 512,
                     map_to(smem_u32(&ctl->parts), lane));
            }
        }
        if (j1 > j0) {
            const int go_on = 0;
            if (!mbar_wait(smem_u32(&ctl->parts), 0, &go_on)) give_up();
        }
        if (!aborted() && n < p.N) {
            const uint32_t f = threadIdx.x % 16 * 8;
            while (j < j1) {
                float z[8] = {};
                for (uint32_t r = 0; r < u.split; r++) {
                    const uint8_t *from =
                        r == rank ? smem + j * 512 : recv + (r - (r > rank)) * slot + (j - j0) * 512;
                    const float4 a = reinterpret_cast<const float4 *>(from + f * 4)[0];
                    const float4 b = reinterpret_cast<const float4 *>(from + f * 4)[1];
                    z[0] += a.x, z[1] += a.y, z[2] += a.z, z[3] += a.w;
                    z[4] += b.x, z[5] += b.y, z[6] += b.z, z[7] += b.w;
                }
#pragma unroll
                for (int i = 0; i < 8; i++) z[i] += bias[i];
                finish8<BF, OUT>(p, z, o, c.m0 + j, n);
                j += blockDim.x / 16;
                if (j < j1) load_operands<OUT>(p, c.m0 + j, n, o);
            }
        }
        cluster_leave();
    }

    // ---- teardown: nothing of this CTA may be in flight when it ends --------------
    __syncthreads();
    if (threadIdx.x == 0 && aborted()) {
        // the latest load into each slot (its phase completes only with the copy; a
        // pair's x and dense copies complete on the leader's barriers)
        const int issued = ctl->issued, got = ctl->raw_issued, go_on = 0;
        for (int it = max(0, issued - (int)stages); side == 0 && it < issued; it++)
            mbar_wait(smem_u32(&ctl->xfull[it % stages]), (uint32_t)(it / stages) & 1u, &go_on);
        for (int it = max(0, got - (int)u.raw_stages); it < got; it++)
            mbar_wait(smem_u32(&ctl->rfull[it % u.raw_stages]), (uint32_t)(it / u.raw_stages) & 1u,
                      &go_on);
    }
    if (threadIdx.x == 32) {
        const int go_on = 0;
        if (!mbar_wait(smem_u32(&ctl->drain), 0, &go_on)) give_up();
    }
    __syncthreads();
    if (PAIR) cluster_leave();  // neither CTA's memory is in use any more
    if (warp == 1) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        tmem_free<PAIR>(tmem, u.tmem_cols);
    }
}

// ---- INT4 stream kernel: a few rows of x -----------------------------------------
//
// Up to 8 NT rows against 128 features: nothing but the stream of packed
// weights costs, and one kernel step per 4.5 bits has to keep up with HBM.
// Each warp takes every WARPS-th K block of 64 of the CTA's range, brought
// into its own two-slot ring by bulk copies (no other warp waits for it), and
// feeds mma.sync m16n8k16 straight from registers: the nibbles less 8 are
// exact in x's type, so a scale block's products are exact integers times x,
// summed in f32, and the block's scale multiplies that sum in f32.  No weight
// is rounded, for any output type.  A lane's A fragment is 8 consecutive k of
// a row and its B fragment the same 8 of a row of x: the order of k inside a
// scale block does not matter to the sum.
//
// The warps' sums meet in shared memory; where tiles are few, the K range is
// also split over a cluster, whose CTAs push their sums to the CTA that
// finishes the row (added in rank order).
constexpr int ST_WARPS = 8, ST_THREADS = ST_WARPS * 32, ST_SLOTS = 2;

struct StreamParams {
    LinParams p;
    uint32_t split, shift;  // CTAs per cluster: 1 << shift
    int vec_x;              // rows of x start on 16-byte boundaries
    Divisor tile, nt;       // by 8 NT rows, by feature tiles
};

// d = a b of m16n8k16, and d += a b.
template <bool BF>
__device__ __forceinline__ void mma_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                          uint32_t a3, uint32_t b0, uint32_t b1) {
    if (BF)
        asm volatile(
            "{\n\t.reg .f32 z;\n\tmov.f32 z, 0f00000000;\n\t"
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
            "{%8,%9}, {z,z,z,z};\n\t}"
            : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm volatile(
            "{\n\t.reg .f32 z;\n\tmov.f32 z, 0f00000000;\n\t"
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
            "{%8,%9}, {z,z,z,z};\n\t}"
            : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <bool BF>
__device__ __forceinline__ void mma_more(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                         uint32_t a3, uint32_t b0, uint32_t b1) {
    if (BF)
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
            "{%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
            "{%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The pairs of a word as nibble - 8 in x's type (see dequant8), in bf16 times 2^-8
// (ST_UNIT): 32 products of x's largest value are then within f32, as its products
// with the weights are.
template <bool BF>
constexpr float ST_UNIT = BF ? 256.0f : 1.0f;
template <bool BF>
__device__ __forceinline__ void nibbles8(uint32_t w, uint32_t (&v)[4]) {
#pragma unroll
    for (int j = 0; j < 4; j++) {
        if (BF) {
            uint32_t b = ((w >> (4 * j)) & 0x000f000fu) | 0x43004300u;
            v[j] = bits_of(__hfma2(*reinterpret_cast<__nv_bfloat162 *>(&b), __float2bfloat162_rn(0.00390625f),
                                   __float2bfloat162_rn(-0.53125f)));
        } else {
            uint32_t b = (j & 1 ? (w >> (8 * (j / 2))) & 0x00f000f0u
                                : (w >> (8 * (j / 2))) & 0x000f000fu) | 0x64006400u;
            const __half2 m = *reinterpret_cast<__half2 *>(&b);
            v[j] = bits_of(j & 1 ? __hfma2(m, __float2half2_rn(0.0625f), __float2half2_rn(-72.0f))
                                 : __hsub2(m, __float2half2_rn(1032.0f)));
        }
    }
}

// 8 values k .. k + 7 of row m of x, zero past the row's end and past `hi`.
__device__ __forceinline__ uint4 load_x8(const StreamParams &q, uint32_t m, uint32_t hi, uint32_t k) {
    uint4 v = make_uint4(0, 0, 0, 0);
    if (m >= hi || k >= q.p.K) return v;  // K is a multiple of 32: 8 values or none
    const uint16_t *s = reinterpret_cast<const uint16_t *>(q.p.x) + (uint64_t)m * q.p.ldx + k;
    if (q.vec_x) return *reinterpret_cast<const uint4 *>(s);
    v.x = s[0] | (uint32_t)s[1] << 16;
    v.y = s[2] | (uint32_t)s[3] << 16;
    v.z = s[4] | (uint32_t)s[5] << 16;
    v.w = s[6] | (uint32_t)s[7] << 16;
    return v;
}

template <bool BF, int NT>
__global__ void __launch_bounds__(ST_THREADS, 2)
    linear_int4_stream_kernel(const __grid_constant__ StreamParams q) {
    constexpr uint32_t ROWS = 8 * NT;
    extern __shared__ __align__(128) uint8_t st_smem[];
    const LinParams &p = q.p;
    uint8_t *ring = st_smem;                                                   // [warp][slot]
    float *recv = reinterpret_cast<float *>(ring + ST_WARPS * ST_SLOTS * PK_BYTES);  // [ROWS][128]
    uint64_t *full = reinterpret_cast<uint64_t *>(recv + ROWS * 128);           // [warp][slot]
    int *abort = reinterpret_cast<int *>(full + ST_WARPS * ST_SLOTS);
    const Groups groups(reinterpret_cast<uint32_t *>(abort + 2), p.E);
    const uint32_t warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31u;
    // a warp's barriers are its own: without groups it can start to load at once
    if (lane == 0) {
        for (int i = 0; i < ST_SLOTS; i++) mbar_init(smem_u32(&full[warp * ST_SLOTS + i]), 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        *abort = 0;
    }
    __syncwarp();
    after_previous_kernel();
    if (p.offsets) {
        if (warp == 1) scan_groups(p, q.tile, groups);
        __syncthreads();
    }
    // the cluster's CTAs are all running before any of them writes to another
    if (q.split > 1) asm volatile("barrier.cluster.arrive.release;" ::: "memory");

    const uint32_t nt = q.nt.d, kbs = (uint32_t)pk_kblocks(p.K);
    const uint32_t rank = blockIdx.x & (q.split - 1), t = blockIdx.x >> q.shift;
    // of the whole cluster alike
    const bool work = !p.offsets || t < groups.first[p.E] * nt;
    uint32_t e = 0, m0 = 0, hi = 0, n0 = 0;
    float acc[8][NT][4];
#pragma unroll
    for (int i = 0; i < 8; i++)
#pragma unroll
        for (int c = 0; c < NT; c++)
#pragma unroll
            for (int j = 0; j < 4; j++) acc[i][c][j] = 0.0f;
    bool ok = true;
    if (work) {
        const uint32_t rt = q.nt.of(t);
        if (p.offsets) {
            e = p.E > 1 ? expert_of(groups.first, p.E, rt) : 0;
            hi = groups.off[e + 1];
            m0 = groups.off[e] + (rt - groups.first[e]) * ROWS;
        } else {
            hi = p.M;
            m0 = rt * ROWS;
        }
        n0 = (t - rt * nt) * 128;
        const uint32_t kb0 = kbs * rank >> q.shift, kb1 = kbs * (rank + 1) >> q.shift;
        const uint8_t *src = reinterpret_cast<const uint8_t *>(p.w) +
                             ((uint64_t)e * nt + n0 / 128) * kbs * PK_BYTES;
        uint8_t *mine = ring + warp * ST_SLOTS * PK_BYTES;
        const auto fetch = [&](uint32_t kb, uint32_t slot) {
            if (kb < kb1 && elect_one()) {
                const uint32_t bar = smem_u32(&full[warp * ST_SLOTS + slot]);
                mbar_expect_tx(bar, PK_BYTES);
                bulk_load(smem_u32(mine + slot * PK_BYTES), src + (uint64_t)kb * PK_BYTES, PK_BYTES, bar);
            }
            __syncwarp();
        };
        const uint32_t gid = lane / 4, tig = lane % 4;
        uint4 x[2][NT];  // of the next K block
        const auto fetch_x = [&](uint32_t kb) {
#pragma unroll
            for (int g = 0; g < 2; g++)
#pragma unroll
                for (int c = 0; c < NT; c++)
                    x[g][c] = load_x8(q, m0 + 8 * c + gid, kb < kb1 ? hi : 0, kb * 64 + g * 32 + tig * 8);
        };
        uint32_t kb = kb0 + warp;
#pragma unroll
        for (uint32_t s = 0; s < ST_SLOTS; s++) fetch(kb + s * ST_WARPS, s);
        fetch_x(kb);
        uint32_t slot = 0, pass = 0;
        for (; kb < kb1; kb += ST_WARPS) {
            if (!mbar_wait_warp(smem_u32(&full[warp * ST_SLOTS + slot]), pass, abort)) {
                ok = false;
                break;
            }
            const uint8_t *blk = mine + slot * PK_BYTES;
            uint4 xs[2][NT];
#pragma unroll
            for (int g = 0; g < 2; g++)
#pragma unroll
                for (int c = 0; c < NT; c++) xs[g][c] = x[g][c];
            fetch_x(kb + ST_WARPS);
#pragma unroll
            for (int g = 0; g < 2; g++) {
                const uint4 *b = xs[g];
                const uint32_t *nib = reinterpret_cast<const uint32_t *>(blk) + (g * 128 + gid) * 4 + tig;
                const uint4 *sc = reinterpret_cast<const uint4 *>(blk + PK_NIB + (g * 128 + gid * 16) * 2);
                uint4 s4;
#pragma unroll
                for (int i = 0; i < 8; i++) {  // rows 16 i + gid and 16 i + 8 + gid
                    if (i % 4 == 0) s4 = sc[i / 4];
                    const uint32_t sb = i % 4 == 0 ? s4.x : i % 4 == 1 ? s4.y : i % 4 == 2 ? s4.z : s4.w;
                    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&sb));
                    uint32_t lo[4], up[4];
                    nibbles8<BF>(nib[16 * i * 4], lo);
                    nibbles8<BF>(nib[(16 * i + 8) * 4], up);
                    float d[NT][4];
#pragma unroll
                    for (int c = 0; c < NT; c++)
                        mma_first<BF>(d[c], lo[0], up[0], lo[1], up[1], b[c].x, b[c].y);
#pragma unroll
                    for (int c = 0; c < NT; c++)
                        mma_more<BF>(d[c], lo[2], up[2], lo[3], up[3], b[c].z, b[c].w);
#pragma unroll
                    for (int c = 0; c < NT; c++) {
                        acc[i][c][0] = fmaf(f.x, d[c][0], acc[i][c][0]);
                        acc[i][c][1] = fmaf(f.x, d[c][1], acc[i][c][1]);
                        acc[i][c][2] = fmaf(f.y, d[c][2], acc[i][c][2]);
                        acc[i][c][3] = fmaf(f.y, d[c][3], acc[i][c][3]);
                    }
                }
            }
            __syncwarp();
            fetch(kb + ST_SLOTS * ST_WARPS, slot);
            if (++slot == ST_SLOTS) {
                slot = 0;
                pass ^= 1u;
            }
        }
        if (!ok) {
            // the copies in flight end before the CTA does (bounded)
            atomicAdd(&g_linear_timeouts, 1u);
            const int go_on = 0;
            for (uint32_t s = 0; s < ST_SLOTS; s++)
                if (kb + s * ST_WARPS < kb1)
                    mbar_wait(smem_u32(&full[warp * ST_SLOTS + (slot + s) % ST_SLOTS]),
                              pass ^ (slot + s >= ST_SLOTS), &go_on);
        }
        // my sums, [row of x][128 features], over my ring (its copies are done)
        __syncwarp();
        float *part = reinterpret_cast<float *>(mine);
#pragma unroll
        for (int i = 0; i < 8; i++)
#pragma unroll
            for (int c = 0; c < NT; c++)
#pragma unroll
                for (int j = 0; j < 4; j++)
                    part[(8 * c + 2 * tig + (j & 1)) * 128 + 16 * i + 8 * (j >> 1) + gid] = acc[i][c][j];
    }
    __syncthreads();
    // a thread per row and 8 features: the warps' sums in warp order
    const uint32_t rows = work ? min(ROWS, hi - m0) : 0;
    const uint32_t row = threadIdx.x / 16, f = threadIdx.x % 16 * 8, n = n0 + f;
    float z[8] = {};
    if (row < rows) {
#pragma unroll
        for (int w = 0; w < ST_WARPS; w++) {
            const float4 *v = reinterpret_cast<const float4 *>(ring + w * ST_SLOTS * PK_BYTES) +
                              (row * 128 + f) / 4;
            const float4 a = v[0], b = v[1];
            z[0] += a.x, z[1] += a.y, z[2] += a.z, z[3] += a.w;
            z[4] += b.x, z[5] += b.y, z[6] += b.z, z[7] += b.w;
        }
    }
    // what the rows that this thread finishes need beside their sums
    const uint32_t mine = (row << q.shift) + rank;  // of a split: row r is finished by CTA r % split
    const bool mine_live = mine < rows && n < p.N;
    float bias[8];
    Operands o;
    if (mine_live) {
        load_bias8<BF>(p, e, n, bias);
        load_operands<OUT_ANY>(p, m0 + mine, n, o);
    }
    const auto finish = [&]() {
#pragma unroll
        for (int j = 0; j < 8; j++) z[j] = fmaf(ST_UNIT<BF>, z[j], bias[j]);
        finish8<BF, OUT_ANY>(p, z, o, m0 + mine, n);
    };
    if (q.split == 1) {
        if (mine_live) finish();
        return;
    }
    // CTA r % split receives the parts of row r at [r / split][source rank]
    asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
    if (row < rows) {
        const uint32_t at = smem_u32(recv + ((row >> q.shift << q.shift) + rank) * 128 + f);
        const uint32_t to = map_to(at, row & (q.split - 1));
        asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(to), "f"(z[0]),
                     "f"(z[1]), "f"(z[2]), "f"(z[3])
                     : "memory");
        asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(to + 16), "f"(z[4]),
                     "f"(z[5]), "f"(z[6]), "f"(z[7])
                     : "memory");
    }
    cluster_barrier();
    if (mine_live) {
#pragma unroll
        for (int j = 0; j < 8; j++) z[j] = 0.0f;
#pragma unroll
        for (uint32_t r = 0; r < 8; r++) {
            if (r >= q.split) break;
            const float4 *v = reinterpret_cast<const float4 *>(recv + ((row << q.shift) + r) * 128 + f);
            const float4 a = v[0], b = v[1];
            z[0] += a.x, z[1] += a.y, z[2] += a.z, z[3] += a.w;
            z[4] += b.x, z[5] += b.y, z[6] += b.z, z[7] += b.w;
        }
        finish();
    }
}

// ---- host side --------------------------------------------------------------------

int code_of(cudaError_t e) {
    if (e == cudaSuccess) return HCT_B200_OK;
    cudaGetLastError();  // it is reported here: nobody else finds it later
    if (e == cudaErrorMemoryAllocation) return HCT_B200_ERR_OUT_OF_MEMORY;
    if (e == cudaErrorNoDevice || e == cudaErrorInsufficientDriver) return HCT_B200_ERR_NO_DEVICE;
    return HCT_B200_ERR_CUDA;
}

// SMs of the current device.
uint32_t sm_count() {
    static PerDevice known;
    int dev = -1;
    cudaGetDevice(&dev);
    const uint32_t n = known.get(dev, [dev] {
        int c = 0;
        return cudaDeviceGetAttribute(&c, cudaDevAttrMultiProcessorCount, dev) == cudaSuccess && c > 0
                   ? (uint32_t)c
                   : 0u;
    });
    return n ? n : 148;
}

// A matrix in memory: rows of `width` bytes, `stride` bytes apart.
struct Extent {
    const void *p;
    uint64_t rows, width, stride;
    uint64_t span() const { return rows && width ? (rows - 1) * stride + width : 0; }
};

// Whether two matrices share a byte; rows of one buffer that sit side by side
// (equal strides, different columns) do not.
bool overlap(const Extent &a, const Extent &b) {
    const uint64_t sa = a.span(), sb = b.span();
    if (!a.p || !b.p || !sa || !sb) return false;
    const uint64_t pa = (uint64_t)(uintptr_t)a.p, pb = (uint64_t)(uintptr_t)b.p;
    if (pa + sa <= pb || pb + sb <= pa) return false;
    if (a.stride != b.stride || !a.stride) return true;
    const uint64_t d = (pb % a.stride + a.stride - pa % a.stride) % a.stride;
    return d < a.width || d + b.width > a.stride;
}

// What both calls check; *nothing where there is no output to write.
int check(const hct_b200_linear_args *a, bool grouped, bool *nothing) {
    *nothing = false;
    if (!a) return HCT_B200_ERR_INVALID_ARGUMENT;
    if (a->x_dtype != HCT_B200_F16 && a->x_dtype != HCT_B200_BF16)
        return HCT_B200_ERR_INVALID_ARGUMENT;
    if (a->out_dtype < HCT_B200_F32 || a->out_dtype > HCT_B200_BF16)
        return HCT_B200_ERR_INVALID_ARGUMENT;
    if (a->weight_form != HCT_B200_WEIGHT_DENSE && a->weight_form != HCT_B200_WEIGHT_INT4)
        return HCT_B200_ERR_INVALID_ARGUMENT;
    if (a->activation < HCT_B200_ACT_NONE || a->activation > HCT_B200_ACT_GELU_TANH)
        return HCT_B200_ERR_INVALID_ARGUMENT;
    if (a->reserved != 0) return HCT_B200_ERR_INVALID_ARGUMENT;
    if (a->d_bias && a->bias_dtype != HCT_B200_F32 && a->bias_dtype != a->x_dtype)
        return HCT_B200_ERR_INVALID_ARGUMENT;
    const uint64_t m = a->rows, n = a->out_features, k = a->in_features;
    if (m >= DIM_LIMIT || n >= DIM_LIMIT || k >= DIM_LIMIT) return HCT_B200_ERR_INVALID_ARGUMENT;
    const uint64_t e = grouped ? a->experts : 1;
    if (grouped) {
        if (a->offsets_bits != 32 && a->offsets_bits != 64) return HCT_B200_ERR_INVALID_ARGUMENT;
        if (e == 0 || e > MAX_EXPERTS) return HCT_B200_ERR_INVALID_ARGUMENT;
    }
    if (m == 0 || n == 0) {
        *nothing = true;
        return HCT_B200_OK;
    }
    // strides are bounded so that no byte offset leaves 64 bits
    const uint64_t lim = 1ull << 30;
    if (a->ldx > lim || a->ldw > lim || a->weight_stride > 1ull << 46 || a->ldgate > lim ||
        a->ldresidual > lim || a->ldout > lim)
        return HCT_B200_ERR_INVALID_ARGUMENT;
    if (!a->d_out || (grouped && !a->d_offsets)) return HCT_B200_ERR_INVALID_ARGUMENT;
    if (k && (!a->d_x || !a->d_weight)) return HCT_B200_ERR_INVALID_ARGUMENT;
    const uint64_t osz = a->out_dtype == HCT_B200_F32 ? 4 : 2;
    const auto misaligned = [](const void *p, uint64_t by) { return (uintptr_t)p % by != 0; };
    if (misaligned(a->d_out, osz) || misaligned(a->d_x, 2) || misaligned(a->d_gate, 2) ||
        misaligned(a->d_residual, osz) ||
        misaligned(a->d_bias, a->bias_dtype == HCT_B200_F32 ? 4 : 2) ||
        (grouped && misaligned(a->d_offsets, a->offsets_bits / 8)))
        return HCT_B200_ERR_INVALID_ARGUMENT;
    const bool dense = a->weight_form == HCT_B200_WEIGHT_DENSE;
    if (misaligned(a->d_weight, dense ? 2 : 128)) return HCT_B200_ERR_INVALID_ARGUMENT;
    if (!dense && k % 32) return HCT_B200_ERR_INVALID_ARGUMENT;
    if (m > 1 && a->ldout < n) return HCT_B200_ERR_INVALID_ARGUMENT;
    const Extent out{a->d_out, m, n * osz, a->ldout * osz};
    const Extent in[] = {
        {k ? a->d_x : nullptr, m, k * 2, a->ldx * 2},
        {a->d_bias, 1, e * n * (a->bias_dtype == HCT_B200_F32 ? 4 : 2), 0},
        {grouped ? a->d_offsets : nullptr, 1, (e + 1) * (uint64_t)(a->offsets_bits / 8), 0},
        {k && !dense ? a->d_weight : nullptr, 1, e * pk_bytes(n, k), 0},
        {k && dense ? a->d_weight : nullptr, 1,
         ((e - 1) * a->weight_stride + (n - 1) * a->ldw + k) * 2, 0},
    };
    for (const Extent &i : in)
        if (overlap(out, i)) return HCT_B200_ERR_INVALID_ARGUMENT;
    const Extent gate{a->d_gate, m, n * 2, a->ldgate * 2};
    const Extent res{a->d_residual, m, n * osz, a->ldresidual * osz};
    const bool same_gate = a->d_gate == a->d_out && osz == 2 && (m == 1 || a->ldgate == a->ldout);
    const bool same_res = a->d_residual == a->d_out && (m == 1 || a->ldresidual == a->ldout);
    if (!same_gate && overlap(out, gate)) return HCT_B200_ERR_INVALID_ARGUMENT;
    if (!same_res && overlap(out, res)) return HCT_B200_ERR_INVALID_ARGUMENT;
    return HCT_B200_OK;
}

using EncodeTiledFn = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *,
                                   const cuuint64_t *, const cuuint64_t *, const cuuint32_t *,
                                   const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                                   CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_fn() {
    static EncodeTiledFn fn = [] {
        void *q = nullptr;
        cudaDriverEntryPointQueryResult r;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &q, cudaEnableDefault, &r) !=
                cudaSuccess ||
            r != cudaDriverEntryPointSuccess)
            q = nullptr;
        return reinterpret_cast<EncodeTiledFn>(q);
    }();
    return fn;
}

// rows of K 16-bit values, `ld` apart, in `batch` matrices `bstride` apart:
// boxes of 64 values x box_rows rows of one matrix.  A 2-D map when batch is 0.
bool operand_map(CUtensorMap *map, bool bf, const void *base, uint64_t K, uint64_t rows, uint64_t ld,
                 uint64_t batch, uint64_t bstride, uint32_t box_rows) {
    const cuuint64_t dims[3] = {K, rows, batch};
    const cuuint64_t strides[2] = {ld * 2, bstride * 2};
    const cuuint32_t box[3] = {BK, box_rows, 1}, one[3] = {1, 1, 1};
    return encode_fn() &&
           encode_fn()(map,
                       bf ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                       batch ? 3 : 2, const_cast<void *>(base), dims, strides, box, one,
                       CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                       CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                       CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Rows that TMA can fetch: 16-byte aligned starts, no two rows overlapping.
bool tma_rows(const void *base, uint64_t rows, uint64_t ld, uint64_t K) {
    return (uintptr_t)base % 16 == 0 && (rows == 1 || (ld % 8 == 0 && ld >= K));
}

inline uint32_t round_to(uint32_t v, uint32_t m) { return (v + m - 1) / m * m; }

// Programmatic serialisation, and a cluster of more than one CTA.
unsigned launch_attributes(cudaLaunchAttribute (&attr)[2], uint32_t cluster) {
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    return cluster > 1 ? 2 : 1;
}

template <class Kernel>
cudaError_t allow_smem(Kernel kernel, uint32_t bytes, std::atomic<uint64_t> &set) {
    // once per device (64 of them remembered); twice by two threads does no harm
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 64 && (set.load(std::memory_order_relaxed) >> dev & 1)) return cudaSuccess;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    if (e == cudaSuccess && dev < 64) set.fetch_or(1ull << dev, std::memory_order_relaxed);
    return e;
}

template <int FORM, bool BF, bool PRECISE, bool PAIR>
cudaError_t launch_umma(const CUtensorMap &tx, const CUtensorMap &tw, const UmmaParams &u,
                        uint32_t grid, uint32_t smem, cudaStream_t s) {
    const auto kernel = linear_umma_kernel<FORM, BF, PRECISE, PAIR>;
    static std::atomic<uint64_t> set{0};
    cudaError_t e = allow_smem(kernel, SMEM_LIMIT, set);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t c = {};
    c.gridDim = dim3(grid);
    c.blockDim = dim3(umma_threads(FORM));
    c.dynamicSmemBytes = smem;
    c.stream = s;
    cudaLaunchAttribute attr[2];
    c.attrs = attr;
    c.numAttrs = launch_attributes(attr, PAIR ? 2 : u.split);
    return cudaLaunchKernelEx(&c, kernel, tx, tw, u);
}

// How many clusters of 2 .. 8 CTAs, one to an SM, the device holds at once: a GPC
// has room for whole ones only (clusters of 8: 8 to 16 of 18).  Asked once for
// each device and size.
uint32_t clusters_at_once(uint32_t size) {
    static PerDevice known[9];
    int dev = 0;
    if (size < 2 || cudaGetDevice(&dev) != cudaSuccess) return 0xffffffffu;
    return known[size].get(dev, [size] {
        const auto kernel = linear_umma_kernel<FORM_DENSE, true, false, false>;
        int n = 0;
        cudaLaunchAttribute attr[2];
        cudaLaunchConfig_t c = {};
        c.gridDim = dim3(size);
        c.blockDim = dim3(umma_threads(FORM_DENSE));
        c.dynamicSmemBytes = SMEM_MIN;
        c.attrs = attr;
        c.numAttrs = launch_attributes(attr, size);
        if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)SMEM_LIMIT) !=
                cudaSuccess ||
            cudaOccupancyMaxActiveClusters(&n, kernel, &c) != cudaSuccess || n < 1) {
            cudaGetLastError();
            n = 1;
        }
        return (uint32_t)n;
    });
}

// CTAs to a tile: the K range is split over a cluster where tiles leave half of
// the SMs idle, as far as all clusters run at once.
uint32_t split_of(uint64_t tiles, uint32_t sms, uint32_t kbs) {
    if (tiles * 2 > sms) return 1;
    uint32_t s = std::min<uint32_t>({8u, (uint32_t)(sms / tiles), kbs});
    while (s > 1 && clusters_at_once(s) < tiles) s--;
    return s;
}

// Rows per tile of M rows on pairs: the height whose waves of tiles take the least
// time, a K step being 2 clocks a row and at least its issuing.
uint32_t pair_rows(uint32_t M, uint32_t nt, uint32_t pairs, uint32_t cap) {
    if (M <= cap) return round_to(M, 16);
    uint32_t rows = cap;
    uint64_t best = ~0ull;
    for (uint32_t bn = cap; bn >= cap / 2; bn -= 16) {
        const uint64_t mts = (M + bn - 1) / bn;
        const uint32_t per = round_to((uint32_t)((M + mts - 1) / mts), 16);
        const uint64_t cost = (mts * nt + pairs - 1) / pairs * std::max(2 * per + 64, 550u);
        if (cost < best) {
            best = cost;
            rows = bn;
        }
    }
    return rows;
}

// Pair or single, tile height, split and ring depths of a call on the
// tensor-core kernel.
cudaError_t run_umma(const LinParams &p, bool grouped, int form, bool bf, cudaStream_t s) {
    const bool int4 = form == FORM_INT4, any = form >= FORM_ANY;
    const bool precise = p.odt == HCT_B200_F32;
    const uint32_t sms = sm_count(), cap = max_rows(form, precise);
    const uint32_t kbs = std::max((p.K + BK - 1) / BK, 1u);
    const uint32_t active = std::min(p.E, p.M), per_expert = p.M / active;
    UmmaParams u{};
    u.p = p;
    u.split = 1;
    // pairs where tiles of 256 features keep every pair busy
    const uint64_t pair_tiles = (uint64_t)((p.N + 255) / 256) * ((p.M + 255) / 256 + (active - 1) / 2);
    const bool pair = !precise && !any && per_expert > 64 && pair_tiles * 2 >= sms;
    const uint32_t nt = pair ? (p.N + 255) / 256 : (p.N + 127) / 128;
    // everything of a plan that follows from the rows that its tiles may have
    uint64_t tiles = 0;  // at most
    uint32_t fixed = 0, stage = 0;
    const auto plan = [&](uint32_t rows) {
        u.bn = rows;
        u.xbox = grouped ? 32 : pair ? rows / 2 : rows;
        tiles = (grouped ? (uint64_t)(p.M / rows + active) : (uint64_t)((p.M + rows - 1) / rows)) * nt;
        // two issuers where their accumulators fit TMEM twice and an operand ring of 6
        // slots (any even number without groups) fits shared memory
        stage = (int4 && precise ? 2 : 1) * A_BYTES + u.bn / (pair ? 2 : 1) * 128;
        u.issuers = u.bn <= (int4 ? 96u : 128u) && !(int4 && precise) ? 2 : 1;
        u.raw_stages = !int4 ? 0 : u.issuers == 2 && u.bn > 64 ? 6 : 9;
        const uint32_t other = u.raw_stages * PK_BYTES + EPI_BYTES;
        fixed = 1024 + other + (uint32_t)sizeof(Ctl) + groups_bytes(p.E);
        u.stages = std::min<uint32_t>(MAX_STAGES, (SMEM_LIMIT - fixed) / stage);
        if (u.issuers == 2) {
            if (form == FORM_DENSE) u.stages &= ~1u;
            else if (u.stages >= 6) u.stages = 6;
            else u.issuers = 1;  // many experts' tables
        }
        // a split tile's parts, the CTA's own and those it receives, take the place of
        // the rings and the staging, which are done with by then
        u.split = pair ? 1 : split_of(tiles, sms, kbs);
        while (u.split > 1 &&
               (u.bn + (u.bn + u.split - 1) / u.split * (u.split - 1)) * 512 > u.stages * stage + other)
            u.split--;
    };
    // Clocks of a plan, roughly: a K step takes its MMAs (2 a row), its issuing (300 with
    // two issuers, else 550; INT4 550), its bytes from L2 (50 a clock to an SM) or the copies
    // of its rows by warps (17 each, 11 in words; 4096 x 4096 x 1001 216 us, K = 1002 142), and
    // a split 2500 more and 40 for a row of its tile that is sent.
    const auto clocks = [&] {
        const uint32_t bytes = (int4 ? PK_BYTES : (uint32_t)A_BYTES) + u.bn * 128;
        const uint64_t step = any ? (128 + u.bn) * (form == FORM_ANY ? 17 : 11)
                                  : std::max({2 * u.bn, u.issuers == 2 && !int4 ? 300u : 550u, bytes / 50});
        return (tiles * u.split + sms - 1) / sms * ((kbs + u.split - 1) / u.split) * step +
               (u.split > 1 ? 2500 + 40 * u.bn * (u.split - 1) / u.split : 0);
    };
    if (pair) {
        plan(grouped ? cap : pair_rows(p.M, nt, sms / 2, cap));
    } else {
        // Lower tiles may use more SMs (196 x 1792 x 1664: 48 rows and 2 parts of K 9.4
        // us, 208 rows and 4 parts 13.6) or not (256 x 8192 x 8192 INT4: 256 rows and 2
        // parts 43 us, 128 rows 56).  linear: M in up to 6 tiles more than it needs,
        // of 48 rows or more (16 where copying bounds: 80 x 64 x 12511 40 us, 53 in one tile);
        // grouped, whose groups are not known here: some heights
        uint32_t best = 0;
        uint64_t least = ~0ull;
        const auto consider = [&](uint32_t rows) {
            plan(rows);
            if (clocks() < least) {
                least = clocks();
                best = rows;
            }
        };
        if (grouped) {
            const uint32_t most = std::min(cap, per_expert > 64 ? 256u : 128u);
            for (uint32_t rows = most; rows >= 64; rows -= 32) {
                consider(rows);
                if (tiles * 2 > sms) break;
            }
        } else {
            const uint32_t needed = (p.M + cap - 1) / cap;
            for (uint32_t mts = needed; mts < needed + 7; mts++) {
                const uint32_t rows = round_to((p.M + mts - 1) / mts, 16);
                if (rows < (any ? 16u : 48u) && mts > needed) break;
                consider(rows);
            }
        }
        plan(best);
    }
    if (tiles > 0x7fffffffull / 8) return cudaErrorInvalidValue;
    u.tmem_stride = round_to(u.bn, 32);
    u.tmem_cols = 64;
    while (u.tmem_cols < 2 * u.issuers * (int4 && precise ? 2 : 1) * u.tmem_stride) u.tmem_cols *= 2;
    u.tile = Divisor(u.bn);
    u.nt = Divisor(nt);
    u.band = Divisor(nt * RASTER);
    const uint32_t grid = pair          ? 2 * (uint32_t)std::min<uint64_t>(tiles, sms / 2)
                          : u.split > 1 ? (uint32_t)tiles * u.split
                                        : (uint32_t)std::min<uint64_t>(tiles, sms);
    const uint32_t smem = std::max(SMEM_MIN, fixed + u.stages * stage);

    alignas(64) CUtensorMap tx{}, tw{};
    if (!any && !operand_map(&tx, bf, p.x, p.K, p.M, p.M == 1 ? round_to(p.K, 8) : p.ldx, 0, 0, u.xbox))
        return cudaErrorInvalidValue;
    if (form == FORM_DENSE) {
        const uint64_t ld = p.N == 1 ? round_to(p.K, 8) : p.ldw;
        if (!operand_map(&tw, bf, p.w, p.K, p.N, ld, p.E, p.E == 1 ? ld * p.N : p.w_stride, 128))
            return cudaErrorInvalidValue;
    }
    const auto launch = [&](auto form_, auto bf_) {
        constexpr int F = decltype(form_)::value;
        constexpr bool B = decltype(bf_)::value;
        if (precise) return launch_umma<F, B, true, false>(tx, tw, u, grid, smem, s);
        if constexpr (F < FORM_ANY)
            if (pair) return launch_umma<F, B, false, true>(tx, tw, u, grid, smem, s);
        return launch_umma<F, B, false, false>(tx, tw, u, grid, smem, s);
    };
    const auto typed = [&](auto form_) {
        return bf ? launch(form_, std::true_type()) : launch(form_, std::false_type());
    };
    if (int4) return typed(std::integral_constant<int, FORM_INT4>());
    if (form == FORM_ANY) return typed(std::integral_constant<int, FORM_ANY>());
    if (form == FORM_WORDS) return typed(std::integral_constant<int, FORM_WORDS>());
    return typed(std::integral_constant<int, FORM_DENSE>());
}

template <bool BF, int NT>
cudaError_t launch_stream(const StreamParams &q, uint32_t grid, cudaStream_t s) {
    static std::atomic<uint64_t> set{0};
    const auto kernel = linear_int4_stream_kernel<BF, NT>;
    const uint32_t fixed = ST_WARPS * ST_SLOTS * (PK_BYTES + 8) + 8 * NT * 128 * 4 + 8;
    cudaError_t e = allow_smem(kernel, fixed + groups_bytes(MAX_EXPERTS), set);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t c = {};
    c.gridDim = dim3(grid);
    c.blockDim = dim3(ST_THREADS);
    c.dynamicSmemBytes = fixed + groups_bytes(q.p.E);
    c.stream = s;
    cudaLaunchAttribute attr[2];
    c.attrs = attr;
    c.numAttrs = launch_attributes(attr, q.split);
    return cudaLaunchKernelEx(&c, kernel, q);
}

constexpr uint32_t STREAM_ROWS = 16;  // rows (per expert with rows) up to which the stream kernel is taken

cudaError_t run_stream(const LinParams &p, bool bf, cudaStream_t s) {
    const uint32_t sms = sm_count(), kbs = (uint32_t)pk_kblocks(p.K);
    const uint32_t active = std::min(p.E, p.M);
    const bool two = p.M / active > 8 || (p.E == 1 && p.M > 8);
    StreamParams q{};
    q.p = p;
    q.vec_x = (uintptr_t)p.x % 16 == 0 && (p.M == 1 || p.ldx % 8 == 0);
    const uint64_t row_tiles = p.E == 1 ? (p.M + (two ? 15 : 7)) / (two ? 16 : 8)
                                        : p.M / (two ? 16 : 8) + active;
    q.tile = Divisor(two ? 16 : 8);
    q.nt = Divisor((p.N + 127) / 128);
    const uint64_t tiles = row_tiles * q.nt.d;
    if (tiles > 0x7fffffffull / 8) return cudaErrorInvalidValue;
    // two CTAs fit an SM; a part keeps at least a block for each warp
    q.split = 1;
    while (q.split < 8 && tiles * q.split * 2 <= 2 * sms && kbs >= q.split * 2 * ST_WARPS) q.split *= 2;
    while (1u << q.shift < q.split) q.shift++;
    const uint32_t grid = (uint32_t)tiles * q.split;
    if (bf) return two ? launch_stream<true, 2>(q, grid, s) : launch_stream<true, 1>(q, grid, s);
    return two ? launch_stream<false, 2>(q, grid, s) : launch_stream<false, 1>(q, grid, s);
}

int run(const hct_b200_linear_args *a, bool grouped, cudaStream_t s) {
    bool nothing = false;
    const int rc = check(a, grouped, &nothing);
    if (rc || nothing) return rc;
    LinParams p{};
    p.x = a->d_x;
    p.w = a->d_weight;
    p.bias = a->d_bias;
    p.gate = a->d_gate;
    p.res = a->d_residual;
    p.offsets = grouped ? a->d_offsets : nullptr;
    p.out = a->d_out;
    p.ldx = (uint32_t)a->ldx;
    p.ldw = (uint32_t)a->ldw;
    p.w_stride = a->weight_stride;
    p.ldgate = (uint32_t)a->ldgate;
    p.ldres = (uint32_t)a->ldresidual;
    p.ldo = (uint32_t)a->ldout;
    p.M = (uint32_t)a->rows;
    p.N = (uint32_t)a->out_features;
    p.K = (uint32_t)a->in_features;
    p.E = grouped ? a->experts : 1;
    p.off64 = a->offsets_bits == 64;
    p.bias_f32 = a->bias_dtype == HCT_B200_F32;
    p.act = a->activation;
    p.odt = a->out_dtype;
    const auto rows16 = [&](const void *q, uint64_t ld, uint64_t size) {
        return (uintptr_t)q % 16 == 0 && (p.M == 1 || ld * size % 16 == 0);
    };
    const uint64_t osz = p.odt == HCT_B200_F32 ? 4 : 2;
    p.vec_gate = rows16(p.gate, p.ldgate, 2);
    p.vec_res = rows16(p.res, p.ldres, osz);
    p.vec_out = rows16(p.out, p.ldo, osz);
    const bool bf = a->x_dtype == HCT_B200_BF16, int4 = a->weight_form == HCT_B200_WEIGHT_INT4;
    const bool x_rows = tma_rows(p.x, p.M, p.ldx, p.K);
    if (int4) {
        // the stream kernel for a few rows, and for any number of rows that TMA cannot
        // fetch or that are empty; but not for many tiles of fewer K blocks than its warps
        // (500 rows on 59 experts of 23104 x 224: 165 us here, 223 there)
        const uint32_t active = std::min(p.E, p.M);
        const bool shorts = p.E > 1 && pk_kblocks(p.K) < ST_WARPS &&
                            (uint64_t)active * ((p.N + 127) / 128) > 2ull * sm_count();
        if (!x_rows || !p.K || (p.M <= STREAM_ROWS * active && !shorts)) return code_of(run_stream(p, bf, s));
        return code_of(run_umma(p, grouped, FORM_INT4, bf, s));
    }
    const bool w_rows = tma_rows(p.w, p.N, p.ldw, p.K) &&
                        (p.E == 1 || (p.w_stride % 8 == 0 && p.w_stride && p.w_stride < 1ull << 38));
    if (p.K && x_rows && w_rows) return code_of(run_umma(p, grouped, FORM_DENSE, bf, s));
    // rows that TMA cannot fetch (500 x 5000 x 4002: 114 us with loads of 4 bytes, 195 of 2)
    const bool words = ((uintptr_t)p.x | (uintptr_t)p.w) % 4 == 0 && p.K % 2 == 0 &&
                       (p.M == 1 || p.ldx % 2 == 0) && (p.N == 1 || p.ldw % 2 == 0) &&
                       (p.E == 1 || p.w_stride % 2 == 0);
    return code_of(run_umma(p, grouped, words ? FORM_WORDS : FORM_ANY, bf, s));
}

}  // namespace
}  // namespace hct

extern "C" {

int hct_b200_linear(const hct_b200_linear_args *args, void *stream) {
    return hct::run(args, false, (cudaStream_t)stream);
}

int hct_b200_grouped_linear(const hct_b200_linear_args *args, void *stream) {
    return hct::run(args, true, (cudaStream_t)stream);
}

int hct_b200_linear_status(void *stream) {
    static hct::ReportedTimeouts reported;
    const cudaStream_t s = (cudaStream_t)stream;
    int dev = 0;
    uint32_t count = 0;
    cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess) e = cudaStreamIsCapturing(s, &capture);
    // a stream that is being captured cannot be waited for: the attempt would end the capture
    if (capture != cudaStreamCaptureStatusNone) return HCT_B200_ERR_UNSUPPORTED;
    if (e == cudaSuccess)
        e = cudaMemcpyFromSymbolAsync(&count, hct::g_linear_timeouts, sizeof(count), 0,
                                      cudaMemcpyDeviceToHost, s);
    if (e == cudaSuccess) e = cudaStreamSynchronize(s);
    if (e != cudaSuccess) return hct::code_of(e);
    return reported.report(dev, count) ? HCT_B200_ERR_TIMEOUT : HCT_B200_OK;
}

size_t hct_b200_int4_weight_bytes(size_t rows, size_t cols) {
    if (!rows || !cols || cols % 32 || rows >= hct::DIM_LIMIT || cols >= hct::DIM_LIMIT) return 0;
    return (size_t)hct::pk_bytes(rows, cols);
}

int hct_b200_int4_weight_pack(const uint8_t *d_data, size_t data_len, size_t rows, size_t cols,
                              void *d_packed, void *stream) {
    using namespace hct;
    const size_t bytes = hct_b200_int4_weight_bytes(rows, cols);
    if (!bytes || !d_data || !d_packed || (uintptr_t)d_packed % 128)
        return HCT_B200_ERR_INVALID_ARGUMENT;
    if (data_len < rows * cols / 16 + rows * cols / 2) return HCT_B200_ERR_SIZE_MISMATCH;
    const uint64_t tasks = bytes / PK_BYTES * 2 * PK_ROWS;
    const unsigned grid = (unsigned)std::min<uint64_t>((tasks + 255) / 256, 32ull * sm_count());
    int4_weight_pack_kernel<<<grid, 256, 0, (cudaStream_t)stream>>>(
        d_data, rows, cols, static_cast<uint8_t *>(d_packed), tasks);
    return code_of(cudaGetLastError());
}

}  // extern "C"
