// Products with decoded weights: linear and grouped_linear.
//
//     out[i][j] = act(sum_k x[i][k] w[j][k] + bias[j]) * gate[i][j] + residual[i][j]
//
// linear is grouped_linear with one expert that owns every row.  Weights are
// dense matrices of x's type or INT4 payloads laid out by
// hct_b200_int4_weight_pack (see Int4Block).
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "common.cuh"

namespace hct {
namespace {

constexpr uint32_t MAX_EXPERTS = 1024;
constexpr uint64_t DIM_LIMIT = 1ull << 31;

// ---- packed INT4 weights ------------------------------------------------------
//
// A packed matrix is a sequence of blocks [ceil(rows / 128)][ceil(cols / 64)],
// each 128 rows x 64 columns (two scale blocks per row), 4608 contiguous
// bytes, so that one bulk copy brings everything a K step of a tile needs:
//   nibbles  [2 scale blocks][128 rows][16 bytes]   (16 B per thread, conflict-free)
//   scales   [2 scale blocks][128 rows] f16
// Each 32-bit word holds the 8 values k = 8 c .. 8 c + 7 of its scale block,
// value 2 j in bits 4 j .. 4 j + 3 and value 2 j + 1 in bits 16 + 4 j .., so
// that (word >> 4 j) & 0x000f000f is the pair (2 j, 2 j + 1) in two 16-bit
// halves.  Rows and scale blocks past the matrix hold zero scales.
constexpr uint32_t PK_ROWS = 128, PK_COLS = 64;
constexpr uint32_t PK_NIB = PK_ROWS * PK_COLS / 2;       // 4096
constexpr uint32_t PK_BYTES = PK_NIB + PK_ROWS * 2 * 2;  // 4608

__host__ __device__ inline uint64_t pk_kblocks(uint64_t cols) { return (cols + PK_COLS - 1) / PK_COLS; }
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
        *reinterpret_cast<uint16_t *>(o + PK_NIB + in * 2) = scale;
    }
}

// ---- what every kernel is given -------------------------------------------------

struct LinParams {
    const void *x, *w, *bias, *gate, *res, *offsets;
    void *out;
    uint64_t ldx, ldw, w_stride, ldgate, ldres, ldo;
    uint32_t M, N, K, E;
    int off64;  // offsets are int64 (else int32)
    int bias_f32, act, odt;
};

// Rows [lo, hi) of expert e, clamped to [0, M] and to lo <= hi; without
// offsets the one expert owns every row.
__device__ __forceinline__ void expert_rows(const LinParams &p, uint32_t e, uint32_t &lo,
                                            uint32_t &hi) {
    if (!p.offsets) {
        lo = 0;
        hi = p.M;
        return;
    }
    int64_t a, b;
    if (p.off64) {
        a = reinterpret_cast<const int64_t *>(p.offsets)[e];
        b = reinterpret_cast<const int64_t *>(p.offsets)[e + 1];
    } else {
        a = reinterpret_cast<const int32_t *>(p.offsets)[e];
        b = reinterpret_cast<const int32_t *>(p.offsets)[e + 1];
    }
    const int64_t m = (int64_t)p.M;
    a = a < 0 ? 0 : a > m ? m : a;
    b = b < a ? a : b > m ? m : b;
    lo = (uint32_t)a;
    hi = (uint32_t)b;
}

// first[e] = number of `tile`-row tiles of the experts before e, first[E] =
// their total.  Called by one whole warp; first is shared memory.
__device__ __forceinline__ void scan_tiles(const LinParams &p, uint32_t tile, uint32_t *first) {
    const uint32_t lane = threadIdx.x & 31u;
    uint32_t base = 0;
    for (uint32_t e0 = 0; e0 < p.E; e0 += 32) {
        const uint32_t e = e0 + lane;
        uint32_t lo = 0, hi = 0;
        if (e < p.E) expert_rows(p, e, lo, hi);
        uint32_t c = (hi - lo + tile - 1) / tile, s = c;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const uint32_t v = __shfl_up_sync(0xffffffffu, s, d);
            if (lane >= (uint32_t)d) s += v;
        }
        if (e < p.E) first[e] = base + s - c;
        base += __shfl_sync(0xffffffffu, s, 31);
    }
    if (lane == 0) first[p.E] = base;
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

__device__ __forceinline__ float h2f(uint16_t v) { return __half2float(__ushort_as_half(v)); }
__device__ __forceinline__ float bf2f(uint16_t v) { return __uint_as_float((uint32_t)v << 16); }
template <bool BF>
__device__ __forceinline__ float from16(uint16_t v) {
    return BF ? bf2f(v) : h2f(v);
}

__device__ __forceinline__ float activate(float z, int act) {
    switch (act) {
        case HCT_B200_ACT_RELU: return z < 0.0f ? 0.0f : z;
        case HCT_B200_ACT_SILU: return z / (1.0f + expf(-z));
        case HCT_B200_ACT_GELU: return 0.5f * z * (1.0f + erff(z * 0.70710678118654752f));
        case HCT_B200_ACT_GELU_TANH:
            return 0.5f * z * (1.0f + tanhf(0.79788456080286536f * (z + 0.044715f * z * z * z)));
        default: return z;
    }
}

__device__ __forceinline__ float load_out_type(const void *p, uint64_t i, int dt) {
    if (dt == HCT_B200_F32) return reinterpret_cast<const float *>(p)[i];
    const uint16_t v = reinterpret_cast<const uint16_t *>(p)[i];
    return dt == HCT_B200_F16 ? h2f(v) : bf2f(v);
}
__device__ __forceinline__ void store_out(void *p, uint64_t i, int dt, float v) {
    if (dt == HCT_B200_F32) reinterpret_cast<float *>(p)[i] = v;
    else if (dt == HCT_B200_F16) reinterpret_cast<__half *>(p)[i] = __float2half_rn(v);
    else reinterpret_cast<__nv_bfloat16 *>(p)[i] = __float2bfloat16_rn(v);
}

template <bool BF>
__device__ __forceinline__ float bias_of(const LinParams &p, uint32_t e, uint32_t n) {
    if (!p.bias) return 0.0f;
    const uint64_t i = (uint64_t)e * p.N + n;
    return p.bias_f32 ? reinterpret_cast<const float *>(p.bias)[i]
                      : from16<BF>(reinterpret_cast<const uint16_t *>(p.bias)[i]);
}

// The epilogue of one output: z is the sum plus bias.
template <bool BF>
__device__ __forceinline__ void finish(const LinParams &p, uint32_t m, uint32_t n, float z) {
    float y = activate(z, p.act);
    if (p.gate)
        y *= from16<BF>(reinterpret_cast<const uint16_t *>(p.gate)[(uint64_t)m * p.ldgate + n]);
    if (p.res) y += load_out_type(p.res, (uint64_t)m * p.ldres + n, p.odt);
    store_out(p.out, (uint64_t)m * p.ldo + n, p.odt, y);
}

// ---- plain kernel: any alignment, any stride ------------------------------------
//
// 32 rows x 64 features per CTA, 32-wide K steps through shared memory, f32
// multiply-adds (2 x 4 outputs per thread).  Every element is loaded by itself
// and checked against its bounds.
constexpr int SM_M = 32, SM_N = 64, SM_K = 32, SM_THREADS = 256;

template <bool BF, bool INT4>
__global__ void __launch_bounds__(SM_THREADS) linear_plain_kernel(const LinParams p) {
    __shared__ uint32_t first[MAX_EXPERTS + 1];
    __shared__ float xs[SM_K][SM_M + 1], ws[SM_K][SM_N + 1];
    const uint32_t tid = threadIdx.x;
    if (tid < 32) scan_tiles(p, SM_M, first);
    __syncthreads();
    const uint32_t n_tiles = (p.N + SM_N - 1) / SM_N;
    const uint64_t tiles = (uint64_t)first[p.E] * n_tiles;
    const uint32_t tn = tid % 16, tm = tid / 16;
    for (uint64_t t = blockIdx.x; t < tiles; t += gridDim.x) {
        const uint32_t mt = (uint32_t)(t / n_tiles), n0 = (uint32_t)(t % n_tiles) * SM_N;
        const uint32_t e = expert_of(first, p.E, mt);
        uint32_t lo, hi;
        expert_rows(p, e, lo, hi);
        const uint32_t m0 = lo + (mt - first[e]) * SM_M;
        float acc[2][4] = {};
        for (uint32_t k0 = 0; k0 < p.K; k0 += SM_K) {
            for (uint32_t i = tid; i < SM_M * SM_K; i += SM_THREADS) {
                const uint32_t k = k0 + i % SM_K, m = m0 + i / SM_K;
                xs[i % SM_K][i / SM_K] =
                    k < p.K && m < hi
                        ? from16<BF>(reinterpret_cast<const uint16_t *>(p.x)[(uint64_t)m * p.ldx + k])
                        : 0.0f;
            }
            for (uint32_t i = tid; i < SM_N * SM_K; i += SM_THREADS) {
                const uint32_t k = k0 + i % SM_K, n = n0 + i / SM_K;
                float v = 0.0f;
                if (k < p.K && n < p.N) {
                    if (INT4) {
                        const uint64_t kb = pk_kblocks(p.K);
                        const uint64_t per = (uint64_t)((p.N + PK_ROWS - 1) / PK_ROWS) * kb;
                        const uint8_t *b = reinterpret_cast<const uint8_t *>(p.w) +
                                           (e * per + n / PK_ROWS * kb + k / PK_COLS) * PK_BYTES;
                        const uint32_t in = (k / 32 % 2) * PK_ROWS + n % PK_ROWS, c = k / 8 % 4;
                        const uint32_t word = *reinterpret_cast<const uint32_t *>(b + in * 16 + c * 4);
                        const uint32_t q = word >> (4 * (k % 8 / 2) + 16 * (k % 2)) & 15u;
                        v = (float)((int)q - 8) *
                            h2f(*reinterpret_cast<const uint16_t *>(b + PK_NIB + in * 2));
                    } else {
                        v = from16<BF>(reinterpret_cast<const uint16_t *>(
                            p.w)[(uint64_t)e * p.w_stride + (uint64_t)n * p.ldw + k]);
                    }
                }
                ws[i % SM_K][i / SM_K] = v;
            }
            __syncthreads();
#pragma unroll 8
            for (int k = 0; k < SM_K; k++) {
                float a[2], b[4];
#pragma unroll
                for (int i = 0; i < 2; i++) a[i] = xs[k][tm + 16 * i];
#pragma unroll
                for (int j = 0; j < 4; j++) b[j] = ws[k][tn + 16 * j];
#pragma unroll
                for (int i = 0; i < 2; i++)
#pragma unroll
                    for (int j = 0; j < 4; j++) acc[i][j] = fmaf(a[i], b[j], acc[i][j]);
            }
            __syncthreads();
        }
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const uint32_t m = m0 + tm + 16 * i, n = n0 + tn + 16 * j;
                if (m < hi && n < p.N) finish<BF>(p, m, n, acc[i][j] + bias_of<BF>(p, e, n));
            }
    }
}

__device__ int g_linear_status;  // HCT_B200_ERR_TIMEOUT once a bounded wait has expired

// ---- host side --------------------------------------------------------------------

int code_of(cudaError_t e) {
    if (e == cudaSuccess) return HCT_B200_OK;
    if (e == cudaErrorMemoryAllocation) return HCT_B200_ERR_OUT_OF_MEMORY;
    if (e == cudaErrorNoDevice || e == cudaErrorInsufficientDriver) return HCT_B200_ERR_NO_DEVICE;
    return HCT_B200_ERR_CUDA;
}

int sm_count() {
    static int n = 0;
    if (!n) {
        int dev = 0, c = 0;
        if (cudaGetDevice(&dev) != cudaSuccess ||
            cudaDeviceGetAttribute(&c, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || c <= 0)
            c = 148;
        n = c;
    }
    return n;
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
    p.ldx = a->ldx;
    p.ldw = a->ldw;
    p.w_stride = a->weight_stride;
    p.ldgate = a->ldgate;
    p.ldres = a->ldresidual;
    p.ldo = a->ldout;
    p.M = (uint32_t)a->rows;
    p.N = (uint32_t)a->out_features;
    p.K = (uint32_t)a->in_features;
    p.E = grouped ? a->experts : 1;
    p.off64 = a->offsets_bits == 64;
    p.bias_f32 = a->bias_dtype == HCT_B200_F32;
    p.act = a->activation;
    p.odt = a->out_dtype;
    const bool bf = a->x_dtype == HCT_B200_BF16, int4 = a->weight_form == HCT_B200_WEIGHT_INT4;
    // at most this many row tiles: one partial tile per expert beside the whole ones
    const uint64_t mt = p.M / SM_M + std::min<uint64_t>(p.E, p.M);
    const uint64_t tiles = mt * ((p.N + SM_N - 1) / SM_N);
    const unsigned grid = (unsigned)std::min<uint64_t>(tiles, 8ull * sm_count());
    if (bf && int4) linear_plain_kernel<true, true><<<grid, SM_THREADS, 0, s>>>(p);
    else if (bf) linear_plain_kernel<true, false><<<grid, SM_THREADS, 0, s>>>(p);
    else if (int4) linear_plain_kernel<false, true><<<grid, SM_THREADS, 0, s>>>(p);
    else linear_plain_kernel<false, false><<<grid, SM_THREADS, 0, s>>>(p);
    return code_of(cudaGetLastError());
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
    const cudaStream_t s = (cudaStream_t)stream;
    int got = 0;
    cudaError_t e = cudaMemcpyFromSymbolAsync(&got, hct::g_linear_status, sizeof(int), 0,
                                              cudaMemcpyDeviceToHost, s);
    if (e == cudaSuccess) e = cudaStreamSynchronize(s);
    if (e != cudaSuccess) return hct::code_of(e);
    if (got) {
        const int zero = 0;
        e = cudaMemcpyToSymbolAsync(hct::g_linear_status, &zero, sizeof(int), 0,
                                    cudaMemcpyHostToDevice, s);
        if (e == cudaSuccess) e = cudaStreamSynchronize(s);
        if (e != cudaSuccess) return hct::code_of(e);
    }
    return got;
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
