// out = residual + act(x . w^T + bias), its backward, and what both need around the matrix products.
//
//   z = x w^T + bias     x [M, K], w [N, K] bf16, bias [N], residual [M, N] optional
//   backward: dz = dout act'(z);  dx = dz w;  dw = dz^T x;  dbias = sum of dz over the rows;  dresidual = dout
// Products on the matrix pipe with fp32 accumulation; bias, activation and residual are applied to the fp32 sums, one rounding
// at the store.  Two more roundings to bf16 in a training step with an activation, both of which any bf16 autograd makes: z is kept in
// bf16 for the slope (fp32 would double what a layer keeps until its backward), and dz goes to the matrix pipe in bf16 (as a sum of two
// it would double the time of both products).  Relative error of dx and dw against 64 bits, 16384 x 1024 -> 4096: 1.66e-3 without an
// activation (the store's own rounding), 2.41e-3 with gelu, gelu_tanh or silu (dz 1.66e-3, z 0.5e-3), 2.87e-3 with relu2, whose slope is z
// itself; dbias, summed before dz is rounded: 1.70, 1.70 and 2.32e-3.
#include "gemm_tn.h"
#include "host_util.h"
#include "launch.h"
#include "linear.h"
#include <algorithm>

namespace ngpt {
// gemm_api.hip
int64_t balanced_part_bytes(int R, int C, int K);
int64_t balanced_part_bytes_here(int R, int C, int K);
int gemm_bf16_clipped(const void* A, int fa, int64_t lda, const void* B, int fb, int64_t ldb, int R, int C, int K, int R_out, int C_out,
                      void* out_bf16, int64_t ldc, float* part32, hipStream_t st);

namespace {

// ---------------------------------------------------------------------------------------------- epilogue of the tile GEMM
// One kernel an activation: five of them behind a switch in one kernel cost it 60 spilled registers.
template <int ACT, bool PRE, bool RES>
struct EpiLinear {
    LinearOut o;
    static constexpr int EXTRA_LDS = 32768;         // 4 KiB per wave
    static constexpr bool NEEDS_SCRATCH = false;
    static constexpr bool JOB_END_NEEDS_SCRATCH = false;
    static constexpr bool DROPS_FRAGMENTS = true;   // the residual's lines in flight next to the accumulators
    static constexpr int TILE_STORES = 16;          // at least: 4 per 32-row block and wave (those past the matrix' end are issued too)
    uint8_t* stage;
    bool stored_all;
    __device__ bool all_stores_issued() const { return stored_all; }
    __device__ void partial(bool, int) {}
    __device__ void begin(int, int, uint8_t* extra) {
        stage = extra + (threadIdx.x >> 6) * 4096;
        stored_all = false;
    }
    __device__ void end(uint8_t*, int, int) {}
    template <class Cfg>
    __device__ void job_begin(int) {}
    template <class Cfg>
    __device__ void job_end(int, int, const AccCoords<Cfg>&, uint8_t*) {}
    template <class Cfg>
    __device__ __forceinline__ void tile(v16f (&acc)[Cfg::TM][Cfg::TN], int r0, int c0, const AccCoords<Cfg>& co, uint8_t*, int lane) {
        static_assert(Cfg::TM == 2 && Cfg::TN == 4 && Cfg::NWAVES * 4096 <= EXTRA_LDS, "64 x 128 wave tiles, 4 KiB of staging each");
        stored_all = o.vec != 0;
        linear_epilogue<ACT, PRE, RES>(o, acc, stage, r0 + co.wave_row0, c0 + co.wave_col0, lane);
    }
};

// ---------------------------------------------------------------------------------------------- around the products
// dst [rows_p, cols_p] = src [rows, cols] with zeros around it; cols_p % 8 == 0.
__global__ __launch_bounds__(256) void pad_copy_kernel(const uint16_t* __restrict__ src, int64_t ld, int rows, int cols, uint16_t* __restrict__ dst,
                                                       int rows_p, int cols_p) {
    const int c8 = cols_p / 8;
    const int64_t n = (int64_t)rows_p * c8;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        const int r = (int)(i / c8), c = (int)(i - (int64_t)r * c8) * 8;
        v4i w = {0, 0, 0, 0};
        if (r < rows && c < cols) w = load_row8(src + (int64_t)r * ld, c, cols);
        *(v4i*)(dst + i * 8) = w;
    }
}

// dst [cols, rows_p] = transpose of src [rows, cols], zeros behind its rows; rows_p % 64 == 0.  64 x 64 blocks through LDS: 16-byte pieces in
// (at any address) and out.
__global__ __launch_bounds__(256) void transpose_pad_kernel(const uint16_t* __restrict__ src, int64_t ld, int rows, int cols, uint16_t* __restrict__ dst,
                                                            int rows_p) {
    __shared__ uint16_t tile[64][64 + 4];
    const int r0 = blockIdx.x * 64, c0 = blockIdx.y * 64, t = threadIdx.x;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int r = (t >> 3) + 32 * i, c = (t & 7) * 8, left = cols - c0 - c;
        v4i w = {0, 0, 0, 0};
        if (r0 + r < rows && left > 0) w = load_row8(src + (int64_t)(r0 + r) * ld, c0 + c, cols);
#pragma unroll
        for (int e = 0; e < 4; ++e) *(uint32_t*)&tile[r][c + 2 * e] = (uint32_t)w[e];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int c = (t >> 3) + 32 * i, r = (t & 7) * 8;
        if (c0 + c >= cols) continue;
        v4i w;
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = (int)((uint32_t)tile[r + 2 * e][c] | ((uint32_t)tile[r + 2 * e + 1][c] << 16));
        *(v4i*)(dst + (int64_t)(c0 + c) * rows_p + r0 + r) = w;
    }
}

// dz = dout act'(z) (zeros in the padding of its [rows_p, cols_p]) and the column sums of dz, in fp32 before dz is rounded: a workgroup
// covers 256 columns and every gridDim.y-th group of 8 rows, its sums go to part[blockIdx.y][N].  dz or part may be null.
// 16384 x 4096 with gelu_tanh: 70 to 72 us (403 MB, 5.6 TB/s, partly from the cache); sums alone, 49152 x 768: 13 us.
constexpr int kColsPerBlock = 256, kRowLanes = 8;
template <int ACT>
__global__ __launch_bounds__(256) void act_grad_kernel(const uint16_t* __restrict__ dout, const uint16_t* __restrict__ pre, int M, int N,
                                                       uint16_t* __restrict__ dz, int rows_p, int cols_p, float* __restrict__ part) {
    __shared__ float red[kRowLanes][kColsPerBlock + 4];
    const int ct = threadIdx.x & 31, rt = threadIdx.x >> 5;
    const int c = blockIdx.x * kColsPerBlock + ct * 8;
    float sum[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (c < cols_p) {
        for (int r = blockIdx.y * kRowLanes + rt; r < rows_p; r += gridDim.y * kRowLanes) {
            v4i g = {0, 0, 0, 0}, o = {0, 0, 0, 0};
            if (r < M && c < N) {
                g = load_row8(dout + (int64_t)r * N, c, N);
                if constexpr (ACT == NGPT_ACT_NONE) {
                    o = g;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        sum[2 * i] += lo16(g[i]);
                        sum[2 * i + 1] += hi16(g[i]);
                    }
                } else {
                    const v4i z = load_row8(pre + (int64_t)r * N, c, N);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float d0 = lo16(g[i]) * act_slope<ACT>(lo16(z[i])), d1 = hi16(g[i]) * act_slope<ACT>(hi16(z[i]));
                        sum[2 * i] += d0;
                        sum[2 * i + 1] += d1;
                        o[i] = (int)cvt_pk_bf16(d0, d1);
                    }
                }
            }
            if (dz) *(v4i*)(dz + (int64_t)r * cols_p + c) = o;
        }
    }
    if (!part) return;
#pragma unroll
    for (int i = 0; i < 8; ++i) red[rt][ct * 8 + i] = sum[i];
    __syncthreads();
    const int col = blockIdx.x * kColsPerBlock + threadIdx.x;
    if (col < N) {
        float v = 0.0f;
#pragma unroll
        for (int i = 0; i < kRowLanes; ++i) v += red[i][threadIdx.x];
        part[(int64_t)blockIdx.y * N + col] = v;
    }
}

// out[c] = bf16(sum over p of part[p][c]), 32 columns a workgroup
__global__ __launch_bounds__(kColSumThreads) void col_sum_kernel(const float* __restrict__ part, int parts, int N, uint16_t* __restrict__ out) {
    __shared__ float red[32][33];
    const int col = blockIdx.x * 32 + (threadIdx.x & 31);
    const float v = col_sum32(part, parts, N, col, col < N, red);
    if (threadIdx.x < 32 && col < N) out[col] = (uint16_t)cvt_pk_bf16(v, v);
}

int64_t up64(int64_t n) { return (n + 63) / 64 * 64; }
int64_t up8(int64_t n) { return (n + 7) / 8 * 8; }
bool on16(const void* p) { return ((uintptr_t)p & 15) == 0; }

int pad_copy(const void* src, int64_t ld, int64_t rows, int64_t cols, void* dst, int64_t rows_p, int64_t cols_p, hipStream_t st) {
    const int64_t n = rows_p * cols_p / 8;
    const int64_t cap = (int64_t)std::max(num_cus(), 1) * 16;
    const int grid = (int)std::min<int64_t>((n + 255) / 256, cap);
    pad_copy_kernel<<<grid, 256, 0, st>>>((const uint16_t*)src, ld, (int)rows, (int)cols, (uint16_t*)dst, (int)rows_p, (int)cols_p);
    return check_launch("pad_copy_kernel");
}

int transpose_pad(const uint16_t* src, int64_t ld, int rows, int cols, uint16_t* dst, int rows_p, hipStream_t st) {
    if ((cols + 63) / 64 > 65535) return fail(NGPT_ERANGE, "transpose_pad: %d columns", cols);
    transpose_pad_kernel<<<dim3(rows_p / 64, (cols + 63) / 64), 256, 0, st>>>(src, ld, rows, cols, dst, rows_p);
    return check_launch("transpose_pad_kernel");
}

// Workgroups along the rows of act_grad_kernel, whatever the device
int act_grad_rows(int64_t M, int64_t N) {
    const int64_t cols = (N + kColsPerBlock - 1) / kColsPerBlock;
    int64_t rows = std::min<int64_t>((M + kRowLanes - 1) / kRowLanes, std::max<int64_t>(1, 2048 / cols));
    return (int)std::max<int64_t>(rows, 1);
}

constexpr int64_t kMaxStride = NGPT_LINEAR_MAX_STRIDE;      // values between rows: 256 rows of a tile lie within 32-bit byte offsets

int check_linear(const char* who, int M, int N, int K, int act) {
    if (M <= 0 || N <= 0 || K <= 0) return fail(NGPT_EINVAL, "%s: empty problem M=%d N=%d K=%d", who, M, N, K);
    if (act < NGPT_ACT_NONE || act > NGPT_ACT_SILU) return fail(NGPT_EINVAL, "%s: activation=%d", who, act);
    if (M > (1 << 29) || N > kMaxStride || K > kMaxStride) return fail(NGPT_ERANGE, "%s: M=%d N=%d K=%d: at most 2^29 rows, 2^21 values each", who, M, N, K);
    return NGPT_OK;
}

// The 256 x 256 tile GEMM reads rows that start on 16 bytes, a multiple of 64 values long.
bool rows_fit(const void* p, int64_t ld, int K) { return K % 64 == 0 && on16(p) && ld % 8 == 0; }

int linear_big(const LinearOut& o, const void* x, int64_t ldx, const void* w, int64_t ldw, int K, int act, hipStream_t st) {
    GemmOperands g{(const uint8_t*)w, (const uint8_t*)x, 2 * ldw, 2 * ldx, o.N, o.M, 2 * K, 1};
    auto go = [&](auto epi) {
        epi.o = o;
        return launch_gemm_fmt<MainCfg, FMT_BF16, FMT_BF16>(g, epi, st, 0);
    };
    return with_act(act, [&](auto kind) {
        constexpr int A = decltype(kind)::value;
        if constexpr (A != NGPT_ACT_NONE) {
            if (o.pre) return o.res ? go(EpiLinear<A, true, true>{}) : go(EpiLinear<A, true, false>{});
        }
        return o.res ? go(EpiLinear<A, false, true>{}) : go(EpiLinear<A, false, false>{});
    });
}

// Which kernel.  The 256 x 256 tiles run at 950 TFLOP/s in full rounds of the compute units (4096 x 4096 x 1024: 36 us), the 128 x 128 tiles at
// 730 (47 us) but with a finer end: the large ones serve full rounds and a last round that is three quarters full (192 of 256: 25 against
// 29 us; 128 of 256: 27 against 24), the rest of the rows goes to the others.
int linear_run(LinearOut o, const uint16_t* x, int64_t ldx, const uint16_t* w, int64_t ldw, int K, int act, hipStream_t st) {
    if (o.M > kFewRows && rows_fit(x, ldx, K) && rows_fit(w, ldw, K)) {
        const int64_t cus = num_cus(), tf = (o.N + 255) / 256, tiles = tf * ((o.M + 255) / 256);
        if (cus <= 0) return fail(NGPT_EINVAL, "no HIP device");
        const int64_t last = tiles % cus;
        if (last == 0 || 4 * last >= 3 * cus) return linear_big(o, x, ldx, w, ldw, K, act, st);
        const int64_t rows = tiles / cus * cus / tf * 256;
        if (rows > 0 && rows < o.M) {
            LinearOut head = o;
            head.M = (int)rows;
            if (int e = linear_big(head, x, ldx, w, ldw, K, act, st)) return e;
            o.M -= (int)rows;
            o.out += rows * o.N;
            if (o.pre) o.pre += rows * o.N;
            if (o.res) o.res += rows * o.ld_res;
            x += rows * ldx;
        }
    }
    return o.M <= kFewRows ? linear_few(o, x, ldx, w, ldw, K, act, st) : linear_mid(o, x, ldx, w, ldw, K, act, st);
}

}  // namespace
}  // namespace ngpt

using namespace ngpt;

extern "C" int ngpt_linear_act_fwd(const void* x_bf16, int64_t ldx, const void* w_bf16, int64_t ldw, const void* bias_bf16,
                                   const void* residual_bf16, int64_t ld_residual, int M, int N, int K, int activation,
                                   void* out_bf16, void* pre_bf16, void* stream) {
    const char* who = "ngpt_linear_act_fwd";
    if (!x_bf16 || !w_bf16 || !out_bf16) return fail(NGPT_EINVAL, "%s: null pointer", who);
    if (int e = check_linear(who, M, N, K, activation)) return e;
    if (pre_bf16 && activation == NGPT_ACT_NONE) return fail(NGPT_EINVAL, "%s: pre is for activations", who);
    if (!on16(bias_bf16)) return fail(NGPT_EALIGN, "%s: the bias starts on 16 bytes", who);
    if (ldx < K || ldw < K || (residual_bf16 && ld_residual < N))
        return fail(NGPT_EALIGN, "%s: row strides ldx=%lld ldw=%lld ld_residual=%lld", who, (long long)ldx, (long long)ldw, (long long)ld_residual);
    if (ldx > kMaxStride || ldw > kMaxStride || (residual_bf16 && ld_residual > kMaxStride))
        return fail(NGPT_ERANGE, "%s: row strides of at most 2^21 values (ldx=%lld ldw=%lld ld_residual=%lld)", who, (long long)ldx, (long long)ldw,
                    (long long)ld_residual);
    hipStream_t st = (hipStream_t)stream;
    LinearOut o{(uint16_t*)out_bf16, (uint16_t*)pre_bf16, (const uint16_t*)bias_bf16, (const uint16_t*)residual_bf16, ld_residual, M, N, 0, 0};
    o.vec = N % 8 == 0 && on16(out_bf16) && on16(pre_bf16);
    o.vec_res = residual_bf16 && N % 8 == 0 && ld_residual % 8 == 0 && on16(residual_bf16);
    ProfileScope prof(PROF_GEMM_BF16, st);
    return linear_run(o, (const uint16_t*)x_bf16, ldx, (const uint16_t*)w_bf16, ldw, K, activation, st);
}

namespace ngpt {
namespace {
// Workspace of the backward: dz [M64, N64] | w^T [K, N64] | x [M64, K8] | parts of dw's split tiles | column sums, each of them where the
// call has a use for it.
struct BwdPlan {
    int64_t M64, N64, K8, dz, w, x, parts, sums, total;
    int sum_rows;
    bool own_dz;      // dz is dout itself where there is no activation and the products can read it in place
    bool copy_x;      // where dw's product cannot read x in place
    // the most that a call of these sizes can use, on any device
    BwdPlan(int M, int N, int K) : own_dz(true), copy_x(true) {
        lay_out(M, N, K, true, true, balanced_part_bytes((int)up64(N), (int)up8(K), (int)(2 * up64(M))));
    }
    // one call on the current device
    BwdPlan(int M, int N, int K, int act, const void* dout, const void* x_, int64_t ldx, bool dx, bool dw, bool dbias) {
        own_dz = (dx || dw) && (act != NGPT_ACT_NONE || !on16(dout) || (dw && (M % 64 || N % 8)));
        copy_x = dw && (M % 64 || K % 8 || ldx % 8 || !on16(x_));
        // (rows of dw that are not whole groups of four are written without split tiles)
        lay_out(M, N, K, dx, dbias, dw && K % 4 == 0 ? balanced_part_bytes_here(own_dz ? (int)up64(N) : N, (int)up8(K), (int)(2 * up64(M))) : 0);
    }

private:
    void lay_out(int M, int N, int K, bool dx, bool dbias, int64_t part_bytes) {
        M64 = up64(M); N64 = up64(N); K8 = up8(K);
        dz = 0;
        w = dz + (own_dz ? align_up(M64 * N64 * 2, 256) : 0);
        x = w + (dx ? align_up(N64 * K * 2, 256) : 0);
        parts = x + (copy_x ? align_up(M64 * K8 * 2, 256) : 0);
        sums = parts + align_up(part_bytes, 256);
        sum_rows = act_grad_rows(M, N);
        total = sums + (dbias ? align_up((int64_t)sum_rows * N * 4, 256) : 0);
    }
};
}  // namespace
}  // namespace ngpt

extern "C" int64_t ngpt_linear_act_bwd_workspace_bytes(int M, int N, int K) {
    if (M <= 0 || N <= 0 || K <= 0 || M > (1 << 29) || N > kMaxStride || K > kMaxStride) return 0;
    return BwdPlan(M, N, K).total;
}

extern "C" int64_t ngpt_linear_act_bwd_workspace_bytes_for(const void* dout_bf16, const void* x_bf16, int64_t ldx, int M, int N, int K, int activation,
                                                           int want_dx, int want_dw, int want_dbias) {
    if (ngpt_linear_act_bwd_workspace_bytes(M, N, K) == 0) return 0;
    return BwdPlan(M, N, K, activation, dout_bf16, x_bf16, ldx, want_dx != 0, want_dw != 0, want_dbias != 0).total;
}

extern "C" int ngpt_linear_act_bwd(const void* dout_bf16, const void* pre_bf16, const void* x_bf16, int64_t ldx, const void* w_bf16, int64_t ldw,
                                   int M, int N, int K, int activation, void* dx_bf16, void* dw_bf16, void* dbias_bf16,
                                   void* workspace, int64_t workspace_bytes, void* stream) {
    const char* who = "ngpt_linear_act_bwd";
    if (!dout_bf16 || (activation != NGPT_ACT_NONE && !pre_bf16) || (dx_bf16 && !w_bf16) || (dw_bf16 && !x_bf16))
        return fail(NGPT_EINVAL, "%s: null pointer", who);
    if (int e = check_linear(who, M, N, K, activation)) return e;
    if ((dw_bf16 && ldx < K) || (dx_bf16 && ldw < K)) return fail(NGPT_EALIGN, "%s: row strides ldx=%lld ldw=%lld", who, (long long)ldx, (long long)ldw);
    if ((dw_bf16 && ldx > kMaxStride) || (dx_bf16 && ldw > kMaxStride))
        return fail(NGPT_ERANGE, "%s: row strides of at most 2^21 values (ldx=%lld ldw=%lld)", who, (long long)ldx, (long long)ldw);
    const BwdPlan p(M, N, K, activation, dout_bf16, x_bf16, ldx, dx_bf16 != nullptr, dw_bf16 != nullptr, dbias_bf16 != nullptr);
    if (p.total > 0 && (!workspace || workspace_bytes < p.total || !on16(workspace)))
        return fail(NGPT_EWORKSPACE, "%s: workspace %lld < %lld bytes", who, (long long)workspace_bytes, (long long)p.total);
    hipStream_t st = (hipStream_t)stream;
    uint8_t* ws = (uint8_t*)workspace;
    const bool own_dz = p.own_dz;
    const uint16_t* dz = own_dz ? (const uint16_t*)(ws + p.dz) : (const uint16_t*)dout_bf16;
    const int64_t ld_dz = own_dz ? p.N64 : N;
    if (own_dz || dbias_bf16) {
        const int rows_p = own_dz ? (int)p.M64 : M, cols_p = own_dz ? (int)p.N64 : (int)up8(N);
        float* part = dbias_bf16 ? (float*)(ws + p.sums) : nullptr;
        const dim3 grid((cols_p + kColsPerBlock - 1) / kColsPerBlock, p.sum_rows);
        auto go = [&](auto kind) {
            act_grad_kernel<decltype(kind)::value><<<grid, 256, 0, st>>>((const uint16_t*)dout_bf16, (const uint16_t*)pre_bf16, M, N,
                                                                         own_dz ? (uint16_t*)(ws + p.dz) : nullptr, rows_p, cols_p, part);
        };
        with_act(activation, go);
        if (int e = check_launch("act_grad_kernel")) return e;
        if (dbias_bf16) {
            col_sum_kernel<<<(N + 31) / 32, kColSumThreads, 0, st>>>(part, p.sum_rows, N, (uint16_t*)dbias_bf16);
            if (int e = check_launch("col_sum_kernel")) return e;
        }
    }
    GemmSlot slot(PROF_GEMM_BF16);
    if (dx_bf16) {
        // dx [M, K] = dz . w: as a forward product with w^T, one pass over w more, but both operands then have the contraction contiguous
        uint16_t* wt = (uint16_t*)(ws + p.w);
        if (int e = transpose_pad((const uint16_t*)w_bf16, ldw, N, K, wt, (int)p.N64, st)) return e;
        LinearOut o{(uint16_t*)dx_bf16, nullptr, nullptr, nullptr, 0, M, K, K % 8 == 0 && on16(dx_bf16), 0};
        // (dz's padding and w^T's are zeros)
        ProfileScope prof(PROF_GEMM_BF16, st);
        if (int e = linear_run(o, dz, ld_dz, wt, p.N64, own_dz ? (int)p.N64 : N, NGPT_ACT_NONE, st)) return e;
    }
    if (dw_bf16) {      // dw [N, K] = dz^T . x, contraction over the M rows of both
        const void* x = x_bf16;
        if (p.copy_x) {
            if (int e = pad_copy(x_bf16, ldx, M, K, ws + p.x, p.M64, p.K8, st)) return e;
            x = ws + p.x;
            ldx = p.K8;
        }
        if (int e = gemm_bf16_clipped(dz, FMT_BF16 | FMT_TRANSPOSED, 2 * ld_dz, x, FMT_BF16 | FMT_TRANSPOSED, 2 * ldx, (int)(own_dz ? p.N64 : N), (int)p.K8,
                                      (int)(2 * p.M64), N, K, dw_bf16, K, (float*)(ws + p.parts), st)) return e;
    }
    return NGPT_OK;
}
