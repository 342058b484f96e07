// out = residual + act(x . w^T + bias), its backward, and what both need around the matrix products.
//
//   z = x w^T + bias     x [M, K], w [N, K] bf16, bias [N], residual [M, N] optional
//   backward: dz = dout act'(z);  dx = dz w;  dw = dz^T x;  dbias = sum of dz over the rows;  dresidual = dout
// Products on the matrix pipe with fp32 accumulation; bias, activation and residual are applied to the fp32 sums, one rounding
// at the store.  Training keeps z in bf16 (the activation's slope is computed from it) and feeds dz to the matrix pipe in bf16.
#include "gemm_tn.h"
#include "host_util.h"
#include "launch.h"
#include <algorithm>

namespace ngpt {
// gemm_api.hip
int64_t balanced_part_bytes(int R, int C, int K);
int gemm_bf16_clipped(const void* A, int fa, int64_t lda, const void* B, int fb, int64_t ldb, int R, int C, int K, int R_out, int C_out,
                      void* out_bf16, int64_t ldc, float* part32, hipStream_t st);

namespace {

// ---------------------------------------------------------------------------------------------- activations
template <int ACT>
__device__ __forceinline__ float act_of(float z) {
    constexpr float kLog2e = 1.4426950408889634f;
    if constexpr (ACT == NGPT_ACT_RELU2) {
        const float r = fmaxf(z, 0.0f);
        return z != z ? z : r * r;
    } else if constexpr (ACT == NGPT_ACT_GELU) {
        return z * (0.5f + 0.5f * erff(z * 0.70710678118654752f));
    } else if constexpr (ACT == NGPT_ACT_GELU_TANH) {      // z (1 + tanh u) / 2 = z sigmoid(2 u)
        const float u = z * __builtin_fmaf(z * z, 0.7978845608028654f * 0.044715f, 0.7978845608028654f);
        return z * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-2.0f * kLog2e * u));
    } else if constexpr (ACT == NGPT_ACT_SILU) {
        return z * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-kLog2e * z));
    } else {
        return z;
    }
}
template <int ACT>
__device__ __forceinline__ float act_slope(float z) {
    constexpr float kLog2e = 1.4426950408889634f;
    if constexpr (ACT == NGPT_ACT_RELU2) {
        return z != z ? z : 2.0f * fmaxf(z, 0.0f);
    } else if constexpr (ACT == NGPT_ACT_GELU) {
        return 0.5f + 0.5f * erff(z * 0.70710678118654752f) + z * 0.3989422804014327f * __builtin_amdgcn_exp2f(-0.5f * kLog2e * z * z);
    } else if constexpr (ACT == NGPT_ACT_GELU_TANH) {
        const float u = z * __builtin_fmaf(z * z, 0.7978845608028654f * 0.044715f, 0.7978845608028654f);
        const float s = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-2.0f * kLog2e * u));
        return s + z * s * (1.0f - s) * 2.0f * __builtin_fmaf(z * z, 3.0f * 0.7978845608028654f * 0.044715f, 0.7978845608028654f);
    } else if constexpr (ACT == NGPT_ACT_SILU) {
        const float s = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-kLog2e * z));
        return s + z * s * (1.0f - s);
    } else {
        return 1.0f;
    }
}
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ float lo16(int w) { return __uint_as_float((uint32_t)w << 16); }
__device__ __forceinline__ float hi16(int w) { return __uint_as_float((uint32_t)w & 0xffff0000u); }

// 8 consecutive bf16 of a row, `n` of which exist; vec: one 16-byte access is allowed.  The value-by-value path is a loop on purpose: the
// compiler stops inlining into a kernel of many basic blocks, and the GEMM's state then lives in scratch memory.
__device__ __forceinline__ v4i load8(const uint16_t* p, int n, bool vec) {
    if (vec && n >= 8) return *(const v4i*)p;
    v4i w = {0, 0, 0, 0};
#pragma unroll 1
    for (int i = min(n, 8) - 1; i >= 0; --i) {
        w.w = (int)__builtin_amdgcn_alignbit((uint32_t)w.w, (uint32_t)w.z, 16);
        w.z = (int)__builtin_amdgcn_alignbit((uint32_t)w.z, (uint32_t)w.y, 16);
        w.y = (int)__builtin_amdgcn_alignbit((uint32_t)w.y, (uint32_t)w.x, 16);
        w.x = (int)(((uint32_t)w.x << 16) | (uint32_t)p[i]);
    }
    return w;
}
__device__ __forceinline__ void store8(uint16_t* p, v4i w, int n, bool vec) {
    if (vec && n >= 8) {
        *(v4i*)p = w;
        return;
    }
#pragma unroll 1
    for (int i = 0; i < min(n, 8); ++i) {
        p[i] = (uint16_t)w.x;
        w.x = (int)__builtin_amdgcn_alignbit((uint32_t)w.y, (uint32_t)w.x, 16);
        w.y = (int)__builtin_amdgcn_alignbit((uint32_t)w.z, (uint32_t)w.y, 16);
        w.z = (int)__builtin_amdgcn_alignbit((uint32_t)w.w, (uint32_t)w.z, 16);
        w.w = (int)((uint32_t)w.w >> 16);
    }
}

// ---------------------------------------------------------------------------------------------- epilogue of the tile GEMM
// The product runs transposed (tile rows = output features, A = w; tile columns = rows of x, B = x): a lane then owns one row of
// x and four consecutive features per accumulator register group.  Every 32-row x 64-feature block passes through the wave's 4 KiB
// of LDS, so that z, the residual and the output cross memory as whole 128-byte lines.  16-byte pieces are XOR-swizzled by
// the row; LDS operations of one wave execute in order, no waits are needed between the steps.
// Memory is reached through descriptors of the tile's rows, whose bounds check stands for the branches at the matrix' end: a kernel of
// many basic blocks is not inlined completely any more, and the GEMM's state then lives in scratch memory.  Rows that do not start on
// 16 bytes are moved value by value, in loops.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer_of(const void* base, int64_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, (int)(bytes < 0x7fffff00 ? bytes : 0x7fffff00), 0x00020000);
}
constexpr int kNowhere = 0x7ffffff0;      // an offset past any descriptor's end

// One kernel an activation: five of them behind a switch in one kernel cost it 60 spilled registers.
template <int WAVES, int ACT, bool PRE, bool RES>
struct EpiLinear {
    uint16_t* out;          // [C, R], row stride R
    uint16_t* pre;          // PRE: z, same shape
    const uint16_t* bias;   // nullable [R], on 16 bytes
    const uint16_t* res;    // RES: [C, R], row stride ld_res
    int64_t ld_res;
    int R, C;
    int vec, vec_res;       // rows of out and pre / of res start on 16 bytes and are whole 8-value pieces
    static constexpr int EXTRA_LDS = WAVES * 4096;
    static constexpr bool NEEDS_SCRATCH = false;
    static constexpr bool JOB_END_NEEDS_SCRATCH = false;
    static constexpr bool DROPS_FRAGMENTS = true;   // the residual's lines in flight next to the accumulators
    static constexpr int TILE_STORES = 8;           // at least: 4 per 32-row block and wave, 2 blocks or more (masked ones are issued too)
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

    // the wave's block of 32 rows x 64 features, `row0` / `col0` its origin in the matrix, value by value
    __device__ __forceinline__ void block_slow(const uint16_t* from, uint16_t* to, int64_t ld, int row0, int col0, int lane) {
#pragma unroll 1
        for (int i = 0; i < 32; ++i) {
            const int m = row0 + i, f = col0 + lane;
            uint16_t* at = (uint16_t*)(stage + i * 128 + (((lane >> 3) ^ (i & 7)) << 4) + (lane & 7) * 2);
            if (m < C && f < R) {
                if (to) to[(int64_t)m * ld + f] = *at;
                else *at = from[(int64_t)m * ld + f];
            }
        }
    }

    template <class Cfg>
    __device__ __forceinline__ void tile(v16f (&acc)[Cfg::TM][Cfg::TN], int r0, int c0, const AccCoords<Cfg>& co, uint8_t*, int lane) {
        static_assert(Cfg::TM == 2 && Cfg::TN >= 2 && Cfg::NWAVES == WAVES, "64-feature wave tiles, 4 KiB of staging each");
        const int h = lane >> 5, j = lane & 31;
        stored_all = vec != 0;
        const int rd_row = lane >> 3, rd_chunk = lane & 7;
        const int f = r0 + co.wave_row0 + rd_chunk * 8;          // this lane's 8 features in the line-wise steps
        const int rows = C - c0;                                 // rows of the matrix from this tile on
        const bool in = f < R;                                   // (R is a multiple of 8 where whole lines are moved)
        const auto buf_out = buffer_of(out + (int64_t)c0 * R, (int64_t)rows * R * 2);
        const auto buf_pre = buffer_of(PRE ? pre + (int64_t)c0 * R : out, PRE ? (int64_t)rows * R * 2 : 0);
        const auto buf_res = buffer_of(RES ? res + (int64_t)c0 * ld_res : out, RES ? ((int64_t)(rows - 1) * ld_res + R) * 2 : 0);
        const auto buf_bias = buffer_of(bias, bias ? ((int64_t)R * 2 + 3) & ~3ll : 0);
        const int off = in ? ((co.wave_col0 + rd_row) * R + f) * 2 : kNowhere;
        const int off_res = RES && in ? (int)(((co.wave_col0 + rd_row) * ld_res + f) * 2) : kNowhere;
        v2i b[8];                                                // bias of the lane's features, packed
#pragma unroll
        for (int i = 0; i < 8; ++i)
            b[i] = __builtin_bit_cast(v2i, __builtin_amdgcn_raw_buffer_load_b64(buf_bias, (r0 + co.wave_row0 + 8 * i + 4 * h) * 2, 0, 0));
        v4i line[4];
        auto load_block = [&](int tn) {
#pragma unroll
            for (int k = 0; k < 4; ++k)
                line[k] = __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(buf_res, in ? off_res + (int)((tn * 32 + 8 * k) * ld_res * 2) : kNowhere, 0, 0));
        };
        auto store_block = [&](int tn, __amdgpu_buffer_rsrc_t buf, uint16_t* to) {
            if (vec) {
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int row = 8 * k + rd_row;
                    const v4i v = *(const v4i*)(stage + row * 128 + ((rd_chunk ^ (row & 7)) << 4));
                    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, v), buf, in ? off + (tn * 32 + 8 * k) * R * 2 : kNowhere, 0, 0);
                }
            } else {
                block_slow(nullptr, to, R, c0 + co.wave_col0 + tn * 32, r0 + co.wave_row0, lane);
            }
        };
        if constexpr (RES) { if (vec_res) load_block(0); }
#pragma unroll
        for (int tn = 0; tn < Cfg::TN; ++tn) {
            const v16f* const a2[2] = {&acc[0][tn], &acc[1][tn]};
            auto z_of = [&](int tm, int g, float (&z)[4]) {
                const v16f& a = *a2[tm];
                const v2i bb = b[tm * 4 + g];
                z[0] = a[4 * g] + lo16(bb.x);
                z[1] = a[4 * g + 1] + hi16(bb.x);
                z[2] = a[4 * g + 2] + lo16(bb.y);
                z[3] = a[4 * g + 3] + hi16(bb.y);
            };
            auto place = [&](int tm, int g) { return stage + j * 128 + (((tm * 4 + g) ^ (j & 7)) << 4) + 8 * h; };
            if constexpr (PRE) {
#pragma unroll
                for (int tm = 0; tm < 2; ++tm)
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        float z[4];
                        z_of(tm, g, z);
                        *(v2i*)place(tm, g) = (v2i){(int)cvt_pk_bf16(z[0], z[1]), (int)cvt_pk_bf16(z[2], z[3])};
                    }
                store_block(tn, buf_pre, pre);
            }
            if constexpr (RES) {
                if (vec_res) {
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const int row = 8 * k + rd_row;
                        *(v4i*)(stage + row * 128 + ((rd_chunk ^ (row & 7)) << 4)) = line[k];
                    }
                    if (tn + 1 < Cfg::TN) load_block(tn + 1);       // in flight while this block is worked on
                } else {
                    block_slow(res, nullptr, ld_res, c0 + co.wave_col0 + tn * 32, r0 + co.wave_row0, lane);
                }
            }
#pragma unroll
            for (int tm = 0; tm < 2; ++tm)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    uint8_t* at = place(tm, g);
                    float z[4];
                    z_of(tm, g, z);
#pragma unroll
                    for (int i = 0; i < 4; ++i) z[i] = act_of<ACT>(z[i]);
                    if constexpr (RES) {
                        const v2i r = *(const v2i*)at;
                        z[0] += lo16(r.x);
                        z[1] += hi16(r.x);
                        z[2] += lo16(r.y);
                        z[3] += hi16(r.y);
                    }
                    *(v2i*)at = (v2i){(int)cvt_pk_bf16(z[0], z[1]), (int)cvt_pk_bf16(z[2], z[3])};
                    if (g & 1) __builtin_amdgcn_sched_barrier(0);   // few temporaries next to the accumulators
                }
            store_block(tn, buf_out, out);
            __builtin_amdgcn_sched_barrier(0);
        }
    }
};

// ---------------------------------------------------------------------------------------------- around the products
// dst [rows_p, cols_p] = src [rows, cols] with zeros around it; cols_p % 8 == 0.
__global__ __launch_bounds__(256) void pad_copy_kernel(const uint16_t* __restrict__ src, int64_t ld, int rows, int cols, uint16_t* __restrict__ dst,
                                                       int rows_p, int cols_p, int vec) {
    const int c8 = cols_p / 8;
    const int64_t n = (int64_t)rows_p * c8;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        const int r = (int)(i / c8), c = (int)(i - (int64_t)r * c8) * 8;
        v4i w = {0, 0, 0, 0};
        if (r < rows) w = load8(src + (int64_t)r * ld + c, cols - c, vec != 0);
        *(v4i*)(dst + i * 8) = w;
    }
}

// dz = dout act'(z) (zeros in the padding of its [rows_p, cols_p]) and the column sums of dz, in fp32 before dz is rounded: a workgroup
// covers 256 columns and every gridDim.y-th group of 8 rows, its sums go to part[blockIdx.y][N].  dz or part may be null.
constexpr int kColsPerBlock = 256, kRowLanes = 8;
template <int ACT>
__global__ __launch_bounds__(256) void act_grad_kernel(const uint16_t* __restrict__ dout, const uint16_t* __restrict__ pre, int M, int N,
                                                       uint16_t* __restrict__ dz, int rows_p, int cols_p, float* __restrict__ part, int vec) {
    __shared__ float red[kRowLanes][kColsPerBlock + 4];
    const int ct = threadIdx.x & 31, rt = threadIdx.x >> 5;
    const int c = blockIdx.x * kColsPerBlock + ct * 8;
    float sum[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (c < cols_p) {
        for (int r = blockIdx.y * kRowLanes + rt; r < rows_p; r += gridDim.y * kRowLanes) {
            v4i g = {0, 0, 0, 0}, o = {0, 0, 0, 0};
            if (r < M && c < N) {
                g = load8(dout + (int64_t)r * N + c, N - c, vec != 0);
                if constexpr (ACT == NGPT_ACT_NONE) {
                    o = g;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        sum[2 * i] += lo16(g[i]);
                        sum[2 * i + 1] += hi16(g[i]);
                    }
                } else {
                    const v4i z = load8(pre + (int64_t)r * N + c, N - c, vec != 0);
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
    pad_copy_kernel<<<grid, 256, 0, st>>>((const uint16_t*)src, ld, (int)rows, (int)cols, (uint16_t*)dst, (int)rows_p, (int)cols_p,
                                          on16(src) && ld % 8 == 0);
    return check_launch("pad_copy_kernel");
}

// Workgroups along the rows of act_grad_kernel, whatever the device
int act_grad_rows(int64_t M, int64_t N) {
    const int64_t cols = (N + kColsPerBlock - 1) / kColsPerBlock;
    int64_t rows = std::min<int64_t>((M + kRowLanes - 1) / kRowLanes, std::max<int64_t>(1, 2048 / cols));
    return (int)std::max<int64_t>(rows, 1);
}

// f(integral_constant) for the activation
template <class F>
auto with_act(int act, F&& f) {
    switch (act) {
        case NGPT_ACT_RELU2: return f(std::integral_constant<int, NGPT_ACT_RELU2>{});
        case NGPT_ACT_GELU: return f(std::integral_constant<int, NGPT_ACT_GELU>{});
        case NGPT_ACT_GELU_TANH: return f(std::integral_constant<int, NGPT_ACT_GELU_TANH>{});
        case NGPT_ACT_SILU: return f(std::integral_constant<int, NGPT_ACT_SILU>{});
        default: return f(std::integral_constant<int, NGPT_ACT_NONE>{});
    }
}

int check_linear(const char* who, int M, int N, int K, int act) {
    if (M <= 0 || N <= 0 || K <= 0) return fail(NGPT_EINVAL, "%s: empty problem M=%d N=%d K=%d", who, M, N, K);
    if (act < NGPT_ACT_NONE || act > NGPT_ACT_SILU) return fail(NGPT_EINVAL, "%s: activation=%d", who, act);
    if (N > (1 << 24) || K > (1 << 24)) return fail(NGPT_ERANGE, "%s: N=%d K=%d", who, N, K);
    return NGPT_OK;
}

// The tile GEMM reads rows that start on 16 bytes, a multiple of 64 values long: other operands are copied into the workspace first.
bool rows_fit(const void* p, int64_t ld, int K) { return K % 64 == 0 && on16(p) && ld % 8 == 0; }

}  // namespace
}  // namespace ngpt

using namespace ngpt;

extern "C" int64_t ngpt_linear_act_fwd_workspace_bytes(int M, int N, int K) {
    const int64_t Kp = up64(K);
    return K % 64 ? align_up(((int64_t)M + N) * Kp * 2, 256) : 0;
}

extern "C" int ngpt_linear_act_fwd(const void* x_bf16, int64_t ldx, const void* w_bf16, int64_t ldw, const void* bias_bf16,
                                   const void* residual_bf16, int64_t ld_residual, int M, int N, int K, int activation,
                                   void* out_bf16, void* pre_bf16, void* workspace, int64_t workspace_bytes, void* stream) {
    const char* who = "ngpt_linear_act_fwd";
    if (!x_bf16 || !w_bf16 || !out_bf16) return fail(NGPT_EINVAL, "%s: null pointer", who);
    if (int e = check_linear(who, M, N, K, activation)) return e;
    if (pre_bf16 && activation == NGPT_ACT_NONE) return fail(NGPT_EINVAL, "%s: pre is for activations", who);
    if (!on16(bias_bf16)) return fail(NGPT_EALIGN, "%s: the bias starts on 16 bytes", who);
    if (ldx < K || ldw < K || (residual_bf16 && ld_residual < N))
        return fail(NGPT_EALIGN, "%s: row strides ldx=%lld ldw=%lld ld_residual=%lld", who, (long long)ldx, (long long)ldw, (long long)ld_residual);
    hipStream_t st = (hipStream_t)stream;
    const int64_t Kp = up64(K);
    if (K % 64 == 0 && !(rows_fit(x_bf16, ldx, K) && rows_fit(w_bf16, ldw, K)))
        return fail(NGPT_EALIGN, "%s: rows of x and w start on 16 bytes where K %% 64 == 0 (ldx=%lld ldw=%lld)", who, (long long)ldx, (long long)ldw);
    if (K % 64) {
        if (!workspace || workspace_bytes < ngpt_linear_act_fwd_workspace_bytes(M, N, K) || !on16(workspace))
            return fail(NGPT_EWORKSPACE, "%s: workspace %lld < %lld bytes", who, (long long)workspace_bytes,
                        (long long)ngpt_linear_act_fwd_workspace_bytes(M, N, K));
        uint16_t* xp = (uint16_t*)workspace;
        uint16_t* wp = xp + (int64_t)M * Kp;
        if (int e = pad_copy(x_bf16, ldx, M, K, xp, M, Kp, st)) return e;
        if (int e = pad_copy(w_bf16, ldw, N, K, wp, N, Kp, st)) return e;
        x_bf16 = xp; w_bf16 = wp;
        ldx = ldw = Kp;
    }
    ProfileScope prof(PROF_GEMM_BF16, st);
    GemmOperands g{(const uint8_t*)w_bf16, (const uint8_t*)x_bf16, 2 * ldw, 2 * ldx, N, M, (int)(2 * Kp), 1};
    auto go = [&](auto epi) {
        using Epi = decltype(epi);
        epi.out = (uint16_t*)out_bf16;
        epi.pre = (uint16_t*)pre_bf16;
        epi.bias = (const uint16_t*)bias_bf16;
        epi.res = (const uint16_t*)residual_bf16;
        epi.ld_res = ld_residual;
        epi.R = N;
        epi.C = M;
        epi.vec = N % 8 == 0 && on16(out_bf16) && on16(pre_bf16);
        epi.vec_res = residual_bf16 && N % 8 == 0 && ld_residual % 8 == 0 && on16(residual_bf16);
        using Cfg = std::conditional_t<Epi::EXTRA_LDS == 8 * 4096, MainCfg, SmallCfg>;
        return launch_gemm_fmt<Cfg, FMT_BF16, FMT_BF16>(g, epi, st, 0);
    };
    const int64_t tiles = ((int64_t)(N + 255) / 256) * ((M + 255) / 256);
    auto pick = [&](auto waves, auto kind) {
        constexpr int W = decltype(waves)::value, A = decltype(kind)::value;
        if constexpr (A != NGPT_ACT_NONE) {
            if (pre_bf16) return residual_bf16 ? go(EpiLinear<W, A, true, true>{}) : go(EpiLinear<W, A, true, false>{});
        }
        return residual_bf16 ? go(EpiLinear<W, A, false, true>{}) : go(EpiLinear<W, A, false, false>{});
    };
    return with_act(activation, [&](auto kind) {
        return 2 * tiles > num_cus() ? pick(std::integral_constant<int, 8>{}, kind) : pick(std::integral_constant<int, 4>{}, kind);
    });
}

namespace ngpt {
namespace {
// Workspace of the backward: dz [M64, N64] | w [N64, K8] | x [M64, K8] (copies of what the products cannot read in place) | parts of split
// tiles | column sums
struct BwdPlan {
    int64_t M64, N64, K8, dz, w, x, parts, sums, total;
    int sum_rows;
    BwdPlan(int M, int N, int K) {
        M64 = up64(M); N64 = up64(N); K8 = up8(K);
        dz = 0;
        w = dz + align_up(M64 * N64 * 2, 256);
        x = w + align_up(N64 * K8 * 2, 256);
        parts = x + align_up(M64 * K8 * 2, 256);
        sums = parts + align_up(std::max(balanced_part_bytes(M, (int)K8, (int)(2 * N64)), balanced_part_bytes((int)N64, (int)K8, (int)(2 * M64))), 256);
        sum_rows = act_grad_rows(M, N);
        total = sums + align_up((int64_t)sum_rows * N * 4, 256);
    }
};
}  // namespace
}  // namespace ngpt

extern "C" int64_t ngpt_linear_act_bwd_workspace_bytes(int M, int N, int K) {
    if (M <= 0 || N <= 0 || K <= 0) return 0;
    return BwdPlan(M, N, K).total;
}

extern "C" int ngpt_linear_act_bwd(const void* dout_bf16, const void* pre_bf16, const void* x_bf16, int64_t ldx, const void* w_bf16, int64_t ldw,
                                   int M, int N, int K, int activation, void* dx_bf16, void* dw_bf16, void* dbias_bf16,
                                   void* workspace, int64_t workspace_bytes, void* stream) {
    const char* who = "ngpt_linear_act_bwd";
    if (!dout_bf16 || (activation != NGPT_ACT_NONE && !pre_bf16) || (dx_bf16 && !w_bf16) || (dw_bf16 && !x_bf16))
        return fail(NGPT_EINVAL, "%s: null pointer", who);
    if (int e = check_linear(who, M, N, K, activation)) return e;
    if ((dw_bf16 && ldx < K) || (dx_bf16 && ldw < K)) return fail(NGPT_EALIGN, "%s: row strides ldx=%lld ldw=%lld", who, (long long)ldx, (long long)ldw);
    const BwdPlan p(M, N, K);
    if (!workspace || workspace_bytes < p.total || !on16(workspace))
        return fail(NGPT_EWORKSPACE, "%s: workspace %lld < %lld bytes", who, (long long)workspace_bytes, (long long)p.total);
    hipStream_t st = (hipStream_t)stream;
    uint8_t* ws = (uint8_t*)workspace;
    const bool need_gemm = dx_bf16 || dw_bf16;
    // dz is dout itself where there is no activation and the products can read it in place
    const bool own_dz = need_gemm && !(activation == NGPT_ACT_NONE && M % 64 == 0 && N % 64 == 0 && on16(dout_bf16));
    const uint16_t* dz = own_dz ? (const uint16_t*)(ws + p.dz) : (const uint16_t*)dout_bf16;
    if (own_dz || dbias_bf16) {
        const int vec = N % 8 == 0 && on16(dout_bf16) && on16(pre_bf16);
        const int rows_p = own_dz ? (int)p.M64 : M, cols_p = own_dz ? (int)p.N64 : (int)up8(N);
        float* part = dbias_bf16 ? (float*)(ws + p.sums) : nullptr;
        const dim3 grid((cols_p + kColsPerBlock - 1) / kColsPerBlock, p.sum_rows);
        auto go = [&](auto kind) {
            act_grad_kernel<decltype(kind)::value><<<grid, 256, 0, st>>>((const uint16_t*)dout_bf16, (const uint16_t*)pre_bf16, M, N,
                                                                         own_dz ? (uint16_t*)(ws + p.dz) : nullptr, rows_p, cols_p, part, vec);
        };
        with_act(activation, go);
        if (int e = check_launch("act_grad_kernel")) return e;
        if (dbias_bf16) {
            col_sum_kernel<<<(N + 31) / 32, kColSumThreads, 0, st>>>(part, p.sum_rows, N, (uint16_t*)dbias_bf16);
            if (int e = check_launch("col_sum_kernel")) return e;
        }
    }
    GemmSlot slot(PROF_GEMM_BF16);
    float* parts = (float*)(ws + p.parts);
    if (dx_bf16) {      // dx [M, K] = dz . w, contraction over the N rows of w
        const void* w = w_bf16;
        if (N % 64 || K % 8 || ldw % 8 || !on16(w)) {
            if (int e = pad_copy(w_bf16, ldw, N, K, ws + p.w, p.N64, p.K8, st)) return e;
            w = ws + p.w;
            ldw = p.K8;
        }
        if (int e = gemm_bf16_clipped(dz, FMT_BF16, 2 * p.N64, w, FMT_BF16 | FMT_TRANSPOSED, 2 * ldw, M, (int)p.K8, (int)(2 * p.N64), M, K, dx_bf16, K,
                                      parts, st)) return e;
    }
    if (dw_bf16) {      // dw [N, K] = dz^T . x, contraction over the M rows of both
        const void* x = x_bf16;
        if (M % 64 || K % 8 || ldx % 8 || !on16(x)) {
            if (int e = pad_copy(x_bf16, ldx, M, K, ws + p.x, p.M64, p.K8, st)) return e;
            x = ws + p.x;
            ldx = p.K8;
        }
        if (int e = gemm_bf16_clipped(dz, FMT_BF16 | FMT_TRANSPOSED, 2 * p.N64, x, FMT_BF16 | FMT_TRANSPOSED, 2 * ldx, (int)p.N64, (int)p.K8,
                                      (int)(2 * p.M64), N, K, dw_bf16, K, parts, st)) return e;
    }
    return NGPT_OK;
}
