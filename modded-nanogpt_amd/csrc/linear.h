// Activations and the epilogue of linear_act, shared by its kernels; the launchers behind ngpt_linear_act_fwd.
#pragma once
#include "common.h"
#include "host_util.h"
#include <type_traits>

namespace ngpt {

// ---------------------------------------------------------------------------------------------- activations
// The normal distribution function, and exp(-z^2 / 2) on the way: Abramowitz & Stegun 7.1.26, erfc(x) = t (a1 + t (a2 + ...)) exp(-x^2) with
// t = 1 / (1 + 0.3275911 x), to 1.5e-7 for x >= 0 (the library's erf takes three times as long).
__device__ __forceinline__ float normal_cdf(float z, float& gauss) {
    gauss = __builtin_amdgcn_exp2f(-0.5f * 1.4426950408889634f * z * z);
    const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(fabsf(z), 0.3275911f * 0.70710678118654752f, 1.0f));
    float p = __builtin_fmaf(t, 0.5f * 1.061405429f, 0.5f * -1.453152027f);
    p = __builtin_fmaf(t, p, 0.5f * 1.421413741f);
    p = __builtin_fmaf(t, p, 0.5f * -0.284496736f);
    p = __builtin_fmaf(t, p, 0.5f * 0.254829592f);
    const float tail = p * t * gauss;
    return z < 0.0f ? tail : 1.0f - tail;
}
template <int ACT>
__device__ __forceinline__ float act_of(float z) {
    constexpr float kLog2e = 1.4426950408889634f;
    if constexpr (ACT == NGPT_ACT_RELU2) {
        const float r = __builtin_elementwise_maximum(z, 0.0f);      // (keeps a NaN, in one instruction)
        return r * r;
    } else if constexpr (ACT == NGPT_ACT_GELU) {
        float gauss;
        return z * normal_cdf(z, gauss);
    } else if constexpr (ACT == NGPT_ACT_GELU_TANH) {      // z (1 + tanh u) / 2 = z sigmoid(2 u)
        constexpr float c = -2.0f * kLog2e * 0.7978845608028654f;
        return z * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z * __builtin_fmaf(z * z, c * 0.044715f, c)));
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
        return 2.0f * __builtin_elementwise_maximum(z, 0.0f);
    } else if constexpr (ACT == NGPT_ACT_GELU) {
        float gauss;
        const float cdf = normal_cdf(z, gauss);
        return __builtin_fmaf(z * 0.3989422804014327f, gauss, cdf);
    } else if constexpr (ACT == NGPT_ACT_GELU_TANH) {
        const float zz = fminf(z * z, 1e12f);      // (s is 0 or 1 long before; an infinite z^2 times s (1 - s) = 0 would be NaN.  z keeps a NaN)
        const float u = z * __builtin_fmaf(zz, 0.7978845608028654f * 0.044715f, 0.7978845608028654f);
        const float s = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-2.0f * kLog2e * u));
        return s + z * s * (1.0f - s) * 2.0f * __builtin_fmaf(zz, 3.0f * 0.7978845608028654f * 0.044715f, 0.7978845608028654f);
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

// Values i .. i + 7 of a row of `len` (zeros behind its end; 0 <= i), 16 bytes at any address: gfx950 takes unaligned global accesses.
// Of a row of 8 values and more, without a branch: the piece is loaded so that it ends with the row at the latest, and shifted down.
__device__ __forceinline__ v4i load_row8_end(const uint16_t* row, int i, int len) {
    const int at = min(i, len - 8), s = i - at;
    v4i w;
    __builtin_memcpy(&w, row + at, 16);
    if (s & 4) w = (v4i){w.z, w.w, 0, 0};
    if (s & 2) w = (v4i){w.y, w.z, w.w, 0};
    if (s & 1)
        w = (v4i){(int)__builtin_amdgcn_alignbit((uint32_t)w.y, (uint32_t)w.x, 16), (int)__builtin_amdgcn_alignbit((uint32_t)w.z, (uint32_t)w.y, 16),
                  (int)__builtin_amdgcn_alignbit((uint32_t)w.w, (uint32_t)w.z, 16), (int)((uint32_t)w.w >> 16)};
    if (s >= 8) w = (v4i){0, 0, 0, 0};
    return w;
}
// of a row of any length, value by value
__device__ __forceinline__ v4i load_row8_short(const uint16_t* row, int i, int len) {
    v4i w = {0, 0, 0, 0};
#pragma unroll 1
    for (int e = min(len - i, 8) - 1; e >= 0; --e) {
        w.w = (int)__builtin_amdgcn_alignbit((uint32_t)w.w, (uint32_t)w.z, 16);
        w.z = (int)__builtin_amdgcn_alignbit((uint32_t)w.z, (uint32_t)w.y, 16);
        w.y = (int)__builtin_amdgcn_alignbit((uint32_t)w.y, (uint32_t)w.x, 16);
        w.x = (int)(((uint32_t)w.x << 16) | (uint32_t)row[i + e]);
    }
    return w;
}
__device__ __forceinline__ v4i load_row8(const uint16_t* row, int i, int len) {
    v4i w = {0, 0, 0, 0};
    if (i + 8 <= len) {
        __builtin_memcpy(&w, row + i, 16);
        return w;
    }
    if (i >= len) return w;
    if (len >= 8) return load_row8_end(row, i, len);
    return load_row8_short(row, i, len);
}
// The first `n` > 0 of 8 values (a loop on purpose: the compiler stops inlining into a kernel of many basic blocks, and a GEMM's state then
// lives in scratch memory).
__device__ __forceinline__ void store_any(uint16_t* p, v4i w, int n) {
    if (n >= 8) {
        __builtin_memcpy(p, &w, 16);
        return;
    }
#pragma unroll 1
    for (int i = 0; i < n; ++i) {
        p[i] = (uint16_t)w.x;
        w.x = (int)__builtin_amdgcn_alignbit((uint32_t)w.y, (uint32_t)w.x, 16);
        w.y = (int)__builtin_amdgcn_alignbit((uint32_t)w.z, (uint32_t)w.y, 16);
        w.z = (int)__builtin_amdgcn_alignbit((uint32_t)w.w, (uint32_t)w.z, 16);
        w.w = (int)((uint32_t)w.w >> 16);
    }
}

// f(integral_constant) for the activation, on the host
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

// ---------------------------------------------------------------------------------------------- epilogue of a wave's tile
// The products run transposed (tile rows = output features, A = w; tile columns = rows of x, B = x): a lane then owns one row of
// x and four consecutive features per accumulator register group.  Every block of 32 rows x 32 TM features passes through the wave's
// 2 TM KiB of LDS, so that z, the residual and the output cross memory as whole lines.  16-byte pieces are XOR-swizzled by
// the row; LDS operations of one wave execute in order, no waits are needed between the steps.
// Memory is reached through descriptors of the wave's rows, whose bounds check stands for the branches at the matrix' end: a kernel of
// many basic blocks is not inlined completely any more, and a GEMM's state then lives in scratch memory.  Rows that do not start on
// 16 bytes go without descriptors, in a loop.
struct LinearOut {
    uint16_t* out;          // [M, N], row stride N
    uint16_t* pre;          // nullable; z, same shape
    const uint16_t* bias;   // nullable [N], on 16 bytes
    const uint16_t* res;    // nullable [M, N], row stride ld_res
    int64_t ld_res;
    int M, N;
    int vec, vec_res;       // rows of out and pre / of res start on 16 bytes and are whole 8-value pieces
};

__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer_of(const void* base, int64_t bytes) {
    bytes = bytes < 0 ? 0 : (bytes < 0x7fffff00 ? bytes : 0x7fffff00);
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, (int)bytes, 0x00020000);
}
constexpr int kNowhere = 0x7ffffff0;      // an offset past any descriptor's end

template <int ACT, bool PRE, bool RES, int TM, int TN>
__device__ __forceinline__ void linear_epilogue(const LinearOut& o, v16f (&acc)[TM][TN], uint8_t* stage, int f0, int m0, int lane) {
    constexpr int CPR = 4 * TM;                   // 16-byte pieces of a block's row
    constexpr int RPI = 64 / CPR;                 // rows that one instruction of the wave moves
    constexpr int NI = 32 / RPI;
    const int h = lane >> 5, j = lane & 31;
    const int rd_row = lane / CPR, rd_chunk = lane % CPR;
    const int N = o.N, rows = o.M - m0;           // rows of the matrix from this tile on
    const int f = f0 + rd_chunk * 8;              // this lane's 8 features in the line-wise steps
    const bool in = f < N;                        // (N is a multiple of 8 where whole lines are moved)
    auto swz = [](int row, int chunk) { return row * (CPR * 16) + ((chunk ^ (TM == 2 ? row & 7 : (row >> 1) & 3)) << 4); };
    const auto buf_out = buffer_of(o.out + (int64_t)m0 * N, (int64_t)rows * N * 2);
    const auto buf_pre = buffer_of(PRE ? o.pre + (int64_t)m0 * N : o.out, PRE ? (int64_t)rows * N * 2 : 0);
    const auto buf_res = buffer_of(RES ? o.res + (int64_t)m0 * o.ld_res : o.out, RES && rows > 0 ? ((int64_t)(rows - 1) * o.ld_res + N) * 2 : 0);
    const auto buf_bias = buffer_of(o.bias, o.bias ? ((int64_t)N * 2 + 3) & ~3ll : 0);
    const int off = in ? (rd_row * N + f) * 2 : kNowhere, off_res = RES && in ? (rd_row * (int)o.ld_res + f) * 2 : kNowhere;
    v2i b[4 * TM];                                // bias of the lane's features, packed
#pragma unroll
    for (int i = 0; i < 4 * TM; ++i) b[i] = __builtin_bit_cast(v2i, __builtin_amdgcn_raw_buffer_load_b64(buf_bias, (f0 + 8 * i + 4 * h) * 2, 0, 0));
    v4i line[NI];
    auto load_block = [&](int tn) {
#pragma unroll
        for (int k = 0; k < NI; ++k)
            line[k] = __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(
                buf_res, in ? off_res + (tn * 32 + RPI * k) * (int)o.ld_res * 2 : kNowhere, 0, 0));
    };
    // a block between memory and the staging area where rows start anywhere: 16 bytes at any byte address, the row's last values one by one
    auto block_slow = [&](int tn, const uint16_t* from, uint16_t* to, int64_t ld) {
        const int left = N - f;
#pragma unroll 1
        for (int k = 0; k < NI; ++k) {
            const int row = RPI * k + rd_row, m = m0 + tn * 32 + row;
            uint8_t* at = stage + swz(row, rd_chunk);
            if (m < o.M && left > 0) {
                if (to) store_any(to + (int64_t)m * ld + f, *(const v4i*)at, left);
                else *(v4i*)at = load_row8(from + (int64_t)m * ld, f, N);
            }
        }
    };
    // All pieces at once where the block's rows and the lane's 8 values all exist (not in the large tiles' kernel: see the number of blocks above)
    auto whole_block = [&](int tn) { return TN <= 2 && m0 + tn * 32 + 32 <= o.M && f + 8 <= N; };
    auto store_block = [&](int tn, __amdgpu_buffer_rsrc_t buf, uint16_t* to) {
        if (o.vec) {
#pragma unroll
            for (int k = 0; k < NI; ++k) {
                const int row = RPI * k + rd_row;
                const v4i v = *(const v4i*)(stage + swz(row, rd_chunk));
                __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, v), buf, in ? off + (tn * 32 + RPI * k) * N * 2 : kNowhere, 0, 2);
            }
        } else if (whole_block(tn)) {
            uint16_t* const at = to + (int64_t)(m0 + tn * 32 + rd_row) * N + f;
            v4i v[NI];
#pragma unroll
            for (int k = 0; k < NI; ++k) v[k] = *(const v4i*)(stage + swz(RPI * k + rd_row, rd_chunk));
#pragma unroll
            for (int k = 0; k < NI; ++k) __builtin_memcpy(at + (int64_t)(RPI * k) * N, &v[k], 16);
        } else {
            block_slow(tn, nullptr, to, N);
        }
    };
    if constexpr (RES) { if (o.vec_res) load_block(0); }
#pragma unroll
    for (int tn = 0; tn < TN; ++tn) {
        auto z_of = [&](int tm, int g, float (&z)[4]) {
            const v16f& a = acc[tm][tn];
            const v2i bb = b[tm * 4 + g];
            z[0] = a[4 * g] + lo16(bb.x);
            z[1] = a[4 * g + 1] + hi16(bb.x);
            z[2] = a[4 * g + 2] + lo16(bb.y);
            z[3] = a[4 * g + 3] + hi16(bb.y);
        };
        auto place = [&](int tm, int g) { return stage + swz(j, tm * 4 + g) + 8 * h; };
        if constexpr (PRE) {
#pragma unroll
            for (int tm = 0; tm < TM; ++tm)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    float z[4];
                    z_of(tm, g, z);
                    *(v2i*)place(tm, g) = (v2i){(int)cvt_pk_bf16(z[0], z[1]), (int)cvt_pk_bf16(z[2], z[3])};
                }
            store_block(tn, buf_pre, o.pre);
        }
        if constexpr (RES) {
            if (o.vec_res) {
#pragma unroll
                for (int k = 0; k < NI; ++k) *(v4i*)(stage + swz(RPI * k + rd_row, rd_chunk)) = line[k];
                if (tn + 1 < TN) load_block(tn + 1);       // in flight while this block is worked on
            } else if (whole_block(tn)) {
                const uint16_t* const at = o.res + (int64_t)(m0 + tn * 32 + rd_row) * o.ld_res + f;
                v4i v[NI];
#pragma unroll
                for (int k = 0; k < NI; ++k) __builtin_memcpy(&v[k], at + (int64_t)(RPI * k) * o.ld_res, 16);
#pragma unroll
                for (int k = 0; k < NI; ++k) *(v4i*)(stage + swz(RPI * k + rd_row, rd_chunk)) = v[k];
            } else {
                block_slow(tn, o.res, nullptr, o.ld_res);
            }
        }
#pragma unroll
        for (int tm = 0; tm < TM; ++tm)
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
        store_block(tn, buf_out, o.out);
        __builtin_amdgcn_sched_barrier(0);
    }
}

// linear_small.hip: any alignment, any K.  The few-row kernel takes M <= kFewRows.
constexpr int kFewRows = 32;
int linear_few(const LinearOut& o, const uint16_t* x, int64_t ldx, const uint16_t* w, int64_t ldw, int K, int act, hipStream_t st);
int linear_mid(const LinearOut& o, const uint16_t* x, int64_t ldx, const uint16_t* w, int64_t ldw, int K, int act, hipStream_t st);

}  // namespace ngpt
