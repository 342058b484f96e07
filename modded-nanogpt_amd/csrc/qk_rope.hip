// Per-head rms norm of queries and keys with the position rotation in the same pass, forward and backward.
//
//   y = rot(x * rsqrt(mean(x^2) + eps) * w)         x one head of one token, D values; w [D] optional
//   rot: the first R of the D values are R / 2 pairs (a, b); (a, b) -> (a cos - b sin, b cos + a sin) with the pair's angle
//        at the token's position.  Pairs are (i, i + R / 2), or (2 i, 2 i + 1) when interleaved; values from R on stay.
//   backward: g = rot by the opposite angle of dy;  dw = sum over rows of g * xn;  g *= w;
//        dx = r * (g - xn * mean(g * xn))   with r = rsqrt(mean(x^2) + eps), xn = x * r, both recomputed from x
//
// All arithmetic is fp32 with one rounding at the store.  A row is a few hundred bytes, so everything between the
// load and the store happens in registers: memory traffic is the only cost that counts.
//
// Layout of the work: a row belongs to LPR lanes of 8 consecutive values each (D <= 8 LPR), a wave holds 64 / LPR rows,
// which are consecutive heads of ONE token: their loads are one contiguous piece and they share the cos / sin values,
// which stay in registers while the wave walks the token's heads.  U steps of loads are issued before the first is used.
#include "common.h"
#include "host_util.h"

namespace ngpt {
namespace {

struct RopeArgs {
    const void *q, *k;             // [B, T, H, D] with strides below (elements), last dimension contiguous
    int64_t q_sb, q_st, q_sh, k_sb, k_st, k_sh;
    const void *dq, *dk;           // backward: gradients of the outputs, strided likewise
    int64_t dq_sb, dq_st, dq_sh, dk_sb, dk_st, dk_sh;
    void *q_out, *k_out;           // forward: rotated heads; backward: gradients of q, k.  Contiguous [B, T, H, D]
    const void *cos, *sin;         // [P, R / 2]
    const void* pos;               // nullable; [B, T] int32 or int64 with strides
    int64_t p_sb, p_st;
    const void *qw, *kw;           // nullable [D]
    float* dw_part;                // backward with weights: [blocks][2][D] fp32
    int B, T, Hq, Hk, D, R, P;
    int pos64, tab_bf16, interleaved;
    float eps;
    int chunks;                    // head chunks per token
    int64_t items;                 // B * T * chunks
};

constexpr int kRopeThreads = 256;

template <class T> __device__ __forceinline__ float load1(const T* p);
template <> __device__ __forceinline__ float load1<uint16_t>(const uint16_t* p) { return bf16_bits_to_f32(*p); }
template <> __device__ __forceinline__ float load1<float>(const float* p) { return *p; }

__device__ __forceinline__ void unpack8(v4i w, float (&x)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        x[2 * i] = __uint_as_float((uint32_t)w[i] << 16);
        x[2 * i + 1] = __uint_as_float((uint32_t)w[i] & 0xffff0000u);
    }
}

// The 8 values of a lane as they come from memory: kept packed until they are used, so that several rows fit in flight.
template <class T, bool AL> struct Raw8;
template <> struct Raw8<uint16_t, true> {
    v4i w;
    __device__ void load(const uint16_t* p, int n) { w = n > 0 ? *(const v4i*)p : (v4i){0, 0, 0, 0}; }
    __device__ void get(float (&x)[8]) const { unpack8(w, x); }
};
template <> struct Raw8<float, true> {
    v4f a, b;
    __device__ void load(const float* p, int n) {
        a = n > 0 ? *(const v4f*)p : (v4f){0, 0, 0, 0};
        b = n > 0 ? *(const v4f*)(p + 4) : (v4f){0, 0, 0, 0};
    }
    __device__ void get(float (&x)[8]) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) { x[i] = a[i]; x[4 + i] = b[i]; }
    }
};
template <class T> struct Raw8<T, false> {      // any alignment, any D: value by value, `n` of them exist
    float v[8];
    __device__ void load(const T* p, int n) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < n ? load1<T>(p + i) : 0.0f;
    }
    __device__ void get(float (&x)[8]) const {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = v[i];
    }
};

template <class T, bool AL>
__device__ __forceinline__ void store8(T* p, const float (&x)[8], int n) {
    if constexpr (AL) {
        if (n <= 0) return;
        if constexpr (sizeof(T) == 2) {
            *(v4i*)p = (v4i){(int)cvt_pk_bf16(x[0], x[1]), (int)cvt_pk_bf16(x[2], x[3]), (int)cvt_pk_bf16(x[4], x[5]), (int)cvt_pk_bf16(x[6], x[7])};
        } else {
            *(v4f*)p = (v4f){x[0], x[1], x[2], x[3]};
            *(v4f*)(p + 4) = (v4f){x[4], x[5], x[6], x[7]};
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n) {
                if constexpr (sizeof(T) == 2) p[i] = (uint16_t)cvt_pk_bf16(x[i], x[i]);
                else p[i] = x[i];
            }
    }
}

// Sum over the LPR lanes of a row; every lane gets it.
template <int LPR>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
    for (int o = LPR / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

// Partner of each of the lane's values in its rotated pair (anything for values that are not rotated).
// AL: R / 2 (pairs of halves) is a multiple of 8, so the partners are the 8 values of one other lane.  Otherwise the
// row goes through the wave's own LDS block; LDS operations of one wave execute in order.
template <int LPR, bool AL>
__device__ __forceinline__ void partners(const float (&x)[8], float (&y)[8], int sub, int lane, int R, int interleaved, float* lds) {
    if (AL && interleaved) {
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = x[i ^ 1];
        return;
    }
    if (AL) {
        const int half = R >> 4;                      // lanes per half
        const int src = sub < half ? lane + half : (sub < 2 * half ? lane - half : lane);
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = __shfl(x[i], src, 64);
        return;
    }
    float* row = lds + (lane - sub) * 8;
#pragma unroll
    for (int i = 0; i < 8; ++i) row[sub * 8 + i] = x[i];
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int e = sub * 8 + i;
        const int p = e >= R ? e : (interleaved ? (e ^ 1) : (e < R / 2 ? e + R / 2 : e - R / 2));
        y[i] = row[p];
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
}

template <class T, int LPR, bool AL, bool BWD, int U>
__global__ __launch_bounds__(kRopeThreads) void qk_rope_kernel(RopeArgs a) {
    constexpr int ROWS = 64 / LPR;                    // rows (heads) of a wave
    constexpr int WAVES = kRopeThreads / 64;
    __shared__ float exch[AL && !BWD ? 1 : WAVES * 512];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int sub = lane & (LPR - 1), row_in_wave = lane / LPR;
    const int e0 = sub * 8;
    const int n = a.D - e0;                           // values of this lane that exist (<= 0: none)
    const int H = a.Hq + a.Hk;
    const float inv_d = 1.0f / (float)a.D;
    float* const lds = exch + (AL && !BWD ? 0 : wave * 512);

    float wq[8], wk[8], dwq[8], dwk[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const bool have = i < n;
        wq[i] = a.qw && have ? load1<T>((const T*)a.qw + e0 + i) : 1.0f;
        wk[i] = a.kw && have ? load1<T>((const T*)a.kw + e0 + i) : 1.0f;
        dwq[i] = dwk[i] = 0.0f;
    }

    for (int64_t item = (int64_t)blockIdx.x * WAVES + wave; item < a.items; item += (int64_t)gridDim.x * WAVES) {
        const int64_t token = item / a.chunks;
        const int chunk = (int)(item - token * a.chunks);
        const int b = (int)(token / a.T), t = (int)(token - (int64_t)b * a.T);
        const int h_end = min(H, (chunk + 1) * ROWS * U);

        // all rows of this chunk are requested first
        Raw8<T, AL> rx[U], rg[BWD ? U : 1];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int h = (chunk * U + u) * ROWS + row_in_wave;
            const bool live = h < h_end;
            const bool is_q = h < a.Hq;
            const T* p = is_q ? (const T*)a.q + (b * a.q_sb + t * a.q_st + h * a.q_sh)
                              : (const T*)a.k + (b * a.k_sb + t * a.k_st + (h - a.Hq) * a.k_sh);
            rx[u].load(p + e0, live ? n : 0);
            if constexpr (BWD) {
                const T* g = is_q ? (const T*)a.dq + (b * a.dq_sb + t * a.dq_st + h * a.dq_sh)
                                  : (const T*)a.dk + (b * a.dk_sb + t * a.dk_st + (h - a.Hq) * a.dk_sh);
                rg[u].load(g + e0, live ? n : 0);
            }
        }
        // cos / sin of the lane's values; sn carries the sign of the partner's term.  A position outside the table reads
        // nothing and makes the token's heads NaN.
        float cs[8], sn[8];
        {
            int64_t pos = t;
            if (a.pos) pos = a.pos64 ? ((const int64_t*)a.pos)[b * a.p_sb + t * a.p_st] : (int64_t)((const int32_t*)a.pos)[b * a.p_sb + t * a.p_st];
            const bool ok = pos >= 0 && pos < a.P;
            const int half = a.R / 2;
            const int64_t base = (ok ? pos : 0) * half;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int e = e0 + i;
                float c = 1.0f, s = 0.0f;
                if (e < a.R) {
                    const int idx = a.interleaved ? e >> 1 : (e < half ? e : e - half);
                    c = a.tab_bf16 ? load1<uint16_t>((const uint16_t*)a.cos + base + idx) : ((const float*)a.cos)[base + idx];
                    s = a.tab_bf16 ? load1<uint16_t>((const uint16_t*)a.sin + base + idx) : ((const float*)a.sin)[base + idx];
                    const bool first = a.interleaved ? !(e & 1) : e < half;
                    if (first != BWD) s = -s;           // forward: a cos - b sin; backward: a cos + b sin
                }
                cs[i] = ok ? c : __uint_as_float(0x7fc00000u);
                sn[i] = s;
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int h = (chunk * U + u) * ROWS + row_in_wave;
            const bool live = h < h_end;
            const bool is_q = h < a.Hq;
            float x[8], y[8], part[8];
            rx[u].get(x);
            float ss = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) ss = __builtin_fmaf(x[i], x[i], ss);
            if constexpr (!BWD) {
                const float r = rsqrtf(group_sum<LPR>(ss) * inv_d + a.eps);
#pragma unroll
                for (int i = 0; i < 8; ++i) x[i] = x[i] * r * (is_q ? wq[i] : wk[i]);
                partners<LPR, AL>(x, part, sub, lane, a.R, a.interleaved, lds);
#pragma unroll
                for (int i = 0; i < 8; ++i) y[i] = __builtin_fmaf(x[i], cs[i], part[i] * sn[i]);
            } else {
                float g[8];
                rg[u].get(g);
                partners<LPR, AL>(g, part, sub, lane, a.R, a.interleaved, lds);
                float gx = 0.0f;
                float gn[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    gn[i] = __builtin_fmaf(g[i], cs[i], part[i] * sn[i]);          // gradient of the normalised, weighted head
                    g[i] = gn[i] * (is_q ? wq[i] : wk[i]);
                    gx = __builtin_fmaf(g[i], x[i], gx);
                }
                const float r = rsqrtf(group_sum<LPR>(ss) * inv_d + a.eps);
                const float m = group_sum<LPR>(gx) * inv_d * r * r;              // mean(g xn) r
#pragma unroll
                for (int i = 0; i < 8; ++i) y[i] = __builtin_fmaf(g[i], r, -(x[i] * r * m));
                if (a.dw_part && live) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const float d = gn[i] * x[i] * r;
                        if (is_q) dwq[i] += d;
                        else dwk[i] += d;
                    }
                }
            }
            if (live) {
                T* o = is_q ? (T*)a.q_out + (token * a.Hq + h) * a.D : (T*)a.k_out + (token * a.Hk + (h - a.Hq)) * a.D;
                store8<T, AL>(o + e0, y, n);
            }
        }
    }
    if constexpr (BWD) {
        if (a.dw_part) {
            // fixed order: lanes of a wave that hold the same values (xor shuffles), then the waves one after the other
            for (int which = 0; which < 2; ++which) {
                __syncthreads();
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    float v = which ? dwk[i] : dwq[i];
#pragma unroll
                    for (int o = LPR; o < 64; o <<= 1) v += __shfl_xor(v, o, 64);
                    if (row_in_wave == 0) exch[wave * 512 + e0 + i] = v;
                }
                __syncthreads();
                for (int d = threadIdx.x; d < a.D; d += kRopeThreads) {
                    float v = 0.0f;
                    for (int w = 0; w < WAVES; ++w) v += exch[w * 512 + d];
                    a.dw_part[((int64_t)blockIdx.x * 2 + which) * a.D + d] = v;
                }
            }
        }
    }
}

// dw[which][d] = sum over blocks of part[block][which][d], 32 columns a workgroup, 8 row groups added in a fixed order.
template <class T>
__global__ __launch_bounds__(256) void rope_dw_kernel(const float* __restrict__ part, int blocks, int D, T* dqw, T* dkw) {
    __shared__ float red[8][32];
    const int c = threadIdx.x & 31, g = threadIdx.x >> 5;
    const int col = blockIdx.x * 32 + c;
    float v = 0.0f;
    if (col < 2 * D)
        for (int b = g; b < blocks; b += 8) v += part[(int64_t)b * 2 * D + col];
    red[g][c] = v;
    __syncthreads();
    if (g == 0 && col < 2 * D) {
        for (int i = 1; i < 8; ++i) v += red[i][c];
        T* out = col < D ? dqw : dkw;
        if (out) {
            const int d = col < D ? col : col - D;
            if constexpr (sizeof(T) == 2) out[d] = (uint16_t)cvt_pk_bf16(v, v);
            else out[d] = v;
        }
    }
}

constexpr int kRopeMaxBlocks = 2048;

template <class T, bool BWD>
int launch_rope(RopeArgs a, bool aligned, int* blocks, hipStream_t st) {      // *blocks: workgroups launched
    int lpr = 2;
    while (lpr * 8 < a.D) lpr *= 2;
    const int rows = 64 / lpr, H = a.Hq + a.Hk, cus = num_cus();
    if (cus <= 0) return fail(NGPT_EINVAL, "no HIP device");
    const int steps = (H + rows - 1) / rows;
    const int64_t tokens = (int64_t)a.B * a.T;
    // Several heads' loads in flight per lane once there are waves enough to fill the compute units without that
    // (a few tokens: every wave takes one step, so that all of them run at once).
    const int u = tokens * steps >= (int64_t)cus * 16 ? (BWD ? 2 : 4) : 1;
    a.chunks = (steps + u - 1) / u;
    a.items = tokens * a.chunks;
    int64_t grid = (a.items + 3) / 4;
    if (grid > kRopeMaxBlocks) grid = kRopeMaxBlocks;
    auto go = [&](auto kernel) { kernel<<<(int)grid, kRopeThreads, 0, st>>>(a); };
    auto pick = [&](auto lpr_c) {
        constexpr int L = decltype(lpr_c)::value;
        if (aligned) {
            if (u == 1) go(qk_rope_kernel<T, L, true, BWD, 1>);
            else go(qk_rope_kernel<T, L, true, BWD, BWD ? 2 : 4>);
        } else {
            if (u == 1) go(qk_rope_kernel<T, L, false, BWD, 1>);
            else go(qk_rope_kernel<T, L, false, BWD, BWD ? 2 : 4>);
        }
    };
    switch (lpr) {
        case 2: pick(std::integral_constant<int, 2>{}); break;
        case 4: pick(std::integral_constant<int, 4>{}); break;
        case 8: pick(std::integral_constant<int, 8>{}); break;
        case 16: pick(std::integral_constant<int, 16>{}); break;
        case 32: pick(std::integral_constant<int, 32>{}); break;
        default: pick(std::integral_constant<int, 64>{}); break;
    }
    *blocks = (int)grid;
    return check_launch("qk_rope_kernel");
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

// Host-side checks shared by both directions.  Returns NGPT_OK and fills `a`.
int rope_args(const char* who, RopeArgs& a, const void* q, const int64_t* qs, const void* k, const int64_t* ks, int dtype, int B, int T, int Hq,
              int Hk, int D, int R, const void* cos, const void* sin, int tab_dtype, int P, const void* pos, int pos64,
              const int64_t* ps, const void* qw, const void* kw, float eps, int interleaved, void* q_out, void* k_out) {
    if (!q || !k || !qs || !ks || !cos || !sin || !q_out || !k_out) return fail(NGPT_EINVAL, "%s: null pointer", who);
    if (dtype != NGPT_DT_BF16 && dtype != NGPT_DT_F32) return fail(NGPT_EINVAL, "%s: dtype=%d", who, dtype);
    if (tab_dtype != NGPT_DT_BF16 && tab_dtype != NGPT_DT_F32) return fail(NGPT_EINVAL, "%s: tab_dtype=%d", who, tab_dtype);
    if (B <= 0 || T <= 0 || Hq <= 0 || Hk <= 0 || P <= 0) return fail(NGPT_EINVAL, "%s: empty problem B=%d T=%d Hq=%d Hk=%d P=%d", who, B, T, Hq, Hk, P);
    if (D < 2 || D > 512) return fail(NGPT_ERANGE, "%s: head size %d outside 2 .. 512", who, D);
    if (R < 2 || R > D || R % 2) return fail(NGPT_EALIGN, "%s: %d rotated values of %d: need an even number from 2 to the head size", who, R, D);
    if (!pos && T > P) return fail(NGPT_ERANGE, "%s: %d positions in the tables, %d tokens in a sequence", who, P, T);
    if (pos && !ps) return fail(NGPT_EINVAL, "%s: positions without strides", who);
    if (!(eps >= 0.0f)) return fail(NGPT_ERANGE, "%s: eps=%g", who, (double)eps);
    a.q = q; a.k = k;
    a.q_sb = qs[0]; a.q_st = qs[1]; a.q_sh = qs[2];
    a.k_sb = ks[0]; a.k_st = ks[1]; a.k_sh = ks[2];
    a.q_out = q_out; a.k_out = k_out;
    a.cos = cos; a.sin = sin; a.tab_bf16 = tab_dtype == NGPT_DT_BF16;
    a.pos = pos; a.pos64 = pos64;
    if (pos) { a.p_sb = ps[0]; a.p_st = ps[1]; }
    a.qw = qw; a.kw = kw;
    a.B = B; a.T = T; a.Hq = Hq; a.Hk = Hk; a.D = D; a.R = R; a.P = P;
    a.eps = eps;
    a.interleaved = interleaved != 0;
    return NGPT_OK;
}

// 16-byte accesses: every row starts on 16 bytes and the pairs' halves are whole 8-value pieces.
bool rope_aligned(const RopeArgs& a, int dtype, bool bwd) {
    const int64_t per16 = dtype == NGPT_DT_BF16 ? 8 : 4;
    bool ok = a.D % 8 == 0 && (a.interleaved ? a.R % 2 == 0 : a.R % 16 == 0) && aligned16(a.q) && aligned16(a.k) && aligned16(a.q_out) && aligned16(a.k_out);
    for (int64_t s : {a.q_sb, a.q_st, a.q_sh, a.k_sb, a.k_st, a.k_sh}) ok = ok && s % per16 == 0;
    if (bwd) {
        ok = ok && aligned16(a.dq) && aligned16(a.dk);
        for (int64_t s : {a.dq_sb, a.dq_st, a.dq_sh, a.dk_sb, a.dk_st, a.dk_sh}) ok = ok && s % per16 == 0;
    }
    return ok;
}

}  // namespace
}  // namespace ngpt

using namespace ngpt;

extern "C" int ngpt_qk_norm_rope(const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides, int dtype,
                                 int B, int T, int Hq, int Hk, int D, int R, const void* cos_tab, const void* sin_tab,
                                 int tab_dtype, int P, const void* positions, int positions_64, const int64_t* pos_strides,
                                 const void* q_weight, const void* k_weight, float eps, int interleaved,
                                 void* q_out, void* k_out, void* stream) {
    RopeArgs a{};
    if (int e = rope_args("ngpt_qk_norm_rope", a, q, q_strides, k, k_strides, dtype, B, T, Hq, Hk, D, R, cos_tab, sin_tab, tab_dtype, P,
                          positions, positions_64, pos_strides, q_weight, k_weight, eps, interleaved, q_out, k_out)) return e;
    const bool al = rope_aligned(a, dtype, false);
    ProfileScope prof(PROF_PRODUCERS, (hipStream_t)stream);
    int blocks = 0;
    return dtype == NGPT_DT_BF16 ? launch_rope<uint16_t, false>(a, al, &blocks, (hipStream_t)stream)
                                 : launch_rope<float, false>(a, al, &blocks, (hipStream_t)stream);
}

extern "C" int64_t ngpt_qk_norm_rope_bwd_workspace_bytes(int D) { return (int64_t)kRopeMaxBlocks * 2 * (D > 0 ? D : 0) * 4; }

extern "C" int ngpt_qk_norm_rope_bwd(const void* dq_out, const int64_t* dq_strides, const void* dk_out, const int64_t* dk_strides,
                                     const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides, int dtype,
                                     int B, int T, int Hq, int Hk, int D, int R, const void* cos_tab, const void* sin_tab,
                                     int tab_dtype, int P, const void* positions, int positions_64, const int64_t* pos_strides,
                                     const void* q_weight, const void* k_weight, float eps, int interleaved,
                                     void* dq, void* dk, void* dq_weight, void* dk_weight,
                                     void* workspace, int64_t workspace_bytes, void* stream) {
    RopeArgs a{};
    if (int e = rope_args("ngpt_qk_norm_rope_bwd", a, q, q_strides, k, k_strides, dtype, B, T, Hq, Hk, D, R, cos_tab, sin_tab, tab_dtype, P,
                          positions, positions_64, pos_strides, q_weight, k_weight, eps, interleaved, dq, dk)) return e;
    if (!dq_out || !dk_out || !dq_strides || !dk_strides) return fail(NGPT_EINVAL, "ngpt_qk_norm_rope_bwd: null pointer");
    a.dq = dq_out; a.dk = dk_out;
    a.dq_sb = dq_strides[0]; a.dq_st = dq_strides[1]; a.dq_sh = dq_strides[2];
    a.dk_sb = dk_strides[0]; a.dk_st = dk_strides[1]; a.dk_sh = dk_strides[2];
    const bool want_dw = dq_weight || dk_weight;
    if (want_dw) {
        if (!workspace || workspace_bytes < ngpt_qk_norm_rope_bwd_workspace_bytes(D))
            return fail(NGPT_EWORKSPACE, "ngpt_qk_norm_rope_bwd: workspace %lld < %lld bytes", (long long)workspace_bytes,
                        (long long)ngpt_qk_norm_rope_bwd_workspace_bytes(D));
        a.dw_part = (float*)workspace;
    }
    const bool al = rope_aligned(a, dtype, true);
    hipStream_t st = (hipStream_t)stream;
    ProfileScope prof(PROF_PRODUCERS, st);
    int blocks = 0;
    if (int e = dtype == NGPT_DT_BF16 ? launch_rope<uint16_t, true>(a, al, &blocks, st) : launch_rope<float, true>(a, al, &blocks, st)) return e;
    if (!want_dw) return NGPT_OK;
    const int grid = (2 * D + 31) / 32;
    if (dtype == NGPT_DT_BF16) rope_dw_kernel<uint16_t><<<grid, 256, 0, st>>>(a.dw_part, blocks, D, (uint16_t*)dq_weight, (uint16_t*)dk_weight);
    else rope_dw_kernel<float><<<grid, 256, 0, st>>>(a.dw_part, blocks, D, (float*)dq_weight, (float*)dk_weight);
    return check_launch("rope_dw_kernel");
}
