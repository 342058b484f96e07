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
//
// Measured: 49152 tokens x 12 bf16 heads of 128, 64 values turned: forward 58 us (302 MB, 5.2 TB/s), backward 97 us (453 MB, 4.7 TB/s); a large
// copy reaches 5.1 on this card.  8193 tokens x 16 fp32 heads of 80 with weights: 22 and 28 us, their sums 4 us.  16 tokens x 20 heads: 4.6 us,
// of which an empty launch is about 2.5 and the rest two dependent round trips (the position, then its row of the tables).
#include "common.h"
#include "host_util.h"
#include <algorithm>

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

// Sum over the LPR lanes of a row; every lane gets it.  Inside 16 lanes by lane permutations of the vector pipe.
template <int CTRL>
__device__ __forceinline__ float permuted(float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}
template <int LPR>
__device__ __forceinline__ float group_sum(float v) {
    v += permuted<0xb1>(v);                        // lanes 1 0 3 2
    v += permuted<0x4e>(v);                        // lanes 2 3 0 1
    v += permuted<0x141>(v);                       // mirrored inside 8
    if (LPR >= 16) v += permuted<0x140>(v);        // mirrored inside 16
    if (LPR >= 32) v += __shfl_xor(v, 16, 64);
    if (LPR >= 64) v += __shfl_xor(v, 32, 64);
    return v;
}

// REG: the halves of the rotated part are whole pieces of 8 values (or the pairs are neighbours), so that a value's partner lies in the same
// place of ONE other lane; rows of the tables then start on 16 bytes.  AL: 16-byte accesses to the heads.
template <class T, int LPR, bool AL, bool REG, bool BWD, bool W, int U>
__global__ __launch_bounds__(kRopeThreads) void qk_rope_kernel(RopeArgs a) {
    constexpr int ROWS = 64 / LPR;                    // rows (heads) of a wave
    constexpr int WAVES = kRopeThreads / 64;
    constexpr bool LDS = !REG || (BWD && W);
    __shared__ __attribute__((aligned(16))) float exch[LDS ? WAVES * 512 : 1];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int sub = lane & (LPR - 1), row_in_wave = lane / LPR;
    const int e0 = sub * 8;
    const int n = a.D - e0;                           // values of this lane that exist (<= 0: none)
    const int H = a.Hq + a.Hk, half = a.R / 2;
    const float inv_d = 1.0f / (float)a.D;
    float* const row_lds = exch + (LDS ? wave * 512 + (lane - sub) * 8 : 0);
    const float nan = __uint_as_float(0x7fc00000u);

    // lane that holds the partners of this lane's values, and the place of the lane's values in a row of the tables
    const int src = a.interleaved || e0 >= a.R ? lane : (e0 < half ? lane + half / 8 : lane - half / 8);
    const int tab0 = a.interleaved ? e0 / 2 : (e0 < half ? e0 : e0 - half);

    float wq[W ? 8 : 1], wk[W ? 8 : 1], dwq[W && BWD ? 8 : 1], dwk[W && BWD ? 8 : 1];
    if constexpr (W) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            wq[i] = a.qw && i < n ? load1<T>((const T*)a.qw + e0 + i) : 1.0f;
            wk[i] = a.kw && i < n ? load1<T>((const T*)a.kw + e0 + i) : 1.0f;
            if constexpr (BWD) dwq[i] = dwk[i] = 0.0f;
        }
    }

    const int tokens = a.B * a.T;                     // (fits: checked on the host)
    for (int token = blockIdx.x * WAVES + wave; token < tokens; token += gridDim.x * WAVES) {
        const int b = token / a.T, t = token - b * a.T;
        const T* const q0 = (const T*)a.q + (b * a.q_sb + t * a.q_st);
        const T* const k0 = (const T*)a.k + (b * a.k_sb + t * a.k_st);
        const T* const dq0 = BWD ? (const T*)a.dq + (b * a.dq_sb + t * a.dq_st) : nullptr;
        const T* const dk0 = BWD ? (const T*)a.dk + (b * a.dk_sb + t * a.dk_st) : nullptr;
        T* const qo = (T*)a.q_out + (int64_t)token * a.Hq * a.D;
        T* const ko = (T*)a.k_out + (int64_t)token * a.Hk * a.D;
        // cos / sin of the lane's values; sn carries the sign of the partner's term (forward: a cos - b sin).  A position outside the
        // tables reads row 0 and makes the token's heads NaN.
        float cs[8], sn[8];
        {
            int64_t pos = t;
            if (a.pos) pos = a.pos64 ? ((const int64_t*)a.pos)[b * a.p_sb + t * a.p_st] : (int64_t)((const int32_t*)a.pos)[b * a.p_sb + t * a.p_st];
            const bool ok = pos >= 0 && pos < a.P;
            const int64_t base = (ok ? pos : 0) * half;
            if (REG && !a.tab_bf16) {
                const float *c = (const float*)a.cos + base + tab0, *s = (const float*)a.sin + base + tab0;
                if (e0 < a.R) {
                    const v4f c0 = *(const v4f*)c, s0 = *(const v4f*)s;
                    if (a.interleaved) {
#pragma unroll
                        for (int i = 0; i < 8; ++i) { cs[i] = c0[i / 2]; sn[i] = s0[i / 2]; }
                    } else {
                        const v4f c1 = *(const v4f*)(c + 4), s1 = *(const v4f*)(s + 4);
#pragma unroll
                        for (int i = 0; i < 4; ++i) { cs[i] = c0[i]; cs[4 + i] = c1[i]; sn[i] = s0[i]; sn[4 + i] = s1[i]; }
                    }
                }
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int e = e0 + i;
                    if (e < a.R) {
                        const int64_t at = base + (a.interleaved ? e >> 1 : (e < half ? e : e - half));
                        cs[i] = a.tab_bf16 ? load1<uint16_t>((const uint16_t*)a.cos + at) : ((const float*)a.cos)[at];
                        sn[i] = a.tab_bf16 ? load1<uint16_t>((const uint16_t*)a.sin + at) : ((const float*)a.sin)[at];
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int e = e0 + i;
                const bool first = a.interleaved ? !(e & 1) : e < half;
                cs[i] = !ok ? nan : (e < a.R ? cs[i] : 1.0f);
                sn[i] = e < a.R ? (first != BWD ? -sn[i] : sn[i]) : 0.0f;
            }
        }
        for (int s0 = blockIdx.y * U; s0 * ROWS < H; s0 += gridDim.y * U) {
            // the loads of all steps are issued before the first is used
            Raw8<T, AL> rx[U], rg[BWD ? U : 1];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int h = (s0 + u) * ROWS + row_in_wave;
                const bool is_q = h < a.Hq;
                const int m = h < H ? n : 0;
                rx[u].load((is_q ? q0 + h * a.q_sh : k0 + (h - a.Hq) * a.k_sh) + e0, m);
                if constexpr (BWD) rg[u].load((is_q ? dq0 + h * a.dq_sh : dk0 + (h - a.Hq) * a.dk_sh) + e0, m);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int h = (s0 + u) * ROWS + row_in_wave;
                const bool live = h < H, is_q = h < a.Hq;
                float x[8], y[8], g[BWD ? 8 : 1], gn[BWD && W ? 8 : 1];
                rx[u].get(x);
                float ss = 0.0f, gx = 0.0f;
#pragma unroll
                for (int i = 0; i < 8; ++i) ss = __builtin_fmaf(x[i], x[i], ss);
                // what is turned: forward x (times the weight), backward dy
                float v[8], part[8];
                if constexpr (BWD) rg[u].get(v);
                else
#pragma unroll
                    for (int i = 0; i < 8; ++i) v[i] = W ? x[i] * (is_q ? wq[i] : wk[i]) : x[i];
                if constexpr (REG) {
                    if (a.interleaved) {
#pragma unroll
                        for (int i = 0; i < 8; ++i) part[i] = v[i ^ 1];
                    } else {
#pragma unroll
                        for (int i = 0; i < 8; ++i) part[i] = __shfl(v[i], src, 64);
                    }
                } else {          // through the wave's own LDS block: LDS operations of one wave execute in order
                    *(v4f*)(row_lds + e0) = (v4f){v[0], v[1], v[2], v[3]};
                    *(v4f*)(row_lds + e0 + 4) = (v4f){v[4], v[5], v[6], v[7]};
                    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const int e = e0 + i;
                        part[i] = row_lds[e >= a.R ? e : (a.interleaved ? (e ^ 1) : (e < half ? e + half : e - half))];
                    }
                    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                }
                if constexpr (!BWD) {
                    const float r = rsqrtf(group_sum<LPR>(ss) * inv_d + a.eps);
#pragma unroll
                    for (int i = 0; i < 8; ++i) y[i] = r * __builtin_fmaf(v[i], cs[i], part[i] * sn[i]);
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const float turned = __builtin_fmaf(v[i], cs[i], part[i] * sn[i]);      // gradient of the normalised, weighted head
                        if constexpr (W) gn[i] = turned;
                        g[i] = W ? turned * (is_q ? wq[i] : wk[i]) : turned;
                        gx = __builtin_fmaf(g[i], x[i], gx);
                    }
                    const float r = rsqrtf(group_sum<LPR>(ss) * inv_d + a.eps);
                    const float m = group_sum<LPR>(gx) * inv_d * r * r;              // mean(g xn) r
#pragma unroll
                    for (int i = 0; i < 8; ++i) y[i] = r * __builtin_fmaf(-x[i], m, g[i]);
                    if constexpr (W) {
                        if (a.dw_part && live) {
#pragma unroll
                            for (int i = 0; i < 8; ++i) {
                                const float d = gn[i] * x[i] * r;
                                if (is_q) dwq[i] += d;
                                else dwk[i] += d;
                            }
                        }
                    }
                }
                if (live) store8<T, AL>((is_q ? qo + h * a.D : ko + (h - a.Hq) * a.D) + e0, y, n);
            }
        }
    }
    if constexpr (BWD && W) {
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
                    a.dw_part[(((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * 2 + which) * a.D + d] = v;
                }
            }
        }
    }
}

// dw[which][d] = sum over blocks of part[block][which][d], 32 columns a workgroup
template <class T>
__global__ __launch_bounds__(kColSumThreads) void rope_dw_kernel(const float* __restrict__ part, int blocks, int D, T* dqw, T* dkw) {
    __shared__ float red[32][33];
    const int col = blockIdx.x * 32 + (threadIdx.x & 31);
    const float v = col_sum32(part, blocks, 2 * (int64_t)D, col, col < 2 * D, red);
    if (threadIdx.x >= 32 || col >= 2 * D) return;
    T* out = col < D ? dqw : dkw;
    if (!out) return;
    const int d = col < D ? col : col - D;
    if constexpr (sizeof(T) == 2) out[d] = (uint16_t)cvt_pk_bf16(v, v);
    else out[d] = v;
}

constexpr int kRopeMaxBlocks = 2048;
constexpr int kRopeSumBlocks = 1024;      // with weight gradients: as many as are resident, each leaves its sums

template <class T, bool BWD>
int launch_rope(RopeArgs a, bool aligned, bool regular, int* blocks, hipStream_t st) {      // *blocks: workgroups launched
    int lpr = 8;
    while (lpr * 8 < a.D) lpr *= 2;
    const int rows = 64 / lpr, H = a.Hq + a.Hk, cus = num_cus();
    if (cus <= 0) return fail(NGPT_EINVAL, "no HIP device");
    const int steps = (H + rows - 1) / rows;
    const int64_t tokens = (int64_t)a.B * a.T;
    // A wave walks all heads of its tokens and has several steps' loads in flight, where there are tokens enough to fill the compute
    // units; with fewer every step is a wave of its own.  The number of steps that leaves the fewest empty ones, the larger first.
    const bool many = tokens >= (int64_t)cus * 16;
    int u = 1;
    if (many && aligned && regular) {
        int best = 1 << 30;
        for (int c = BWD ? 3 : 4; c >= 2; --c) {
            const int waste = (steps + c - 1) / c * c - steps;
            if (waste < best) { best = waste; u = c; }
        }
    }
    int64_t gx = (tokens + 3) / 4;
    const int gy = many ? 1 : std::min(steps, kRopeSumBlocks);
    const int most = a.dw_part ? kRopeSumBlocks : kRopeMaxBlocks;
    if (gx * gy > most) gx = most / gy;
    if (gx < 1) gx = 1;
    const bool weights = a.qw || a.kw || a.dw_part;
    const dim3 grid((unsigned)gx, (unsigned)gy);
    auto go = [&](auto kernel) { kernel<<<grid, kRopeThreads, 0, st>>>(a); };
    auto pick = [&](auto lpr_c) {
        constexpr int L = decltype(lpr_c)::value;
        auto steps_of = [&](auto w_c) {
            constexpr bool W = decltype(w_c)::value;
            if (u == 1) go(qk_rope_kernel<T, L, true, true, BWD, W, 1>);
            else if (u == 2) go(qk_rope_kernel<T, L, true, true, BWD, W, 2>);
            else if (u == 3) go(qk_rope_kernel<T, L, true, true, BWD, W, 3>);
            else if constexpr (!BWD) go(qk_rope_kernel<T, L, true, true, BWD, W, 4>);
        };
        if (!aligned) go(qk_rope_kernel<T, L, false, false, BWD, true, 1>);
        else if (!regular) go(qk_rope_kernel<T, L, true, false, BWD, true, 1>);
        else if (weights) steps_of(std::true_type{});
        else steps_of(std::false_type{});
    };
    switch (lpr) {
        case 8: pick(std::integral_constant<int, 8>{}); break;
        case 16: pick(std::integral_constant<int, 16>{}); break;
        case 32: pick(std::integral_constant<int, 32>{}); break;
        default: pick(std::integral_constant<int, 64>{}); break;
    }
    *blocks = (int)(gx * gy);
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
    if ((int64_t)B * T > (1 << 30)) return fail(NGPT_ERANGE, "%s: %lld tokens", who, (long long)B * T);
    if (Hq > (1 << 20) || Hk > (1 << 20)) return fail(NGPT_ERANGE, "%s: Hq=%d Hk=%d", who, Hq, Hk);
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

// 16-byte accesses: every head starts on 16 bytes.
bool rope_aligned(const RopeArgs& a, int dtype, bool bwd) {
    const int64_t per16 = dtype == NGPT_DT_BF16 ? 8 : 4;
    bool ok = a.D % 8 == 0 && aligned16(a.q) && aligned16(a.k) && aligned16(a.q_out) && aligned16(a.k_out);
    for (int64_t s : {a.q_sb, a.q_st, a.q_sh, a.k_sb, a.k_st, a.k_sh}) ok = ok && s % per16 == 0;
    if (bwd) {
        ok = ok && aligned16(a.dq) && aligned16(a.dk);
        for (int64_t s : {a.dq_sb, a.dq_st, a.dq_sh, a.dk_sb, a.dk_st, a.dk_sh}) ok = ok && s % per16 == 0;
    }
    return ok;
}
// Halves of whole 8-value pieces (pairs of neighbours: whole pieces), rows of the tables on 16 bytes.
bool rope_regular(const RopeArgs& a) { return (a.interleaved ? a.R % 8 == 0 : a.R % 16 == 0) && aligned16(a.cos) && aligned16(a.sin); }

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
    return dtype == NGPT_DT_BF16 ? launch_rope<uint16_t, false>(a, al, rope_regular(a), &blocks, (hipStream_t)stream)
                                 : launch_rope<float, false>(a, al, rope_regular(a), &blocks, (hipStream_t)stream);
}

extern "C" int64_t ngpt_qk_norm_rope_bwd_workspace_bytes(int D) { return (int64_t)kRopeSumBlocks * 2 * (D > 0 ? D : 0) * 4; }

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
    if (int e = dtype == NGPT_DT_BF16 ? launch_rope<uint16_t, true>(a, al, rope_regular(a), &blocks, st) : launch_rope<float, true>(a, al, rope_regular(a), &blocks, st)) return e;
    if (!want_dw) return NGPT_OK;
    const int grid = (2 * D + 31) / 32;
    if (dtype == NGPT_DT_BF16) rope_dw_kernel<uint16_t><<<grid, kColSumThreads, 0, st>>>(a.dw_part, blocks, D, (uint16_t*)dq_weight, (uint16_t*)dk_weight);
    else rope_dw_kernel<float><<<grid, kColSumThreads, 0, st>>>(a.dw_part, blocks, D, (float*)dq_weight, (float*)dk_weight);
    return check_launch("rope_dw_kernel");
}
