// linear_act for few rows and for sizes or alignments that the 256 x 256 tile GEMM does not serve.
//
// Loads go through registers here, 16 bytes at any byte address (gfx950 takes unaligned global loads), so rows may start anywhere and K is any
// length; only a row's last, incomplete piece is read value by value.
#include "linear.h"
#include <algorithm>

namespace ngpt {
namespace {

// values k .. k + 7 of a row of K; zeros behind its end
__device__ __forceinline__ v4i load_k8(const uint16_t* row, int k, int K) {
    v4i w = {0, 0, 0, 0};
    if (k + 8 <= K) __builtin_memcpy(&w, row + k, 16);
    else if (k < K) w = load8(row + k, K - k, false);
    return w;
}

template <class F>
__device__ __forceinline__ void act_switch(int act, F&& f) {      // wave-uniform
    switch (act) {
        case NGPT_ACT_RELU2: f(std::integral_constant<int, NGPT_ACT_RELU2>{}); break;
        case NGPT_ACT_GELU: f(std::integral_constant<int, NGPT_ACT_GELU>{}); break;
        case NGPT_ACT_GELU_TANH: f(std::integral_constant<int, NGPT_ACT_GELU_TANH>{}); break;
        case NGPT_ACT_SILU: f(std::integral_constant<int, NGPT_ACT_SILU>{}); break;
        default: f(std::integral_constant<int, NGPT_ACT_NONE>{}); break;
    }
}

// ---------------------------------------------------------------------------------------------- few rows
// Every weight is read once and used for at most 64 rows: the bound is the weights' way from memory, and for one token the launch and one
// round trip.  A workgroup owns 16 FT features; its waves share the contraction in units of 64 values (a line of every weight row), with all
// loads of U units in flight, multiply on 16x16x32 matrix instructions (rows past M repeat the last and are dropped) and add up through LDS
// in wave order.
// Matrix instruction: lane l, q = l / 16: A row / B column l % 16, contraction 8 q .. 8 q + 7; D column l % 16, rows 4 q .. 4 q + 3.
template <int FT, int MT, int U>
__global__ __launch_bounds__(1024) void linear_few_kernel(LinearOut o, const uint16_t* __restrict__ x, int64_t ldx, const uint16_t* __restrict__ w,
                                                          int64_t ldw, int K, int act) {
    extern __shared__ __attribute__((aligned(16))) v4f part[];      // [wave][FT][MT][lane]
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const int r = lane & 15, q = lane >> 4;
    const int f0 = blockIdx.x * 16 * FT;
    const uint16_t *wr[FT], *xr[MT];
#pragma unroll
    for (int i = 0; i < FT; ++i) wr[i] = w + (int64_t)min(f0 + 16 * i + r, o.N - 1) * ldw;
#pragma unroll
    for (int i = 0; i < MT; ++i) xr[i] = x + (int64_t)min(16 * i + r, o.M - 1) * ldx;
    v4f acc[FT][MT];
#pragma unroll
    for (int i = 0; i < FT; ++i)
#pragma unroll
        for (int j = 0; j < MT; ++j) acc[i][j] = (v4f){0, 0, 0, 0};
    const int units = (K + 63) / 64;
    for (int u0 = wave; u0 < units; u0 += waves * U) {
        v4i a[U][2][FT], b[U][2][MT];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                const int k = (u0 + u * waves) * 64 + s * 32 + q * 8;      // past the end: zeros
#pragma unroll
                for (int i = 0; i < FT; ++i) a[u][s][i] = load_k8(wr[i], k, K);
#pragma unroll
                for (int j = 0; j < MT; ++j) b[u][s][j] = load_k8(xr[j], k, K);
            }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int i = 0; i < FT; ++i)
#pragma unroll
                    for (int j = 0; j < MT; ++j)
                        acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, a[u][s][i]), __builtin_bit_cast(v8bf, b[u][s][j]),
                                                                            acc[i][j], 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < FT; ++i)
#pragma unroll
        for (int j = 0; j < MT; ++j) part[((wave * FT + i) * MT + j) * 64 + lane] = acc[i][j];
    __syncthreads();
    for (int t = wave; t < FT * MT; t += waves) {
        v4f z = part[t * 64 + lane];
        for (int p = 1; p < waves; ++p) z += part[(p * FT * MT + t) * 64 + lane];
        const int i = t / MT, j = t % MT;
        const int m = 16 * j + r, f = f0 + 16 * i + 4 * q, left = o.N - f;
        if (m >= o.M || left <= 0) continue;
        const int64_t at = (int64_t)m * o.N + f;
        float y[4];
        uint32_t pre[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            y[e] = z[e] + (o.bias && e < left ? bf16_bits_to_f32(o.bias[f + e]) : 0.0f);
            pre[e] = cvt_pk_bf16(y[e], y[e]) & 0xffffu;
        }
        act_switch(act, [&](auto kind) {
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = act_of<decltype(kind)::value>(y[e]);
        });
        if (o.res) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (e < left) y[e] += bf16_bits_to_f32(o.res[(int64_t)m * o.ld_res + f + e]);
        }
        if (o.vec) {      // (N % 8 == 0: the four features exist)
            *(v2i*)(o.out + at) = (v2i){(int)cvt_pk_bf16(y[0], y[1]), (int)cvt_pk_bf16(y[2], y[3])};
            if (o.pre) *(v2i*)(o.pre + at) = (v2i){(int)(pre[0] | pre[1] << 16), (int)(pre[2] | pre[3] << 16)};
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (e < left) {
                    o.out[at + e] = (uint16_t)cvt_pk_bf16(y[e], y[e]);
                    if (o.pre) o.pre[at + e] = (uint16_t)pre[e];
                }
        }
    }
}

// ---------------------------------------------------------------------------------------------- tiles of 128 x 128 or 64 x 64
// Four waves as 2 x 2, TM x TM matrix tiles of 32 x 32 each.  A k-step is 64 values: rows of 128 bytes in LDS, their eight 16-byte pieces
// swizzled by the row as in gemm_tn.h.  Operands pass through registers, loaded two k-steps ahead of their use; two LDS stages, one barrier a
// k-step.  Several workgroups share a compute unit and cover each other's latencies.
template <int TM>
struct MidCfg {
    static constexpr int B = 64 * TM;                 // tile edge
    static constexpr int LOADS = 2 * B * 8 / 256;     // 16-byte pieces a thread moves per k-step, A then B
    static constexpr int STAGE = 2 * B * 128;         // bytes
    static constexpr int SMEM = 2 * STAGE;
};

template <int TM, bool PRE, bool RES>
__global__ __launch_bounds__(256, 2) void linear_mid_kernel(LinearOut o, const uint16_t* __restrict__ x, int64_t ldx, const uint16_t* __restrict__ w,
                                                            int64_t ldw, int K, int act) {
    using Cfg = MidCfg<TM>;
    __shared__ __attribute__((aligned(1024))) uint8_t smem[Cfg::SMEM];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wr = wave >> 1, wc = wave & 1;
    // tiles in runs of consecutive numbers per XCD (workgroup b runs on XCD b % 8); features fastest inside groups of 8 row tiles
    const int tf = (o.N + Cfg::B - 1) / Cfg::B, tm = (o.M + Cfg::B - 1) / Cfg::B, total = tf * tm;
    int t = blockIdx.x;
    if (total % 8 == 0) t = (t & 7) * (total >> 3) + (t >> 3);
    const int per = 8 * tf, grp = t / per, gsz = min(tm - grp * 8, 8), in_grp = t - grp * per;
    const int f0 = (in_grp / gsz) * Cfg::B, m0 = (grp * 8 + in_grp % gsz) * Cfg::B;

    // thread -> piece tid % 8 of row tid / 8 (+ 32 per load); rows past the end repeat the last (dropped by the epilogue)
    const int lrow = tid >> 3, chunk = tid & 7;
    uint32_t off[Cfg::LOADS];
#pragma unroll
    for (int i = 0; i < Cfg::LOADS; ++i) {
        const bool is_w = i < Cfg::LOADS / 2;
        const int row = lrow + 32 * (is_w ? i : i - Cfg::LOADS / 2);
        off[i] = is_w ? (uint32_t)(min(row, o.N - 1 - f0) * ldw) : (uint32_t)(min(row, o.M - 1 - m0) * ldx);
    }
    const uint16_t* const wt = w + (int64_t)f0 * ldw;
    const uint16_t* const xt = x + (int64_t)m0 * ldx;
    v4i reg[Cfg::LOADS];
    const int steps = (K + 63) / 64;
    auto load = [&](int kt) {
        const int k = kt * 64 + chunk * 8;
        if (kt * 64 + 64 <= K) {
#pragma unroll
            for (int i = 0; i < Cfg::LOADS; ++i) __builtin_memcpy(&reg[i], (i < Cfg::LOADS / 2 ? wt : xt) + off[i] + k, 16);
        } else {
#pragma unroll
            for (int i = 0; i < Cfg::LOADS; ++i) reg[i] = load_k8((i < Cfg::LOADS / 2 ? wt : xt) + off[i], k, K);
        }
    };
    auto put = [&](int stage) {
        uint8_t* s = smem + stage * Cfg::STAGE;
#pragma unroll
        for (int i = 0; i < Cfg::LOADS; ++i) {
            const int row = lrow + 32 * i;           // B's rows follow A's
            *(v4i*)(s + row * 128 + ((chunk ^ ((row >> 1) & 7)) << 4)) = reg[i];
        }
    };
    v16f acc[TM][TM];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TM; ++j) acc[i][j] = (v16f){0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
    int fa[TM], fb[TM];
#pragma unroll
    for (int i = 0; i < TM; ++i) {
        const int ra = wr * 32 * TM + i * 32 + (lane & 31), rb = Cfg::B + wc * 32 * TM + i * 32 + (lane & 31);
        fa[i] = ra * 128 + (((lane >> 5) ^ ((ra >> 1) & 7)) << 4);
        fb[i] = rb * 128 + (((lane >> 5) ^ ((rb >> 1) & 7)) << 4);
    }
    load(0);
    put(0);
    if (steps > 1) load(1);
    for (int kt = 0; kt < steps; ++kt) {
        wg_barrier();                                // stage kt % 2 is complete, stage (kt + 1) % 2 has been read
        if (kt + 1 < steps) put((kt + 1) & 1);
        if (kt + 2 < steps) load(kt + 2);
        const uint8_t* s = smem + (kt & 1) * Cfg::STAGE;
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) {             // 16 values: chunks 2 ks, 2 ks + 1
            v8bf a[TM], b[TM];
#pragma unroll
            for (int i = 0; i < TM; ++i) a[i] = *(const v8bf*)(s + (fa[i] ^ (ks * 32)));
#pragma unroll
            for (int i = 0; i < TM; ++i) b[i] = *(const v8bf*)(s + (fb[i] ^ (ks * 32)));
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int j = 0; j < TM; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[i], b[j], acc[i][j], 0, 0, 0);
        }
    }
    wg_barrier();                                    // the stages become the waves' staging areas
    uint8_t* const stage = smem + wave * 2048 * TM;
    act_switch(act, [&](auto kind) {
        linear_epilogue<decltype(kind)::value, PRE, RES>(o, acc, stage, f0 + wr * 32 * TM, m0 + wc * 32 * TM, lane);
    });
}

}  // namespace

int linear_few(const LinearOut& o, const uint16_t* x, int64_t ldx, const uint16_t* w, int64_t ldw, int K, int act, hipStream_t st) {
    const int cus = num_cus();
    if (cus <= 0) return fail(NGPT_EINVAL, "no HIP device");
    auto go = [&](auto ft, auto mt, auto u) {
        constexpr int FT = decltype(ft)::value, MT = decltype(mt)::value, U = decltype(u)::value;
        const int groups = (o.N + 16 * FT - 1) / (16 * FT), units = (K + 63) / 64;
        // waves that share a group's contraction: as many as there are units for, fewer where the groups alone fill the compute units
        int waves = groups <= cus ? 16 : (groups <= 2 * cus ? 8 : 4);
        while (waves > 1 && waves > units) waves /= 2;
        const int lds = waves * FT * MT * 1024;
        static_assert(16 * FT * MT * 1024 <= 65536, "fits without asking for more");
        linear_few_kernel<FT, MT, U><<<groups, 64 * waves, lds, st>>>(o, x, ldx, w, ldw, K, act);
        return check_launch("linear_few_kernel");
    };
    std::integral_constant<int, 1> c1;
    std::integral_constant<int, 2> c2;
    std::integral_constant<int, 4> c4;
    if (o.M <= 16) return go(c1, c1, c4);
    if (o.M <= 32) return go(c1, c2, c2);
    return go(c1, c4, c2);
}

int linear_mid(const LinearOut& o, const uint16_t* x, int64_t ldx, const uint16_t* w, int64_t ldw, int K, int act, hipStream_t st) {
    auto go = [&](auto tm_c) {
        constexpr int TM = decltype(tm_c)::value, B = MidCfg<TM>::B;
        const int64_t tiles = (int64_t)((o.N + B - 1) / B) * ((o.M + B - 1) / B);
        if (tiles > 0x7fffffff) return fail(NGPT_ERANGE, "linear_mid: M=%d N=%d", o.M, o.N);
        auto run = [&](auto kernel) { kernel<<<(unsigned)tiles, 256, 0, st>>>(o, x, ldx, w, ldw, K, act); };
        if (o.pre) o.res ? run(linear_mid_kernel<TM, true, true>) : run(linear_mid_kernel<TM, true, false>);
        else o.res ? run(linear_mid_kernel<TM, false, true>) : run(linear_mid_kernel<TM, false, false>);
        return check_launch("linear_mid_kernel");
    };
    const int64_t big = (int64_t)((o.N + 127) / 128) * ((o.M + 127) / 128);
    return big >= 4 * (int64_t)num_cus() ? go(std::integral_constant<int, 2>{}) : go(std::integral_constant<int, 1>{});
}

}  // namespace ngpt
