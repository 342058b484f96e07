// linear_act for few rows and for sizes or alignments that the 256 x 256 tile GEMM does not serve.
//
// Loads go through registers here, 16 bytes at any byte address (gfx950 takes unaligned global loads), so rows may start anywhere and K is any
// length; only a row's last, incomplete piece is read value by value.
#include "linear.h"
#include "launch.h"
#include <algorithm>

namespace ngpt {
namespace {

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
// A 4 x 4 exchange in every quad of lanes: register j of lane p takes what lane j of its quad holds in register p.
__device__ __forceinline__ void quad_transpose(v4i (&v)[4], bool odd, bool high) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        auto swap = [&](auto perm, bool up, int& lo, int& hi) {
            constexpr int P = decltype(perm)::value;
            const int from_hi = __builtin_amdgcn_update_dpp(0, hi, P, 0xf, 0xf, true), from_lo = __builtin_amdgcn_update_dpp(0, lo, P, 0xf, 0xf, true);
            const int l = up ? from_hi : lo, h = up ? hi : from_lo;
            lo = l;
            hi = h;
        };
        int t[4] = {v[0][e], v[1][e], v[2][e], v[3][e]};
        std::integral_constant<int, 0xB1> one;      // lane ^ 1
        std::integral_constant<int, 0x4E> two;      // lane ^ 2
        swap(one, odd, t[0], t[1]);
        swap(one, odd, t[2], t[3]);
        swap(two, high, t[0], t[2]);
        swap(two, high, t[1], t[3]);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j][e] = t[j];
    }
}

// Every weight is read once and used for at most 32 rows: the bound is the weights' way from memory, and for one token the launch and one
// round trip.  A workgroup owns 16 features; its waves share the contraction in units of 128 values, with all loads of U units in flight,
// multiply on 16x16x32 matrix instructions (rows past M repeat the last and are dropped) and add up through LDS in wave order.
// Matrix instruction: lane l, q = l / 16: A row / B column l % 16, contraction 8 q .. 8 q + 7; D column l % 16, rows 4 q .. 4 q + 3.
// Loaded in that order the four lanes of a quad would read from four rows, and the load unit takes such an instruction at about 45 clocks.  So
// load j reads rows j, 4 + j, 8 + j and 12 + j with the quad's lanes side by side, and the quads exchange in registers: lane (q, 4 a + p) then
// holds of row 4 a + p the piece 4 q + j of the unit in register j, for both operands.
// 12 x 4096 -> 1024: 7.0 us (8.8 without the exchange), 16 x 2048 -> 2048: 4.1 (6.0), 32 x 4096 -> 1024: 7.4 (12.9), 1 x 1024 -> 4096: 4.1, of which
// an empty launch is about 2.5; rows at odd addresses, 12 x 4095 -> 1023: 10.8.  Only N / 16 workgroups work, so a narrow result with a long
// contraction stays furthest from the memory's rate.  (Groups of 8 or 4 features: no shorter at any of these, 16 x 2048 -> 2048 9.7 with 4.)
template <int MT, int U>
__global__ __launch_bounds__(1024) void linear_few_kernel(LinearOut o, const uint16_t* __restrict__ x, int64_t ldx, const uint16_t* __restrict__ w,
                                                          int64_t ldw, int K, int act) {
    extern __shared__ __attribute__((aligned(16))) v4f part[];      // [wave][MT][lane]
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const int r = lane & 15, q = lane >> 4;
    const bool odd = lane & 1, high = lane & 2;
    const int f0 = blockIdx.x * 16, row0 = r & 12, k0 = 32 * q + 8 * (lane & 3);
    const uint16_t *wr[4], *xr[MT][4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        wr[j] = w + (int64_t)min(f0 + row0 + j, o.N - 1) * ldw + k0;
#pragma unroll
        for (int m = 0; m < MT; ++m) xr[m][j] = x + (int64_t)min(16 * m + row0 + j, o.M - 1) * ldx + k0;
    }
    v4f acc[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) acc[m] = (v4f){0, 0, 0, 0};
    // U units a pass, all of whose loads are in flight together; the last units, one of which may end inside the contraction, one by one
    auto pass = [&](int u0, auto count, auto load) {
        constexpr int C = decltype(count)::value;
        v4i a[C][4], b[C][MT][4];
#pragma unroll
        for (int u = 0; u < C; ++u) {
            const int k = (u0 + u * waves) * 128;
#pragma unroll
            for (int j = 0; j < 4; ++j) a[u][j] = load(wr[j], k);
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int j = 0; j < 4; ++j) b[u][m][j] = load(xr[m][j], k);
        }
        __builtin_amdgcn_sched_barrier(0);      // first every load of the pass, then the exchanges that wait for them
#pragma unroll
        for (int u = 0; u < C; ++u) {
            quad_transpose(a[u], odd, high);
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                quad_transpose(b[u][m], odd, high);
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    acc[m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, a[u][j]), __builtin_bit_cast(v8bf, b[u][m][j]), acc[m],
                                                                     0, 0, 0);
            }
        }
    };
    auto whole = [](const uint16_t* at, int k) {
        v4i v;
        __builtin_memcpy(&v, at + k, 16);
        return v;
    };
    std::integral_constant<int, 1> one;
    int u0 = wave;
    for (; (u0 + (U - 1) * waves + 1) * 128 <= K; u0 += waves * U) pass(u0, std::integral_constant<int, U>{}, whole);
    for (; (u0 + 1) * 128 <= K; u0 += waves) pass(u0, one, whole);
    if (u0 * 128 < K) {
        if (K >= 8) pass(u0, one, [K, k0](const uint16_t* at, int k) { return load_row8_end(at - k0, k0 + k, K); });
        else pass(u0, one, [K, k0](const uint16_t* at, int k) { return load_row8_short(at - k0, k0 + k, K); });
    }
#pragma unroll
    for (int m = 0; m < MT; ++m) part[(wave * MT + m) * 64 + lane] = acc[m];
    __syncthreads();
    for (int t = wave; t < MT; t += waves) {
        v4f z = part[t * 64 + lane];
        for (int p = 1; p < waves; ++p) z += part[(p * MT + t) * 64 + lane];
        const int m = 16 * t + r, f = f0 + 4 * q, left = o.N - f;
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
// KG groups of four waves share a tile and cut its contraction between them; each group works as 2 x 2 waves of TM x TM matrix tiles of 32 x 32
// with LDS stages of its own, and the groups' sums meet in LDS, in order.  A k-step is 64 values: rows of 128 bytes in LDS, their eight 16-byte
// pieces swizzled by the row as in gemm_tn.h.  Operands pass through registers, requested three k-steps ahead of their use; two LDS stages, one
// barrier a k-step.  A k-step of one group is mostly latency: several groups or workgroups on a compute unit cover each other's.
// 4096 x 1024 -> 1024 with bias and residual: 17.5 us (490 TFLOP/s), 2048 x 4096 -> 2048: 54 us (638); 1531 x 1004 -> 2311, rows at odd
// addresses: 25.5 us, the same on 16-byte rows of 1024: 16.8.  (Two groups on a 128 x 128 tile: 16.9 us where there is exactly one tile a
// compute unit, 24.4 against 18.6 just above, as only one such workgroup fits.)
template <int TM, int KG>
struct MidCfg {
    static constexpr int B = 64 * TM;                 // tile edge
    static constexpr int LOADS = 2 * B * 8 / 256;     // 16-byte pieces a thread moves per k-step, A then B
    static constexpr int STAGE = 2 * B * 128;         // bytes
    static constexpr int SMEM = 2 * STAGE * KG;
    static constexpr int THREADS = 256 * KG;
};

template <int TM, int KG, bool PRE, bool RES>
__global__ __launch_bounds__(256 * KG, KG == 4 ? 4 : 2) void linear_mid_kernel(LinearOut o, const uint16_t* __restrict__ x, int64_t ldx,
                                                                               const uint16_t* __restrict__ w, int64_t ldw, int K, int act) {
    using Cfg = MidCfg<TM, KG>;
    extern __shared__ __attribute__((aligned(1024))) uint8_t smem_all[];
    const int tid = threadIdx.x & 255, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int kg = __builtin_amdgcn_readfirstlane(threadIdx.x >> 8);
    const int wr = wave >> 1, wc = wave & 1;
    uint8_t* const smem = smem_all + kg * 2 * Cfg::STAGE;
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
    const int steps = (K + 63) / 64, mine = (steps + KG - 1) / KG, kt0 = kg * mine;      // every group walks `mine` steps, empty ones included
    auto load = [&](int kt, v4i (&reg)[Cfg::LOADS]) {
        const int k = (kt0 + kt) * 64 + chunk * 8;
        if (kt >= mine) return;
        if ((kt0 + kt) * 64 + 64 <= K) {
#pragma unroll
            for (int i = 0; i < Cfg::LOADS; ++i) __builtin_memcpy(&reg[i], (i < Cfg::LOADS / 2 ? wt : xt) + off[i] + k, 16);
        } else if (K >= 8) {
#pragma unroll
            for (int i = 0; i < Cfg::LOADS; ++i) reg[i] = load_row8_end((i < Cfg::LOADS / 2 ? wt : xt) + off[i], k, K);
        } else {
#pragma unroll
            for (int i = 0; i < Cfg::LOADS; ++i) reg[i] = load_row8_short((i < Cfg::LOADS / 2 ? wt : xt) + off[i], k, K);
        }
    };
    auto put = [&](int stage, const v4i (&reg)[Cfg::LOADS]) {
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
    v4i even[Cfg::LOADS], odd[Cfg::LOADS];
    // one k-step: `reg` holds step kt + 1 and is refilled with step kt + 3
    auto step = [&](int kt, v4i (&reg)[Cfg::LOADS]) {
        wg_barrier();                                // stage kt % 2 is complete, stage (kt + 1) % 2 has been read
        if (kt + 1 < mine) put((kt + 1) & 1, reg);
        load(kt + 3, reg);
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
    };
    load(0, even);
    put(0, even);
    load(1, odd);
    load(2, even);
    for (int kt = 0; kt < mine; kt += 2) {
        step(kt, odd);
        if (kt + 1 < mine) step(kt + 1, even);
    }
    wg_barrier();                                    // the stages are free
    if constexpr (KG > 1) {
        // groups 1 .. leave their sums: [group][wave][tile][quarter][lane] of 16 bytes
        v4f* const part = (v4f*)smem_all;
        if (kg > 0) {
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int j = 0; j < TM; ++j)
#pragma unroll
                    for (int v = 0; v < 4; ++v)
                        part[((((kg - 1) * 4 + wave) * TM * TM + i * TM + j) * 4 + v) * 64 + lane] =
                            (v4f){acc[i][j][4 * v], acc[i][j][4 * v + 1], acc[i][j][4 * v + 2], acc[i][j][4 * v + 3]};
        }
        wg_barrier();
        if (kg > 0) return;
#pragma unroll
        for (int g = 0; g < KG - 1; ++g)
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int j = 0; j < TM; ++j)
#pragma unroll
                    for (int v = 0; v < 4; ++v) {
                        const v4f p = part[(((g * 4 + wave) * TM * TM + i * TM + j) * 4 + v) * 64 + lane];
#pragma unroll
                        for (int e = 0; e < 4; ++e) acc[i][j][4 * v + e] += p[e];
                    }
    }
    // staging areas of the remaining waves, behind the sums
    constexpr int kSums = (KG - 1) * 4 * TM * TM * 4096;
    static_assert(kSums + 4 * 2048 * TM <= Cfg::SMEM, "sums and staging areas fit the stages");
    uint8_t* const stage = smem_all + kSums + wave * 2048 * TM;
    act_switch(act, [&](auto kind) {
        linear_epilogue<decltype(kind)::value, PRE, RES>(o, acc, stage, f0 + wr * 32 * TM, m0 + wc * 32 * TM, lane);
    });
}

}  // namespace

int linear_few(const LinearOut& o, const uint16_t* x, int64_t ldx, const uint16_t* w, int64_t ldw, int K, int act, hipStream_t st) {
    const int cus = num_cus();
    if (cus <= 0) return fail(NGPT_EINVAL, "no HIP device");
    auto go = [&](auto mt, auto u) {
        constexpr int MT = decltype(mt)::value, U = decltype(u)::value;
        const int groups = (o.N + 15) / 16, units = (K + 127) / 128;
        // waves that share a group's contraction: as many as there are units for, fewer where the groups alone fill the compute units
        int waves = groups <= cus ? 16 : (groups <= 2 * cus ? 8 : 4);
        while (waves > 1 && waves > units) waves /= 2;
        const int lds = waves * MT * 1024;
        static_assert(16 * MT * 1024 <= 65536, "fits without asking for more");
        linear_few_kernel<MT, U><<<groups, 64 * waves, lds, st>>>(o, x, ldx, w, ldw, K, act);
        return check_launch("linear_few_kernel");
    };
    std::integral_constant<int, 1> c1;
    std::integral_constant<int, 2> c2;
    if (o.M <= 16) return go(c1, c2);
    return go(c2, c1);
}

int linear_mid(const LinearOut& o, const uint16_t* x, int64_t ldx, const uint16_t* w, int64_t ldw, int K, int act, hipStream_t st) {
    const int cus = num_cus();
    if (cus <= 0) return fail(NGPT_EINVAL, "no HIP device");
    auto go = [&](auto tm_c, auto kg_c) {
        constexpr int TM = decltype(tm_c)::value, KG = decltype(kg_c)::value;
        using Cfg = MidCfg<TM, KG>;
        const int64_t tiles = (int64_t)((o.N + Cfg::B - 1) / Cfg::B) * ((o.M + Cfg::B - 1) / Cfg::B);
        if (tiles > 0x7fffffff) return fail(NGPT_ERANGE, "linear_mid: M=%d N=%d", o.M, o.N);
        auto run = [&](auto pre, auto res) {
            auto kernel = linear_mid_kernel<TM, KG, decltype(pre)::value, decltype(res)::value>;
            static PerDeviceOnce configured;         // one per instantiation of this lambda, i.e. per kernel
            if (int e = configured.run([&] { return allow_lds(kernel, Cfg::SMEM); })) return e;
            kernel<<<(unsigned)tiles, Cfg::THREADS, Cfg::SMEM, st>>>(o, x, ldx, w, ldw, K, act);
            return check_launch("linear_mid_kernel");
        };
        std::true_type yes;
        std::false_type no;
        if (o.pre) return o.res ? run(yes, yes) : run(yes, no);
        return o.res ? run(no, yes) : run(no, no);
    };
    std::integral_constant<int, 1> c1;
    std::integral_constant<int, 2> c2;
    std::integral_constant<int, 4> c4;
    auto tiles = [&](int b) { return (int64_t)((o.N + b - 1) / b) * ((o.M + b - 1) / b); };
    // one 128 x 128 tile for every compute unit (1024 x 1024 -> 4096: 16.3 us, tiles of 64: 17.9; 2048 x 4096 -> 1024, half as many: 49 against 34)
    if (tiles(128) >= cus) return go(c2, c1);
    // Tiles of 64: a contraction in two where there are few (1024 x 1024 -> 1024: 7.1 us, in one piece 8.0, in four 7.5), in four where it is long
    // as well (1024 x 4096 -> 1024: 18.9 us, in two 20.3, in one piece 27.6).
    const int64_t t64 = tiles(64);
    const int steps = (K + 63) / 64;
    if (t64 >= 3 * (int64_t)cus || steps < 4) return go(c1, c1);
    if (t64 > cus || steps < 32) return go(c1, c2);
    return go(c1, c4);
}

}  // namespace ngpt
