// Distillation loss against a teacher's top logits, and its gradient.
//
//   z = softcap(l) / tau      softcap(l) = A sigmoid((l + B) / C), or l itself;   q = softmax(z) over the V columns
//   p over the listed columns: softmax of the teacher's listed logits / tau, or exp(t / tau - lse_t) with the teacher's own
//   log-sum-exp given; the rest of its mass, 1 - sum p, then stands against the rest of the student's
//   loss = weight tau^2 ( sum_j p_j (log p_j - log q_{id_j})  [ + P (log P - log Q) ] )     P = 1 - sum p, Q = 1 - sum_{listed} q
//   d loss / d z_v tau^-1 = weight tau ( q_v F_v - p_v ),  F_v = sum p + P on listed columns, sum p + P - P / Q elsewhere
//   (F = 1 without the rest), and the softcap's slope A / C sigma (1 - sigma) on top.
// Entries whose id is not a column are ignored; a row without entries has loss 0 and gradient 0; a row of weight 0 too.
//
// A row is 100 KB (50304 bf16), read once and, with a gradient, written once: the bound is memory.  One workgroup of 1024
// threads owns a row at a time; every thread keeps its pieces of the row in registers from the load to the store.
//  * the exponentials are taken relative to a reference of the thread's own (its maximum; the cap's upper end with a softcap,
//    which needs no maximum), so one workgroup reduction of (reference, sum) pairs is all that a row needs;
//  * what is kept per logit is the gradient up to the row's factor, e or e sigma (1 - sigma), in fp32;
//  * wave 0 prepares the listed columns of the row meanwhile (normaliser, duplicates, the student's logits there) and hands
//    every one to the thread that owns the column, by a list in LDS: each byte of the gradient is stored once.
#include "common.h"
#include "host_util.h"
#include <cmath>

namespace ngpt {
namespace {

constexpr int kDistThreads = 1024;
constexpr int kDistWaves = kDistThreads / 64;
constexpr int kDistMaxTop = 512;          // listed columns a row may have (each takes 40 bytes of LDS)

enum : int { DIST_LOSS = 0, DIST_FUSED = 1, DIST_BWD = 2 };

struct DistArgs {
    const void* logits;       // [T, V], row stride ld
    int64_t ld;
    const void* ids;          // [T, K] int32 or int64
    const float* teacher;     // [T, K]
    const float* teacher_lse; // nullable [T]
    const float* weight;      // nullable [T]
    const float* dloss;       // DIST_BWD: [T], stride dloss_st
    int64_t dloss_st;
    float* losses;            // DIST_LOSS, DIST_FUSED: [T]
    float* stats;             // DIST_LOSS: written if given, DIST_BWD: read.  [T] of StatRow
    void* grad;               // [T, V], row stride ldg
    int64_t ldg;
    int T, V, K, ids64;
    int vec_grad;             // the gradient's rows have the same offset to 16 bytes as the logits' rows
    float tau;
    float grad_scale;
    float k1, k0;             // softcap: 2^(k1 l + k0) = exp(-(l + B) / C)
    float k2;                 // exp(z) = 2^(k2 sigma) (softcap) or 2^(k2 l)
    float slope;              // A / C (softcap) or 1
};

template <class T> struct Elem;
template <> struct Elem<uint16_t> {
    static constexpr int PER = 8;
    static __device__ float at(v4i w, int i) {
        const uint32_t x = (uint32_t)w[i >> 1];
        return __uint_as_float((i & 1) ? (x & 0xffff0000u) : (x << 16));
    }
    static __device__ float one(const uint16_t* p) { return bf16_bits_to_f32(*p); }
};
template <> struct Elem<float> {
    static constexpr int PER = 4;
    static __device__ float at(v4i w, int i) { return __int_as_float(w[i]); }
    static __device__ float one(const float* p) { return *p; }
};

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

// A row starts anywhere on its element size.  Pieces are the 16-byte blocks of the address space that it touches; the
// first and the last may belong to it in part only and are then read and written value by value.
struct RowSpan {
    int shift;       // values between the start of the first block and the row
    int pieces;
    template <class T>
    __device__ RowSpan(const T* row, int V) {
        shift = (int)(((uintptr_t)row & 15) / sizeof(T));
        pieces = (V + shift + Elem<T>::PER - 1) / Elem<T>::PER;
    }
};

template <class T>
__device__ __forceinline__ v4i load_piece(const T* row, int V, const RowSpan& sp, int i) {
    // values outside the row read as -inf
    constexpr int PER = Elem<T>::PER;
    constexpr int kNegInf = sizeof(T) == 2 ? (int)0xff80ff80u : (int)0xff800000u;
    const int c0 = i * PER - sp.shift;             // column of the piece's first value
    v4i w = {kNegInf, kNegInf, kNegInf, kNegInf};
    if (i < sp.pieces) {
        if (c0 >= 0 && c0 + PER <= V) {
            w = *(const v4i*)(row + c0);
        } else {
#pragma unroll
            for (int e = 0; e < PER; ++e) {
                const int c = c0 + e;
                if (c >= 0 && c < V) {
                    if constexpr (sizeof(T) == 2) w[e >> 1] = (e & 1) ? (int)(((uint32_t)w[e >> 1] & 0xffffu) | ((uint32_t)row[c] << 16))
                                                                     : (int)(((uint32_t)w[e >> 1] & 0xffff0000u) | (uint32_t)row[c]);
                    else w[e] = __float_as_int(row[c]);
                }
            }
        }
    }
    return w;
}

template <class T>
__device__ __forceinline__ void store_piece(T* row, int V, const RowSpan& sp, int i, const float* g, bool vec) {
    constexpr int PER = Elem<T>::PER;
    const int c0 = i * PER - sp.shift;
    if (i >= sp.pieces) return;
    if (vec && c0 >= 0 && c0 + PER <= V) {
        if constexpr (sizeof(T) == 2)
            *(v4i*)(row + c0) = (v4i){(int)cvt_pk_bf16(g[0], g[1]), (int)cvt_pk_bf16(g[2], g[3]), (int)cvt_pk_bf16(g[4], g[5]), (int)cvt_pk_bf16(g[6], g[7])};
        else
            *(v4f*)(row + c0) = (v4f){g[0], g[1], g[2], g[3]};
        return;
    }
#pragma unroll
    for (int e = 0; e < PER; ++e) {
        const int c = c0 + e;
        if (c >= 0 && c < V) {
            if constexpr (sizeof(T) == 2) row[c] = (uint16_t)cvt_pk_bf16(g[e], g[e]);
            else row[c] = g[e];
        }
    }
}

// What z is proportional to: sigma (softcap) or the logit itself.
template <bool CAP>
__device__ __forceinline__ float z_arg(float l, const DistArgs& a) {
    if constexpr (CAP) return __builtin_amdgcn_rcpf(1.0f + exp2_hw(__builtin_fmaf(l, a.k1, a.k0)));
    else return l;
}

// 2^(k2 (arg - ref)).  The difference comes first: two logits at the type's lowest value are equal, k2 times them is not finite.
// A sigma is at most 1 and the reference there is 1, so one multiply-add does.
template <bool CAP>
__device__ __forceinline__ float rel_exp(float arg, float ref, float k2) {
    if constexpr (CAP) return exp2_hw(__builtin_fmaf(arg, k2, -(ref * k2)));
    else return exp2_hw((arg - ref) * k2);
}

// Row statistics that the forward leaves for the backward: q = rel_exp(arg, ref) * inv_sum; P / Q.
struct StatRow {
    float ref, inv_sum, rest_ratio, unused;
};

// The listed columns of one row, prepared by one wave, in LDS.
struct TopLds {
    int head[kDistThreads];          // first entry of a thread's list, -1: none
    int next[kDistMaxTop];
    int pos[kDistMaxTop];            // id + the row's shift; -1: not a column, or a repetition of an earlier entry
    float p[kDistMaxTop];            // the teacher's probability (repetitions added up)
    float arg[kDistMaxTop];          // z_arg of the student's logit
    float ref, sum;                  // largest arg of the listed columns; sum of rel_exp(arg, ref) over them, each counted once
    float cross;                     // sum p k2 (arg - ref)
    float sum_p, ent, rest_p;        // sum p; sum p log p [ + P log P ]; P
    int any;                         // entries that are columns
};

// Wave 0: everything about the listed columns that does not need the row's sum.
template <class T, bool CAP, bool TAIL>
__device__ __forceinline__ void prepare_top(const DistArgs& a, int row, const T* lrow, int shift, TopLds& tp, double* td, int lane) {
    constexpr int PER = Elem<T>::PER;
    const int K = a.K, V = a.V;
    auto lds_done = [] { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); };    // LDS of one wave is in order; keeps the compiler from reordering
    double tmax = -INFINITY;
    bool nan = false;
    int any = 0;
    for (int e = lane; e < K; e += 64) {
        const int64_t g = (int64_t)row * K + e;
        const int64_t c = a.ids64 ? ((const int64_t*)a.ids)[g] : (int64_t)((const int32_t*)a.ids)[g];
        const double t = (double)a.teacher[g] / (double)a.tau;
        const bool ok = c >= 0 && c < V;
        tp.pos[e] = ok ? (int)c + shift : -1;
        td[e] = t;
        if (ok) {
            ++any;
            tp.arg[e] = z_arg<CAP>(Elem<T>::one(lrow + c), a);
            nan = nan || t != t;
            tmax = t > tmax ? t : tmax;
        }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const double other = __shfl_xor(tmax, o, 64);
        tmax = other > tmax ? other : tmax;
        any += __shfl_xor(any, o, 64);
    }
    nan = __any(nan);
    // The mass outside the list is a small difference of numbers near one: the teacher's side is computed in 64 bits.
    double lse;
    if constexpr (TAIL) {
        lse = (double)a.teacher_lse[row];
    } else {
        if (tmax == -INFINITY && !nan) any = 0;         // nothing to distil from
        double s = 0.0;
        if (any)
            for (int e = lane; e < K; e += 64)
                if (tp.pos[e] >= 0) s += exp(td[e] - tmax);
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
        lse = tmax + log(s);
    }
    double sum_p = 0.0, ent = 0.0;
    float amax = -INFINITY;
    for (int e = lane; e < K; e += 64) {
        float p = 0.0f;
        if (any && tp.pos[e] >= 0) {
            const double lp = td[e] - lse, pe = exp(lp);
            if (pe != 0.0) {
                sum_p += pe;
                ent += pe * lp;
                p = (float)pe;
            }
            amax = fmaxf(amax, tp.arg[e]);
        }
        tp.p[e] = p;
    }
    amax = wave_max(amax);
    const float ref = amax > -INFINITY ? amax : 0.0f;
    float cross = 0.0f;
    for (int e = lane; e < K; e += 64) {
        const float p = tp.p[e];
        if (p != 0.0f) cross += p * ((tp.arg[e] - ref) * a.k2);
        // into the owner's list
        const int pos = tp.pos[e];
        if (pos >= 0) tp.next[e] = atomicExch(&tp.head[(pos / PER) % kDistThreads], e);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        sum_p += __shfl_xor(sum_p, o, 64);
        ent += __shfl_xor(ent, o, 64);
    }
    cross = wave_sum(cross);
    lds_done();
    // A column listed more than once: its first entry takes the sum of the p, in list order (an owner's list is short).
    for (int e = lane; e < K; e += 64) {
        const int pos = tp.pos[e];
        double total = -1.0;                            // a repetition
        if (pos >= 0) {
            bool first = true, repeated = false;
            for (int o = tp.head[(pos / PER) % kDistThreads]; o >= 0; o = tp.next[o])
                if (o != e && tp.pos[o] == pos) {
                    repeated = true;
                    first = first && o > e;
                }
            if (first) {
                float sum = tp.p[e];
                if (repeated)
                    for (int o = e + 1; o < K; ++o)
                        if (tp.pos[o] == pos) sum += tp.p[o];
                total = sum;
            }
        }
        td[e] = total;
    }
    lds_done();
    int distinct = 0;
    float top_sum = 0.0f;
    for (int e = lane; e < K; e += 64)
        if (tp.pos[e] >= 0) {
            if (td[e] == -1.0) {
                tp.pos[e] = -1;
            } else {
                tp.p[e] = (float)td[e];
                ++distinct;
                top_sum += rel_exp<CAP>(tp.arg[e], ref, a.k2);
            }
        }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) distinct += __shfl_xor(distinct, o, 64);
    top_sum = wave_sum(top_sum);
    if (lane == 0) {
        const double rest = TAIL && distinct < V ? (sum_p < 1.0 ? 1.0 - sum_p : sum_p - sum_p) : 0.0;     // (NaN stays NaN; every column listed: no rest)
        tp.ref = ref;
        tp.sum = top_sum;
        tp.cross = cross;
        tp.sum_p = (float)sum_p;
        tp.rest_p = (float)rest;
        tp.ent = (float)(ent + (rest > 0.0 ? rest * log(rest) : 0.0));
        tp.any = any;
    }
}

// Visits the entries of this thread's list that lie in the given sweep: f(entry, index among the sweep's values).
template <int NCH, int PER, class F>
__device__ __forceinline__ void for_listed(const TopLds& tp, int tid, int seg, F&& f) {
    for (int e = tp.head[tid]; e >= 0; e = tp.next[e]) {
        const int pos = tp.pos[e];
        if (pos < 0) continue;
        const int s = (pos / PER - tid) / kDistThreads - seg * NCH;
        if (s >= 0 && s < NCH) f(e, s * PER + pos % PER);
    }
}

// A sum relative to m taken relative to M >= m.  One whose reference is -inf is empty (or NaN, which is kept).
__device__ __forceinline__ float rescale(float s, float m, float M, float k2) { return m == -INFINITY ? s : s * exp2_hw((m - M) * k2); }

template <class T, int NCH, bool CAP, bool TAIL, int MODE>
__global__ __launch_bounds__(kDistThreads, MODE == DIST_FUSED ? 4 : 8) void distill_kernel(DistArgs a) {
    constexpr int PER = Elem<T>::PER;
    constexpr int N = NCH * PER;                        // values a thread holds
    constexpr int SEG = NCH * kDistThreads;             // pieces that one sweep over the registers covers
    constexpr float kLn2 = 0.6931471805599453f;
    __shared__ TopLds top[2];
    __shared__ double td[kDistMaxTop];
    __shared__ float red_m[2][kDistWaves], red_s[2][kDistWaves];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int V = a.V;
    // the cap is the largest z: no maximum is needed.  A value of -inf in place of one that is not summed adds exactly this:
    const float pad = CAP ? exp2_hw(-a.k2) : 0.0f;

    top[0].head[tid] = -1;
    top[1].head[tid] = -1;
    __syncthreads();

    int par = 0;
    for (int row = blockIdx.x; row < a.T; row += gridDim.x, par ^= 1) {
        const T* const lrow = (const T*)a.logits + (int64_t)row * a.ld;
        const RowSpan sp(lrow, V);
        TopLds& tp = top[par];
        const float weight = a.weight ? a.weight[row] : 1.0f;
        v4i raw[NCH];
        auto load_seg = [&](int seg) {
#pragma unroll
            for (int s = 0; s < NCH; ++s) raw[s] = load_piece<T>(lrow, V, sp, seg * SEG + s * kDistThreads + tid);
        };
        load_seg(0);
        if (wave == 0) prepare_top<T, CAP, TAIL>(a, row, lrow, sp.shift, tp, td, lane);
        if (TAIL || MODE == DIST_BWD) __syncthreads();

        float d[MODE == DIST_LOSS ? 1 : N];
        float m = CAP ? 1.0f : -INFINITY, S = 0.0f;         // reference, in units of z_arg, and the sum relative to it
        int skipped = 0;                                // values of this thread that are not summed
        const int segs = (sp.pieces + SEG - 1) / SEG;
        // Exponentials of one sweep, relative to `m`, and (forward) their sum.  With the rest of the teacher's mass in play
        // the sum is over the columns that are not listed: those are set to -inf first.
        auto sweep = [&](int seg) {
            if constexpr (MODE != DIST_BWD) {
                if constexpr (TAIL) {
                    for_listed<NCH, PER>(tp, tid, seg, [&](int, int idx) {
                        ++skipped;
#pragma unroll
                        for (int i = 0; i < NCH * 4; ++i)
                            if (i == idx * 4 / PER) {
                                if constexpr (PER == 4) raw[i >> 2][i & 3] = (int)0xff800000u;
                                else raw[i >> 2][i & 3] = (idx & 1) ? (int)(((uint32_t)raw[i >> 2][i & 3] & 0xffffu) | 0xff800000u)
                                                                   : (int)(((uint32_t)raw[i >> 2][i & 3] & 0xffff0000u) | 0xff80u);
                            }
                    });
                }
                if constexpr (CAP) {
#pragma unroll
                    for (int s = 0; s < NCH; ++s) {
                        const int c0 = (seg * SEG + s * kDistThreads + tid) * PER - sp.shift;
                        skipped += PER - max(0, min(c0 + PER, V) - max(c0, 0));
                    }
                } else {
                    float top_l = -INFINITY;
#pragma unroll
                    for (int i = 0; i < N; ++i) top_l = fmaxf(top_l, Elem<T>::at(raw[i / PER], i % PER));
                    const float mnew = fmaxf(m, top_l);
                    if (mnew > m) {
                        S = rescale(S, m, mnew, a.k2);
                        m = mnew;
                    }
                }
            }
            const float ref = m == -INFINITY ? 0.0f : m;      // nothing but -inf so far: every exponential is 0
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float arg = z_arg<CAP>(Elem<T>::at(raw[i / PER], i % PER), a);
                const float ex = rel_exp<CAP>(arg, ref, a.k2);
                if constexpr (MODE != DIST_BWD) S += ex;
                if constexpr (MODE != DIST_LOSS) d[i] = CAP ? ex * (arg * (1.0f - arg)) : ex;
            }
        };
        // Gradient of one sweep: f times what the thread holds; listed columns from their own statistics.
        auto emit = [&](int seg, float f, float base, float ref, float inv_sum, bool none) {
            T* const grow = (T*)a.grad + (int64_t)row * a.ldg;
            if (none) {
#pragma unroll
                for (int i = 0; i < N; ++i) d[i] = 0.0f;
            } else {
#pragma unroll
                for (int i = 0; i < N; ++i) d[i] *= f;
                for_listed<NCH, PER>(tp, tid, seg, [&](int e, int idx) {
                    const float arg = tp.arg[e];
                    const float q = rel_exp<CAP>(arg, ref, a.k2) * inv_sum;
                    const float v = base * (q * (tp.sum_p + tp.rest_p) - tp.p[e]) * (CAP ? arg * (1.0f - arg) : 1.0f);
#pragma unroll
                    for (int i = 0; i < N; ++i) d[i] = i == idx ? v : d[i];
                });
            }
#pragma unroll
            for (int s = 0; s < NCH; ++s)
                store_piece<T>(grow, V, sp, seg * SEG + s * kDistThreads + tid, &d[s * PER], a.vec_grad != 0);
        };

        if constexpr (MODE == DIST_BWD) {
            const StatRow st = ((const StatRow*)a.stats)[row];
            const float base = weight * a.dloss[(int64_t)row * a.dloss_st] * a.tau * a.slope;
            const bool none = tp.any == 0 || weight == 0.0f;
            m = st.ref;
            for (int seg = 0; seg < segs; ++seg) {
                if (seg) load_seg(seg);
                sweep(seg);
                emit(seg, base * st.inv_sum * (tp.sum_p + tp.rest_p - st.rest_ratio), base, st.ref, st.inv_sum, none);
            }
        } else {
            sweep(0);
            if constexpr (MODE == DIST_LOSS) {
                for (int seg = 1; seg < segs; ++seg) {
                    load_seg(seg);
                    sweep(seg);
                }
            }
            if constexpr (CAP) S = __builtin_fmaf(-(float)skipped, pad, S);
            const float wm = CAP ? m : wave_max(m);
            const float ws = wave_sum(rescale(S, m, wm, a.k2));
            if (lane == 0) {
                red_m[par][wave] = wm;
                red_s[par][wave] = ws;
            }
            __syncthreads();
            float M = red_m[par][0];
#pragma unroll
            for (int w = 1; w < kDistWaves; ++w) M = fmaxf(M, red_m[par][w]);
            float sum = 0.0f;
#pragma unroll
            for (int w = 0; w < kDistWaves; ++w) sum += rescale(red_s[par][w], red_m[par][w], M, a.k2);
            float rest_ratio = 0.0f, p_logq = 0.0f;
            if constexpr (TAIL) {
                // the sum so far is Q's; with the listed columns it is the row's
                const float rest_m = M, rest_s = sum;
                M = fmaxf(M, tp.ref);
                sum = rescale(rest_s, rest_m, M, a.k2) + rescale(tp.sum, tp.ref, M, a.k2);
                if (!(tp.rest_p <= 0.0f)) {
                    const float log2q = (rest_m - M) * a.k2 + (__builtin_amdgcn_logf(rest_s) - __builtin_amdgcn_logf(sum));
                    p_logq = tp.rest_p * log2q;
                    rest_ratio = tp.rest_p * exp2_hw(-log2q);
                }
            }
            const float inv_sum = 1.0f / sum;
            const bool none = tp.any == 0 || weight == 0.0f;
            if (tid == 0) {
                const float lse_rel = (M - tp.ref) * a.k2 + __builtin_amdgcn_logf(sum);       // relative to the listed columns' reference
                const float kl = tp.ent + kLn2 * (tp.sum_p * lse_rel - tp.cross - p_logq);
                a.losses[row] = none ? 0.0f : weight * a.tau * a.tau * kl;
                if (MODE == DIST_LOSS && a.stats) ((StatRow*)a.stats)[row] = StatRow{M, inv_sum, rest_ratio, 0.0f};
            }
            if constexpr (MODE == DIST_FUSED) {
                const float base = weight * a.tau * a.grad_scale * a.slope;
                emit(0, base * inv_sum * rescale(1.0f, m, M, a.k2) * (tp.sum_p + tp.rest_p - rest_ratio), base, M, inv_sum, none);
            }
        }
        tp.head[tid] = -1;          // wave 0 fills this buffer again two rows on, behind the next row's barrier
    }
}

template <class T, int NCH, bool CAP, bool TAIL, int MODE>
int launch_distill(const DistArgs& a, hipStream_t st) {
    const int cus = num_cus();
    if (cus <= 0) return fail(NGPT_EINVAL, "no HIP device");
    const int resident = cus * (MODE == DIST_FUSED ? 1 : 2);
    distill_kernel<T, NCH, CAP, TAIL, MODE><<<a.T < resident ? a.T : resident, kDistThreads, 0, st>>>(a);
    return check_launch("distill_kernel");
}

// Pieces of a row that starts anywhere: one more than the aligned count.
template <class T> int most_pieces(int V) { return V / Elem<T>::PER + 2; }

template <class T, bool CAP, bool TAIL>
int run_distill(const DistArgs& a, int mode, hipStream_t st) {
    if (mode == DIST_LOSS) return launch_distill<T, 2, CAP, TAIL, DIST_LOSS>(a, st);
    if (mode == DIST_BWD) return launch_distill<T, 2, CAP, TAIL, DIST_BWD>(a, st);
    // the row in registers: 16, 32 or 56 values a thread
    constexpr int BIG = sizeof(T) == 2 ? 7 : 14;
    const int pieces = most_pieces<T>(a.V);
    if (pieces <= 2 * kDistThreads) return launch_distill<T, 2, CAP, TAIL, DIST_FUSED>(a, st);
    if (pieces <= 4 * kDistThreads) return launch_distill<T, 4, CAP, TAIL, DIST_FUSED>(a, st);
    return launch_distill<T, BIG, CAP, TAIL, DIST_FUSED>(a, st);
}
// Columns of a row that fits the registers wherever it starts
template <class T> constexpr int fused_max_cols() { return ((sizeof(T) == 2 ? 7 : 14) * kDistThreads - 2) * Elem<T>::PER; }

int run_distill(const DistArgs& a, int dtype, int mode, hipStream_t st) {
    const bool cap = a.k1 != 0.0f, tail = a.teacher_lse != nullptr;
    auto go = [&](auto t) {
        using T = decltype(t);
        if (cap) return tail ? run_distill<T, true, true>(a, mode, st) : run_distill<T, true, false>(a, mode, st);
        return tail ? run_distill<T, false, true>(a, mode, st) : run_distill<T, false, false>(a, mode, st);
    };
    return dtype == NGPT_DT_BF16 ? go(uint16_t{}) : go(float{});
}

int distill_args(const char* who, DistArgs& a, const void* logits, int dtype, int64_t ld, const void* ids, int ids_64, const float* teacher,
                 const float* teacher_lse, const float* weight, int T, int V, int K, float tau, float A, float B, float C) {
    if (!logits || !ids || !teacher) return fail(NGPT_EINVAL, "%s: null pointer", who);
    if (dtype != NGPT_DT_BF16 && dtype != NGPT_DT_F32) return fail(NGPT_EINVAL, "%s: dtype=%d", who, dtype);
    if (T <= 0 || V <= 0 || K <= 0) return fail(NGPT_EINVAL, "%s: empty problem T=%d V=%d K=%d", who, T, V, K);
    if (K > kDistMaxTop) return fail(NGPT_ERANGE, "%s: %d listed columns a row, at most %d", who, K, kDistMaxTop);
    if (V > (1 << 24)) return fail(NGPT_ERANGE, "%s: %d columns, at most 2^24", who, V);
    if (ld < V) return fail(NGPT_EALIGN, "%s: row stride %lld < V=%d", who, (long long)ld, V);
    if ((uintptr_t)logits % (dtype == NGPT_DT_BF16 ? 2 : 4)) return fail(NGPT_EALIGN, "%s: logits not aligned to their type", who);
    if (!(tau > 0.0f) || !std::isfinite(tau)) return fail(NGPT_ERANGE, "%s: temperature %g", who, (double)tau);
    constexpr double kLog2e = 1.4426950408889634;
    if (C == 0.0f) {
        a.k1 = a.k0 = 0.0f;
        a.k2 = (float)(kLog2e / tau);
        a.slope = 1.0f;
    } else {
        // exp(z) relative to the cap must not underflow for the smallest z, 0
        if (!(A > 0.0f) || !(C > 0.0f) || !std::isfinite(A) || !std::isfinite(B) || !std::isfinite(C) || !(A / tau <= 80.0f))
            return fail(NGPT_ERANGE, "%s: softcap A=%g B=%g C=%g at temperature %g: need A, C > 0 and A / temperature <= 80", who, (double)A,
                        (double)B, (double)C, (double)tau);
        a.k1 = (float)(-kLog2e / C);
        a.k0 = (float)(-kLog2e * B / C);
        a.k2 = (float)(kLog2e * A / tau);
        a.slope = A / C;
        if (a.k1 == 0.0f) return fail(NGPT_ERANGE, "%s: softcap C=%g", who, (double)C);
    }
    a.logits = logits; a.ld = ld; a.ids = ids; a.ids64 = ids_64; a.teacher = teacher; a.teacher_lse = teacher_lse; a.weight = weight;
    a.T = T; a.V = V; a.K = K; a.tau = tau;
    return NGPT_OK;
}

int set_grad(const char* who, DistArgs& a, int dtype, void* grad, int64_t ldg) {
    if (!grad) return fail(NGPT_EINVAL, "%s: null pointer", who);
    const int size = dtype == NGPT_DT_BF16 ? 2 : 4;
    if (ldg < a.V) return fail(NGPT_EALIGN, "%s: gradient row stride %lld < V=%d", who, (long long)ldg, a.V);
    if ((uintptr_t)grad % size) return fail(NGPT_EALIGN, "%s: gradient not aligned to its type", who);
    a.grad = grad; a.ldg = ldg;
    // whole pieces of the gradient start on 16 bytes where those of the logits do
    a.vec_grad = (((uintptr_t)grad - (uintptr_t)a.logits) & 15) == 0 && ((ldg - a.ld) * size) % 16 == 0;
    return NGPT_OK;
}

}  // namespace
}  // namespace ngpt

using namespace ngpt;

extern "C" int ngpt_distill_fused_max_cols(int dtype) { return dtype == NGPT_DT_BF16 ? fused_max_cols<uint16_t>() : fused_max_cols<float>(); }

extern "C" int64_t ngpt_distill_stats_bytes(int T) { return (int64_t)(T > 0 ? T : 0) * (int64_t)sizeof(StatRow); }

extern "C" int ngpt_distill_fwd(const void* logits, int dtype, int64_t ld, const void* ids, int ids_64, const float* teacher,
                                const float* teacher_lse, const float* row_weight, int T, int V, int K, float temperature,
                                float A, float B, float C, float* losses, float* stats, void* stream) {
    DistArgs a{};
    if (int e = distill_args("ngpt_distill_fwd", a, logits, dtype, ld, ids, ids_64, teacher, teacher_lse, row_weight, T, V, K, temperature, A, B, C)) return e;
    if (!losses) return fail(NGPT_EINVAL, "ngpt_distill_fwd: null pointer");
    a.losses = losses; a.stats = stats;
    return run_distill(a, dtype, DIST_LOSS, (hipStream_t)stream);
}

extern "C" int ngpt_distill_bwd(const void* logits, int dtype, int64_t ld, const void* ids, int ids_64, const float* teacher,
                                const float* teacher_lse, const float* row_weight, int T, int V, int K, float temperature,
                                float A, float B, float C, const float* stats, const float* dlosses, int64_t dlosses_stride,
                                void* grad, int64_t ld_grad, void* stream) {
    DistArgs a{};
    if (int e = distill_args("ngpt_distill_bwd", a, logits, dtype, ld, ids, ids_64, teacher, teacher_lse, row_weight, T, V, K, temperature, A, B, C)) return e;
    if (!stats || !dlosses) return fail(NGPT_EINVAL, "ngpt_distill_bwd: null pointer");
    if (int e = set_grad("ngpt_distill_bwd", a, dtype, grad, ld_grad)) return e;
    a.stats = (float*)stats; a.dloss = dlosses; a.dloss_st = dlosses_stride;
    return run_distill(a, dtype, DIST_BWD, (hipStream_t)stream);
}

extern "C" int ngpt_distill_fwd_bwd(const void* logits, int dtype, int64_t ld, const void* ids, int ids_64, const float* teacher,
                                    const float* teacher_lse, const float* row_weight, int T, int V, int K, float temperature,
                                    float A, float B, float C, float grad_scale, float* losses, void* grad, int64_t ld_grad, void* stream) {
    DistArgs a{};
    if (int e = distill_args("ngpt_distill_fwd_bwd", a, logits, dtype, ld, ids, ids_64, teacher, teacher_lse, row_weight, T, V, K, temperature, A, B, C)) return e;
    if (!losses) return fail(NGPT_EINVAL, "ngpt_distill_fwd_bwd: null pointer");
    if (int e = set_grad("ngpt_distill_fwd_bwd", a, dtype, grad, ld_grad)) return e;
    if (V > ngpt_distill_fused_max_cols(dtype))
        return fail(NGPT_ERANGE, "ngpt_distill_fwd_bwd: a row of %d columns does not fit the registers of a workgroup; use ngpt_distill_fwd and ngpt_distill_bwd", V);
    a.losses = losses; a.grad_scale = grad_scale;
    return run_distill(a, dtype, DIST_FUSED, (hipStream_t)stream);
}
