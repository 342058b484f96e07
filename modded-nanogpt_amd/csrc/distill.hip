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
// A row is 100 KB (50304 bf16), read once and, with a gradient, written once: the bound is memory.  One workgroup of 960 + 64
// threads owns a row at a time; every one of the 960 keeps its pieces of the row in registers from the load to the store.
//  * the exponentials are taken relative to a reference of the thread's own (its maximum; the cap's upper end with a softcap,
//    which needs no maximum), so one workgroup reduction of (reference, sum) pairs is all that a row needs;
//  * with a softcap no input gives an exponential of 0.  What is not summed (places outside the row, and the listed columns where the
//    rest's mass is summed) is read as -inf, summed and subtracted.  Relative to 2^k2_up, the power of two above the cap, -inf adds
//    2^-k2_up, the smallest term there is and a power of two as well: a thread's sum of such terms alone is exact and leaves nothing
//    behind, and next to one real term they cost it at most 64 roundings of 2^-24.  (Relative to the cap itself every one of up to 960
//    threads left about 1e-6 of such a term, all of one sign: 0.01 to 0.04 of a single column's term at A / temperature = 1.)
//  * what is kept per logit is the gradient up to the row's factor, e or e sigma (1 - sigma), in fp32;
//  * a sixteenth wave prepares the listed columns (normaliser, repetitions, the student's logits there) of the NEXT row and hands
//    every one to the thread that owns the column, by a list in LDS; the owner stores it after the piece it lies in;
//  * the next row's loads are issued before this row is reduced and written: one barrier a row.
// Measured: 8192 rows of 50304 bf16 with softcap and 64 listed columns, loss and gradient in one pass: 317 to 322 us (1.65 GB, 5.1 to 5.2 TB/s: a
// large copy's rate; 1331 us with rows in branches and the lists on the row's own waves).  1003 rows of 50257 fp32 with the rest's mass: loss 47 to 57 us
// (202 MB), gradient 80 us (403 MB, 5.0 TB/s).  Seven rows, loss only: 7.9 us, one row's way through one compute unit.
#include "common.h"
#include "host_util.h"
#include <cmath>

namespace ngpt {
namespace {

typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));

constexpr int kDistThreads = 960;                         // threads that hold the row
constexpr int kDistWaves = kDistThreads / 64;
constexpr int kDistBlock = kDistThreads + 64;             // and one wave for the listed columns
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
    float k2_up, from_up;     // softcap: the whole number next above k2, and 2^(k2_up - k2)
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

// Value by value only where a piece lies in the row in part (a loop: it is rare, and code size matters more).
template <class T>
__device__ __forceinline__ v4i load_piece(const T* row, int V, const RowSpan& sp, int i) {
    // values outside the row read as -inf
    constexpr int PER = Elem<T>::PER;
    constexpr int kNegInf = sizeof(T) == 2 ? (int)0xff80ff80u : (int)0xff800000u;
    const int c0 = i * PER - sp.shift;             // column of the piece's first value
    if (c0 >= 0 && c0 + PER <= V) return *(const v4i*)(row + c0);
    v4i w = {kNegInf, kNegInf, kNegInf, kNegInf};
    if (i < sp.pieces) {
#pragma unroll 1
        for (int e = PER - 1; e >= 0; --e) {       // the piece as one 128-bit number, shifted up value by value
            const int c = c0 + e;
            const bool in = c >= 0 && c < V;
            if constexpr (sizeof(T) == 2) {
                w.w = (int)__builtin_amdgcn_alignbit((uint32_t)w.w, (uint32_t)w.z, 16);
                w.z = (int)__builtin_amdgcn_alignbit((uint32_t)w.z, (uint32_t)w.y, 16);
                w.y = (int)__builtin_amdgcn_alignbit((uint32_t)w.y, (uint32_t)w.x, 16);
                w.x = (int)(((uint32_t)w.x << 16) | (in ? (uint32_t)row[c] : 0xff80u));
            } else {
                w.w = w.z;
                w.z = w.y;
                w.y = w.x;
                w.x = in ? __float_as_int(row[c]) : kNegInf;
            }
        }
    }
    return w;
}

// Where the matrix starts on 16 bytes (AL), rows are accessed through a descriptor of the row's blocks.  Its bounds check replaces the
// branches (reads past the row's last 4 bytes give 0, writes there are dropped), and a piece's address is one 32-bit offset.  What a row's
// first and last block hold of its neighbours is read (it is part of the matrix, or of the last value's own 4 bytes) and not used.
template <class T>
__device__ __forceinline__ __amdgpu_buffer_rsrc_t row_buffer(const T* row, int V, const RowSpan& sp) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(row - sp.shift), 0, (int)(((sp.shift + V) * sizeof(T) + 3) & ~3u), 0x00020000);
}
// A word of a piece: values before `lo` and from `hi` on (counted from the word's first) become -inf.
template <class T>
__device__ __forceinline__ int keep_values(int w, int lo, int hi) {
    if constexpr (sizeof(T) == 4) return lo <= 0 && hi > 0 ? w : (int)0xff800000u;
    const uint32_t a = lo <= 0 && hi > 0 ? (uint32_t)w & 0xffffu : 0xff80u;
    const uint32_t b = lo <= 1 && hi > 1 ? (uint32_t)w & 0xffff0000u : 0xff800000u;
    return (int)(a | b);
}

template <class T> __device__ __forceinline__ void store_one(T* p, float v);
template <> __device__ __forceinline__ void store_one<uint16_t>(uint16_t* p, float v) { *p = (uint16_t)cvt_pk_bf16(v, v); }
template <> __device__ __forceinline__ void store_one<float>(float* p, float v) { *p = v; }

template <class T>
__device__ __forceinline__ void store_piece(T* row, int V, const RowSpan& sp, int i, const float* g, bool vec) {
    constexpr int PER = Elem<T>::PER;
    const int c0 = i * PER - sp.shift;
    if (vec && c0 >= 0 && c0 + PER <= V) {
        if constexpr (sizeof(T) == 2)
            *(v4i*)(row + c0) = (v4i){(int)cvt_pk_bf16(g[0], g[1]), (int)cvt_pk_bf16(g[2], g[3]), (int)cvt_pk_bf16(g[4], g[5]), (int)cvt_pk_bf16(g[6], g[7])};
        else
            *(v4f*)(row + c0) = (v4f){g[0], g[1], g[2], g[3]};
        return;
    }
    if (i >= sp.pieces) return;
#pragma unroll
    for (int e = 0; e < PER; ++e) {
        const int c = c0 + e;
        if (c >= 0 && c < V) store_one<T>(row + c, g[e]);
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

// One wave: everything about the listed columns that does not need the row's sum.
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

template <class T, int NCH, bool CAP, bool TAIL, int MODE, bool AL>
__global__ __launch_bounds__(kDistBlock, NCH * Elem<T>::PER > 16 ? 4 : 8) void distill_kernel(DistArgs a) {
    constexpr int PER = Elem<T>::PER;
    constexpr int N = NCH * PER;                        // values a thread holds
    constexpr int SEG = NCH * kDistThreads;             // pieces that one sweep over the registers covers
    constexpr float kLn2 = 0.6931471805599453f;
    // Three buffers: the list wave works a row ahead, and the others may be one barrier behind it.
    // A first row's lists are waited for only where they are used ahead of the row's own barrier.
    constexpr bool kListsFirst = TAIL || MODE == DIST_BWD;
    constexpr bool kAhead = N <= 16;                    // registers for a second sweep's loads
    __shared__ TopLds top[3];
    __shared__ double td[kDistMaxTop];
    __shared__ __attribute__((aligned(16))) float red_m[2][kDistWaves + 1], red_s[2][kDistWaves + 1];      // (the list wave's entry is an empty sum)
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int V = a.V;
    const int step = gridDim.x;

    if (wave == kDistWaves) {
        // ---- the wave of the listed columns ----
        if (lane < 2) {
            red_m[lane][kDistWaves] = -INFINITY;
            red_s[lane][kDistWaves] = 0.0f;
        }
        for (int i = lane; i < kDistThreads; i += 64) top[0].head[i] = top[1].head[i] = top[2].head[i] = -1;
        auto prepare = [&](int row, int buf) {
            if (row >= a.T) return;
            const T* lrow = (const T*)a.logits + (int64_t)row * a.ld;
            prepare_top<T, CAP, TAIL>(a, row, lrow, RowSpan(lrow, V).shift, top[buf], td, lane);
        };
        prepare(blockIdx.x, 0);
        if constexpr (kListsFirst) __syncthreads();
        int buf = 1;
        for (int row = blockIdx.x; row < a.T; row += step) {
            prepare(row + step, buf);
            buf = buf == 2 ? 0 : buf + 1;
            __syncthreads();
        }
        return;
    }

    // ---- the waves that hold the row ----
    // the cap is the largest z: no maximum is needed.  A value of -inf in place of one that is not summed adds exactly this:
    const float pad = CAP ? exp2_hw(-a.k2_up) : 0.0f;
    v4i raw[NCH];
    auto load_seg = [&](int row, int seg, v4i (&raw)[NCH]) {
        const T* const lrow = (const T*)a.logits + (int64_t)row * a.ld;
        int t = tid;
        asm volatile("" : "+v"(t));          // offsets are rebuilt here: kept across the row they would be spilled
        if constexpr (AL) {
            const auto buf = row_buffer(lrow, V, RowSpan(lrow, V));
#pragma unroll
            for (int s = 0; s < NCH; ++s) {
                const int i = seg * SEG + s * kDistThreads + t;
                raw[s] = __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(buf, i * 16, 0, 0));
            }
        } else {
            const RowSpan sp(lrow, V);
#pragma unroll
            for (int s = 0; s < NCH; ++s) raw[s] = load_piece<T>(lrow, V, sp, seg * SEG + s * kDistThreads + t);
        }
    };
    if ((int)blockIdx.x < a.T) load_seg(blockIdx.x, 0, raw);
    if constexpr (kListsFirst) __syncthreads();

    int par = 0, buf = 0;
    for (int row = blockIdx.x; row < a.T; row += step, par ^= 1, buf = buf == 2 ? 0 : buf + 1) {
        const RowSpan sp((const T*)a.logits + (int64_t)row * a.ld, V);
        TopLds& tp = top[buf];
        const float weight = a.weight ? a.weight[row] : 1.0f;
        float d[MODE == DIST_LOSS ? 1 : N];
        float m = CAP ? 1.0f : -INFINITY, S = 0.0f;         // reference, in units of z_arg, and the sum relative to it
        int skipped = 0;                                // values of this thread that are not summed
        const int segs = (sp.pieces + SEG - 1) / SEG;
        // Places outside the row in `count` of this thread's pieces, from piece `first` of the row on.  Counted behind the sweeps: across them
        // the count is a register more (4096 rows of 50304 fp32 fused: 387 against 429 us).  With the rest's mass, where the listed columns are
        // counted anyway, sweep by sweep and from the thread's own number (8192 rows of bf16 fused: 339 against 350).
        auto outside = [&](int first, int count) {
            int t = tid;
            if constexpr (!TAIL) asm volatile("" : "+v"(t));
            const int mine = max(0, min((sp.pieces - first - t + kDistThreads - 1) / kDistThreads, count));       // pieces that exist
            int n = PER * (count - mine);
            if (t == 0 && first == 0) n += sp.shift;
            if (mine > 0 && first + (mine - 1) * kDistThreads + t == sp.pieces - 1) n += sp.pieces * PER - sp.shift - V;
            return n;
        };
        // Exponentials of one sweep, relative to `m`, and (forward) their sum.  With the rest of the teacher's mass in play
        // the sum is over the columns that are not listed: those are set to -inf first.
        auto sweep = [&](int seg) {
            if constexpr (AL && MODE != DIST_BWD) {      // what was read outside the row
                constexpr int WORD = 4 / sizeof(T);
                int t = tid;
                asm volatile("" : "+v"(t));
                if (seg == 0 && wave == 0 && sp.shift > 0) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) raw[0][i] = t == 0 ? keep_values<T>(raw[0][i], sp.shift - i * WORD, WORD) : raw[0][i];
                }
#pragma unroll
                for (int s = 0; s < NCH; ++s)
                    if (seg * SEG + (s + 1) * kDistThreads >= sp.pieces) {       // the row's last piece, and none
                        const int left = V + sp.shift - (seg * SEG + s * kDistThreads + t) * PER;
#pragma unroll
                        for (int i = 0; i < 4; ++i) raw[s][i] = keep_values<T>(raw[s][i], 0, left - i * WORD);
                    }
            }
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
                    if constexpr (TAIL) skipped += outside(seg * SEG, NCH);
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
                const float ex = CAP && MODE != DIST_BWD ? exp2_hw(__builtin_fmaf(arg, a.k2, -a.k2_up)) : rel_exp<CAP>(arg, ref, a.k2);
                if constexpr (MODE != DIST_BWD) S += ex;
                if constexpr (MODE != DIST_LOSS) {
                    const float u = ex * arg;
                    d[i] = CAP ? __builtin_fmaf(-u, arg, u) : ex;
                    asm volatile("" : "+v"(d[i]));       // here and now: moved behind the barrier (as the sum's additions would be) it keeps two values alive
                }
                if (i % 8 == 7) {
                    asm volatile("" : "+v"(S));
                    __builtin_amdgcn_sched_barrier(0);      // eight chains at a time: more would not fit the registers
                }
            }
        };
        // Gradient of one sweep: f times what the thread holds; then the listed columns, from their own statistics, by the same
        // thread (its stores to one address stay in order).
        auto emit = [&](int seg, float f, float base, float ref, float inv_sum, bool none) {
            T* const grow = (T*)a.grad + (int64_t)row * a.ldg;
            int t = tid;
            asm volatile("" : "+v"(t));
            if constexpr (AL) {
                const auto buf = row_buffer(grow, V, sp);
                const bool ragged = (V + sp.shift) % PER != 0;
#pragma unroll
                for (int s = 0; s < NCH; ++s) {
#pragma unroll
                    for (int e = 0; e < PER; ++e) d[s * PER + e] = none ? 0.0f : d[s * PER + e] * f;
                    const float* g = &d[s * PER];
                    u32x4 w;
                    if constexpr (sizeof(T) == 2) w = (u32x4){cvt_pk_bf16(g[0], g[1]), cvt_pk_bf16(g[2], g[3]), cvt_pk_bf16(g[4], g[5]), cvt_pk_bf16(g[6], g[7])};
                    else w = (u32x4){__float_as_uint(g[0]), __float_as_uint(g[1]), __float_as_uint(g[2]), __float_as_uint(g[3])};
                    const int i = seg * SEG + s * kDistThreads + t;
                    // pieces that are the row's in part: out of bounds here, value by value below
                    const bool part = (i == 0 && sp.shift > 0) || (i == sp.pieces - 1 && ragged);
                    __builtin_amdgcn_raw_buffer_store_b128(w, buf, part ? 0x7ffffff0 : i * 16, 0, 0);
                }
#pragma unroll
                for (int s = 0; s < NCH; ++s) {
                    const int first = seg * SEG + s * kDistThreads;
                    if ((first == 0 && sp.shift > 0) || (ragged && first < sp.pieces && first + kDistThreads >= sp.pieces)) {
                        const int i = first + t;
                        if ((i == 0 && sp.shift > 0) || (i == sp.pieces - 1 && ragged)) {
#pragma unroll
                            for (int e = 0; e < PER; ++e) {
                                const int c = i * PER + e - sp.shift;
                                if (c >= 0 && c < V) store_one<T>(grow + c, d[s * PER + e]);
                            }
                        }
                    }
                }
            } else {
#pragma unroll
                for (int s = 0; s < NCH; ++s) {
                    float g[PER];
#pragma unroll
                    for (int e = 0; e < PER; ++e) g[e] = none ? 0.0f : d[s * PER + e] * f;
                    store_piece<T>(grow, V, sp, seg * SEG + s * kDistThreads + t, g, a.vec_grad != 0);
                }
            }
            if (!none)
                for_listed<NCH, PER>(tp, tid, seg, [&](int e, int) {
                    const float arg = tp.arg[e];
                    const float q = rel_exp<CAP>(arg, ref, a.k2) * inv_sum;
                    store_one<T>(grow + (tp.pos[e] - sp.shift), base * (q * (tp.sum_p + tp.rest_p) - tp.p[e]) * (CAP ? arg * (1.0f - arg) : 1.0f));
                });
        };

        // The sweep behind this one, of this row or of the next: requested before this one is worked on.
        auto load_ahead = [&](int seg, v4i (&next)[NCH]) {
            if (MODE != DIST_FUSED && seg + 1 < segs) load_seg(row, seg + 1, next);
            else if (row + step < a.T) load_seg(row + step, 0, next);
        };
        auto take = [&](const v4i (&next)[NCH]) {
#pragma unroll
            for (int s = 0; s < NCH; ++s) raw[s] = next[s];
        };

        if constexpr (MODE == DIST_BWD) {
            const StatRow st = ((const StatRow*)a.stats)[row];
            const float base = weight * a.dloss[(int64_t)row * a.dloss_st] * a.tau * a.slope;
            const bool none = tp.any == 0 || weight == 0.0f;
            m = st.ref;
            for (int seg = 0; seg < segs; ++seg) {
                v4i next[NCH];
                load_ahead(seg, next);
                sweep(seg);
                emit(seg, base * st.inv_sum * (tp.sum_p + tp.rest_p - st.rest_ratio), base, st.ref, st.inv_sum, none);
                take(next);
            }
            tp.head[tid] = -1;
            __syncthreads();
        } else {
            if constexpr (MODE == DIST_LOSS && kAhead) {
                for (int seg = 0; seg < segs; ++seg) {
                    v4i next[NCH];
                    load_ahead(seg, next);
                    sweep(seg);
                    take(next);
                }
            } else {
                for (int seg = 0; seg < (MODE == DIST_LOSS ? segs : 1); ++seg) {
                    sweep(seg);
                    load_ahead(seg, raw);        // in flight while this row is reduced and written
                }
            }
            if constexpr (CAP) {
                if constexpr (!TAIL) skipped = outside(0, segs * NCH);
                S = __builtin_fmaf(-(float)skipped, pad, S) * a.from_up;
            }
            const float wm = CAP ? m : wave_max(m);
            const float ws = wave_sum(rescale(S, m, wm, a.k2));
            if (lane == 0) {
                red_m[par][wave] = wm;
                red_s[par][wave] = ws;
            }
            __syncthreads();
            // four waves at a time: the values of the row fill the registers
            static_assert((kDistWaves + 1) % 4 == 0, "whole quadruples");
            float M = m;
            if constexpr (!CAP) {
                M = -INFINITY;
#pragma unroll 1
                for (int w = 0; w < kDistWaves + 1; w += 4) {
                    const v4f x = *(const v4f*)&red_m[par][w];
                    M = fmaxf(M, fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])));
                }
            }
            float sum = 0.0f;
#pragma unroll 1
            for (int w = 0; w < kDistWaves + 1; w += 4) {
                const v4f x = *(const v4f*)&red_m[par][w], y = *(const v4f*)&red_s[par][w];
#pragma unroll
                for (int q = 0; q < 4; ++q) sum += CAP ? y[q] : rescale(y[q], x[q], M, a.k2);
            }
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
                emit(0, base * inv_sum * (CAP ? a.from_up : rescale(1.0f, m, M, a.k2)) * (tp.sum_p + tp.rest_p - rest_ratio), base, M, inv_sum, none);
            }
            tp.head[tid] = -1;      // filled again three rows on, two barriers from here
        }
    }
}

template <class T, int NCH, bool CAP, bool TAIL, int MODE>
int launch_distill(const DistArgs& a, hipStream_t st) {
    const int cus = num_cus();
    if (cus <= 0) return fail(NGPT_EINVAL, "no HIP device");
    const int resident = cus * (NCH * Elem<T>::PER > 16 ? 1 : 2);
    const int grid = a.T < resident ? a.T : resident;
    if (((uintptr_t)a.logits & 15) == 0 && (MODE == DIST_LOSS || a.vec_grad))
        distill_kernel<T, NCH, CAP, TAIL, MODE, true><<<grid, kDistBlock, 0, st>>>(a);
    else
        distill_kernel<T, NCH, CAP, TAIL, MODE, false><<<grid, kDistBlock, 0, st>>>(a);
    return check_launch("distill_kernel");
}

// Pieces of a row that starts anywhere: one more than the aligned count.
template <class T> int most_pieces(int V) { return V / Elem<T>::PER + 2; }

template <class T, bool CAP, bool TAIL>
int run_distill(const DistArgs& a, int mode, hipStream_t st) {
    constexpr int BIG = sizeof(T) == 2 ? 7 : 14;        // pieces a thread: 56 values
    // Loss or gradient alone: two workgroups a compute unit in short sweeps; with no more rows than compute units a row's whole
    // latency counts, and the wide sweep has all of the row in flight at once.
    const bool few = a.T <= num_cus();
    if (mode == DIST_LOSS) return few ? launch_distill<T, BIG, CAP, TAIL, DIST_LOSS>(a, st) : launch_distill<T, 16 / Elem<T>::PER, CAP, TAIL, DIST_LOSS>(a, st);
    if (mode == DIST_BWD) return launch_distill<T, 16 / Elem<T>::PER, CAP, TAIL, DIST_BWD>(a, st);
    // the row in registers: 16, 32 or 56 values a thread
    const int pieces = most_pieces<T>(a.V);
    if (pieces <= 16 / Elem<T>::PER * kDistThreads) return launch_distill<T, 16 / Elem<T>::PER, CAP, TAIL, DIST_FUSED>(a, st);
    if (pieces <= 32 / Elem<T>::PER * kDistThreads) return launch_distill<T, 32 / Elem<T>::PER, CAP, TAIL, DIST_FUSED>(a, st);
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
    if (T > (1 << 30)) return fail(NGPT_ERANGE, "%s: %d rows, at most 2^30", who, T);
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
        a.k2_up = std::ceil(a.k2);
        a.from_up = (float)std::exp2((double)a.k2_up - (double)a.k2);
        a.slope = A / C;
        if (a.k1 == 0.0f || !std::isfinite(a.k1) || !std::isfinite(a.k0) || !std::isfinite(a.slope))
            return fail(NGPT_ERANGE, "%s: softcap A=%g B=%g C=%g: 1 / C, B / C or A / C outside 32-bit floats", who, (double)A, (double)B, (double)C);
    }
    // (0 times an infinite 1 / temperature would be NaN for the largest logit)
    if (!std::isfinite(a.k2)) return fail(NGPT_ERANGE, "%s: temperature %g: its reciprocal is not a 32-bit float", who, (double)tau);
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
