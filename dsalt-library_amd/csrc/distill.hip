// Loss of a student's logits s [rows, V] against a teacher's top logits z [rows, K] at token ids, and
// against labels, with its gradient. Per row, with p = softmax(z / tau) over the row's slots and
// q = softmax(s / tau), q1 = softmax(s) over the vocabulary:
//   loss = (1 - lam) tau^2 sum_k p_k (ln p_k - ln q[id_k]) - lam ln q1[label]
//   d s  = (1 - lam) tau (q - sum_k p_k e[id_k]) + lam (q1 - e[label])
// A slot counts where its id lies in [0, V) and its logit is not -inf; a row without slots has no first
// term. Rows whose label is ignore_index (or lies outside [0, V)) count for nothing; the mean is over
// the others.
//
// The forward reads the logits once with running maxima and sums: exponents are fma(s, c, -m c), c =
// log2(e) / tau, in the forward and in the backward. What the rounding of m c left is the exponent at s = m; sums that
// go on to another maximum leave theirs behind, and it drops out of every quotient. From |m c| = 2^16 on (a
// mask that leaves nothing: the residue is 2^-24 of m c, and of a mask of -1e10 its power is no longer finite)
// exponents are (s - m) c. At tau = 2 the exponential at 1 is the square of that at tau. It keeps m and the sums'
// inverses of each row, and the backward reads the logits once more and writes the gradient, each rounded
// once from fp32 under the upstream gradient that it is given (formed in the forward it would be rounded
// before a loss scale is known, which in fp16 loses most of a vocabulary's small probabilities).
//
// Rows of up to 4096 logits take one wave, longer ones four; few long rows are cut into slices whose
// sums a second kernel joins, but for a lone one, which sixteen waves take. Long rows are bound by HBM bytes:
// 6473 x 32000 bf16 at tau = 2 with labels, 88 us forward (4.7 TB/s; 126 right behind a backward, whose gradients
// still drain) and 155-201 us backward (5.3-4.1 TB/s: what the forward left in the last-level cache counts); at
// tau = 1.5, with two exponentials a logit, 98 and 201 us; fp32 146 and 378 us. A
// loop that loaded a run only behind the last one's sums took 124 us. Short rows are bound by what a row
// costs beside its logits, the label, the slots and a wave's joins: 60000 x 1500 88 and 133 us.
#include "launch.h"
#include "lanes.h"
#include "rotary.h"

#include <algorithm>

namespace dsalt {
namespace {

constexpr int kStats = 5;         // of a row: m, 1 / sum at tau, 1 / sum at 1, the teacher's m, 1 / the teacher's sum
// Logits of a row that one wave takes. One wave and four, in us: 16384 x 2100 bf16 36 and 56 forward, 50 and 61
// backward; 16384 x 4000 47 and 62, 77 and 77; 8000 x 8000 39 and 39, 69 and 61.
constexpr int kRowMax = 4096;
// Logits of a lone row that one workgroup of 16 waves takes and ends by itself, with its reduction; beyond, slices and
// their join. us of each: 5000 bf16 4.2 and 6.5, 32000 5.8 and 6.7, 50257 6.2 and 6.6, 100003 8.2 and 6.9.
constexpr int kLoneMax = 65536;
constexpr int kSlice = 2048;      // least logits of a slice
constexpr int kSliceGroups = 1024;  // workgroups that slices are made for

struct DistillParams {
    const void *logits, *teacher, *ids, *labels;
    int64_t rows, logits_stride, teacher_stride, ids_stride, ignore_index;
    int vocab, k, teacher_dtype, ids64, labels64, splits;
    float c, inv_tau, kl_w, lam;  // kl_w = (1 - lam) tau^2
    float *part;                  // [rows][splits][3]
    float *row_loss, *stats;
    float *loss;                  // of a reduction
    int mean, reduce;
    int lone;  // the reduction of one row, which is its loss
    const float *d_loss;
    void *d_logits;
    float grad_w;  // (1 - lam) tau
};

template <typename DT>
__device__ __forceinline__ constexpr int elem_size() { return std::is_same<DT, F32>::value ? 4 : 2; }
template <typename DT>
struct Vec {
    static constexpr int N = 16 / elem_size<DT>();
    __device__ static __forceinline__ void get(uint4 u, float *f) {
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if constexpr (std::is_same<DT, F32>::value) f[e] = __uint_as_float(w[e]);
            else {
                f[2 * e] = DT::lo_f32(w[e]);
                f[2 * e + 1] = DT::hi_f32(w[e]);
            }
        }
    }
    __device__ static __forceinline__ uint4 put(const float *f) {
        if constexpr (std::is_same<DT, F32>::value)
            return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
        else return make_uint4(DT::pack2(f[0], f[1]), DT::pack2(f[2], f[3]), DT::pack2(f[4], f[5]), DT::pack2(f[6], f[7]));
    }
};

__device__ __forceinline__ float wave_maxf(float x) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) x = fmaxf(x, __shfl_xor(x, o));
    return x;
}
__device__ __forceinline__ float wave_maximum(float x) {  // NaN stays
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) x = __builtin_elementwise_maximum(x, __shfl_xor(x, o));
    return x;
}
// Which exponentials a logit has: at tau, also at 1, or at 1 as the square of that at tau = 2.
enum { kOne = 0, kTwo = 1, kSquare = 2 };

// A maximum as a reference for exp2 (of nothing but -inf any finite one will do), and exponents against it.
struct Reference {
    float m, mc, mc1;
    bool far;  // m c is too large for its residue
    __device__ __forceinline__ Reference(float max, float c) : m(max == -INFINITY ? 0.f : max), mc(m * c), mc1(m * kLog2e) {
        far = !(fmaxf(fabsf(mc), fabsf(mc1)) < 65536.f);
    }
    __device__ __forceinline__ float at(float v, float c) const { return far ? (v - m) * c : fmaf(v, c, -mc); }
    __device__ __forceinline__ float at1(float v) const { return far ? (v - m) * kLog2e : fmaf(v, kLog2e, -mc1); }
    // the exponents that take sums against the maximum `max` to this reference
    __device__ __forceinline__ float from(float max, float c) const {
        const Reference o(max, c);
        return at(max, c) - o.at(o.m, c);
    }
    __device__ __forceinline__ float from1(float max, float c) const {
        const Reference o(max, c);
        return at1(max) - o.at1(o.m);
    }
    // the exponent at temperature 1
    template <int KIND>
    __device__ __forceinline__ float label(float v, float c) const {
        return KIND == kTwo ? at1(v) : KIND == kSquare ? 2.f * at(v, c) : at(v, c);
    }
};

// Running maximum and sums of the exponentials.
template <int KIND>
struct Running {
    float m = -INFINITY, s = 0.f, s1 = 0.f;
    __device__ __forceinline__ void rescale(float mn, float c) {
        const Reference r(mn, c);
        const float t = fast_exp2(r.from(m, c));
        s *= t;
        if (KIND == kTwo) s1 *= fast_exp2(r.from1(m, c));
        if (KIND == kSquare) s1 *= t * t;
        m = mn;
    }
    template <int N>
    __device__ __forceinline__ void add(const float (&v)[N], float c) {
        float mn = m;  // NaN stays: the row is NaN then
#pragma unroll
        for (int i = 0; i + 1 < N; i += 2) mn = max3f(mn, v[i], v[i + 1]);
        if (N % 2) mn = __builtin_elementwise_maximum(mn, v[N - 1]);
        if (mn != m) rescale(mn, c);
        const Reference r(m, c);
        float t = 0.f, t1 = 0.f;
        if (!r.far) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float x = fast_exp2(fmaf(v[i], c, -r.mc));
                t += x;
                if (KIND == kTwo) t1 += fast_exp2(fmaf(v[i], kLog2e, -r.mc1));
                if (KIND == kSquare) t1 = fmaf(x, x, t1);
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float x = fast_exp2(r.at(v[i], c));
                t += x;
                if (KIND == kTwo) t1 += fast_exp2(r.at1(v[i]));
                if (KIND == kSquare) t1 = fmaf(x, x, t1);
            }
        }
        s += t;
        if (KIND != kOne) s1 += t1;
    }
    __device__ __forceinline__ void join(float m2, float t, float t1, float c) {
        rescale(__builtin_elementwise_maximum(m, m2), c);
        const Reference r(m, c);
        const float x = fast_exp2(r.from(m2, c));
        s += t * x;
        if (KIND == kTwo) s1 += t1 * fast_exp2(r.from1(m2, c));
        if (KIND == kSquare) s1 += t1 * (x * x);
    }
    __device__ __forceinline__ void join_wave(float c) {
        rescale(wave_maximum(m), c);
        s = group_sum_lanes(s, 64);
        if (KIND != kOne) s1 = group_sum_lanes(s1, 64);
    }
};

__device__ __forceinline__ int64_t load_int(const void *p, int64_t i, int is64) {
    return is64 ? static_cast<const int64_t *>(p)[i] : static_cast<const int32_t *>(p)[i];
}
// The row's label; -1: the row does not count; vocab: rows are not labelled.
__device__ __forceinline__ int row_label(const DistillParams &p, int64_t row) {
    if (!p.labels) return p.vocab;
    const int64_t l = load_int(p.labels, row, p.labels64);
    return l == p.ignore_index || l < 0 || l >= p.vocab ? -1 : (int)l;
}
// Slot k's logit, -inf where the slot does not count, and its id.
__device__ __forceinline__ float slot(const DistillParams &p, int64_t row, int k, int &id) {
    const int64_t i = load_int(p.ids, row * p.ids_stride + k, p.ids64);
    id = i >= 0 && i < p.vocab ? (int)i : -1;
    if (id < 0) return -INFINITY;
    const int64_t at = row * p.teacher_stride + k;
    const float z = p.teacher_dtype == DSALT_DTYPE_F32    ? Elem<F32>::ld(p.teacher, at)
                    : p.teacher_dtype == DSALT_DTYPE_BF16 ? Elem<BF16>::ld(p.teacher, at)
                                                          : Elem<F16>::ld(p.teacher, at);
    if (z == -INFINITY) id = -1;
    return z;
}

// What a row's end needs of memory, read before the row itself: its label, and the lane's first slot.
template <typename DT>
struct RowEnd {
    int label, id = -1;
    float t = -INFINITY, at_id = 0.f, at_label = 0.f;  // the slot's logit; the student's at the id and at the label
    __device__ __forceinline__ RowEnd(const DistillParams &p, int64_t row, int lane, bool ends = true) : label(ends ? row_label(p, row) : -1) {
        const char *logits = static_cast<const char *>(p.logits) + row * p.logits_stride * elem_size<DT>();
        if (label < 0) return;
        if (p.kl_w != 0.f && lane < p.k) t = slot(p, row, lane, id);
        if (id >= 0) at_id = Elem<DT>::ld(logits, id);
        if (p.lam != 0.f) at_label = Elem<DT>::ld(logits, label);
    }
};

// A row's loss and statistics from its maximum and sums, by one wave.
template <typename DT, int KIND>
__device__ __forceinline__ void finish_row(const DistillParams &p, int64_t row, const Running<KIND> &run, const RowEnd<DT> &end,
                                           int lane) {
    const int label = end.label;
    const Reference ref(run.m, p.c);
    const float s1 = KIND == kOne ? run.s : run.s1;
    const char *logits = static_cast<const char *>(p.logits) + row * p.logits_stride * elem_size<DT>();
    float tm = -INFINITY, ts = 0.f, kl = 0.f;
    if (p.kl_w != 0.f && label >= 0) {
        int id;
        tm = end.t;
        for (int k = 64 + lane; k < p.k; k += 64) tm = fmaxf(tm, slot(p, row, k, id));
        tm = wave_maxf(tm);
        if (tm == -INFINITY) tm = 0.f;
        // over tau behind the difference: over a tau below 1 the type's lowest value has no finite quotient
        const auto exponent = [&](float t) { return (t - tm) * p.inv_tau; };
        bool any = end.id >= 0;
        ts = end.id >= 0 ? expf(exponent(end.t)) : 0.f;
        for (int k = 64 + lane; k < p.k; k += 64) {
            const float t = slot(p, row, k, id);
            any |= id >= 0;
            ts += id >= 0 ? expf(exponent(t)) : 0.f;
        }
        ts = group_sum_lanes(ts, 64);
        if (__ballot(any)) {
            const float lt = logf(ts), ls = log2f(run.s);
            const auto term = [&](float t, float v) {
                const float lp = exponent(t) - lt, w = expf(exponent(t)) / ts;
                const float lq = (ref.at(v, p.c) - ls) * kLn2;
                return w != 0.f ? w * (lp - lq) : 0.f;
            };
            if (end.id >= 0) kl = term(end.t, end.at_id);
            for (int k = 64 + lane; k < p.k; k += 64) {
                const float t = slot(p, row, k, id);
                if (id >= 0) kl += term(t, Elem<DT>::ld(logits, id));
            }
            kl = group_sum_lanes(kl, 64);
        }
    }
    if (lane) return;
    float loss = p.kl_w * kl;
    if (p.lam != 0.f && label >= 0)
        loss += p.lam * (log2f(s1) - ref.template label<KIND>(end.at_label, p.c)) * kLn2;
    p.row_loss[row] = label < 0 ? 0.f : loss;
    if (p.stats) {
        if (p.lone) p.stats[kStats] = 1.f;
        float *st = p.stats + row * kStats;
        st[0] = ref.m;
        st[1] = 1.f / run.s;
        st[2] = 1.f / s1;
        st[3] = tm;
        st[4] = ts == 0.f ? 0.f : 1.f / ts;  // 0: the row has no teacher
    }
}

// The elements of a slice [first, last) of a row as the lanes take them: 16-byte vectors between the
// first and the last 16-byte boundary, and single elements before and behind.
struct Span {
    int head, vecs, tail_at, tail;
    template <typename DT>
    __device__ __forceinline__ static Span of(const char *row, int first, int last) {
        constexpr int VE = Vec<DT>::N;
        Span s;
        const uintptr_t a = (uintptr_t)(row + (int64_t)first * elem_size<DT>());
        s.head = min((int)(((16 - (a & 15)) & 15) / elem_size<DT>()), last - first);
        s.vecs = (last - first - s.head) / VE;
        s.tail_at = first + s.head + s.vecs * VE;
        s.tail = last - s.tail_at;
        return s;
    }
};
__device__ __forceinline__ void slice_of(const DistillParams &p, int split, int &first, int &last) {
    const int per = (p.vocab + p.splits - 1) / p.splits;
    first = min(split * per, p.vocab);
    last = min(first + per, p.vocab);
}

// NW waves a row (or slice), of a workgroup of at least four.
template <typename DT, int KIND, int NW>
__global__ void __launch_bounds__(NW > 4 ? NW * 64 : 256) distill_rows_kernel(const DistillParams p) {
    constexpr int VE = Vec<DT>::N, NT = NW * 64, U = NW > 4 ? 4 : 32 / VE;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int64_t item = NW == 1 ? (int64_t)blockIdx.x * 4 + wave : blockIdx.x;
    const int64_t row = item / p.splits;
    const int split = (int)(item - row * p.splits);
    if (row >= p.rows) return;  // a whole wave (NW = 1); never with more
    const int t = NW == 1 ? lane : threadIdx.x;
    const char *base = static_cast<const char *>(p.logits) + row * p.logits_stride * elem_size<DT>();
    int first, last;
    slice_of(p, split, first, last);
    const Span sp = Span::of<DT>(base, first, last);
    const uint4 *body = reinterpret_cast<const uint4 *>(base + (int64_t)(first + sp.head) * elem_size<DT>());
    // whole runs of U vectors a lane, the next one's loads before this one's sums; what is left is loaded ahead
    const int runs = sp.vecs / (NT * U);
    uint4 u[U], rest[U];
    const uint4 *at = body + t;
    if (runs)
#pragma unroll
        for (int j = 0; j < U; ++j) u[j] = at[j * NT];
    const RowEnd<DT> end(p, row, lane, p.splits == 1);  // a split's row is ended by the join
    Running<KIND> run;
    if (t < sp.head + sp.tail) {
        const float v[1] = {Elem<DT>::ld(base, t < sp.head ? first + t : sp.tail_at + t - sp.head)};
        run.add(v, p.c);
    }
    const int behind = sp.vecs - runs * NT * U;
#pragma unroll
    for (int j = 0; j < U; ++j)
        if (j * NT + t < behind) rest[j] = body[runs * NT * U + j * NT + t];
    for (int i = 0; i < runs; ++i) {
        at += NT * U;
        uint4 next[U];
        if (i + 1 < runs)
#pragma unroll
            for (int j = 0; j < U; ++j) next[j] = at[j * NT];
        float v[U * VE];
#pragma unroll
        for (int j = 0; j < U; ++j) Vec<DT>::get(u[j], v + j * VE);
        run.add(v, p.c);
#pragma unroll
        for (int j = 0; j < U; ++j) u[j] = next[j];
    }
#pragma unroll
    for (int j = 0; j < U; ++j)
        if (j * NT + t < behind) {
            float v[VE];
            Vec<DT>::get(rest[j], v);
            run.add(v, p.c);
        }
    run.join_wave(p.c);
    if constexpr (NW > 1) {
        __shared__ float lds[NW][3];
        if (lane == 0) {
            lds[wave][0] = run.m;
            lds[wave][1] = run.s;
            lds[wave][2] = run.s1;
        }
        __syncthreads();
        if (wave) return;
        run = Running<KIND>();
        if (lane < NW) {
            run.m = lds[lane][0];
            run.s = lds[lane][1];
            run.s1 = lds[lane][2];
        }
        run.join_wave(p.c);
    }
    if (p.splits == 1) return finish_row<DT, KIND>(p, row, run, end, lane);
    if (lane == 0) {
        float *out = p.part + item * 3;
        out[0] = run.m;
        out[1] = run.s;
        out[2] = run.s1;
    }
}

// Sum of the rows' losses, over the number that count for a mean: 16 waves of one workgroup.
__device__ __forceinline__ void reduce_rows(const DistillParams &p, float *lds) {
    float sum = 0.f;
    int count = 0;
    for (int64_t r = threadIdx.x; r < p.rows; r += 1024) {
        sum += p.row_loss[r];
        count += row_label(p, r) >= 0;
    }
    sum = group_sum_lanes(sum, 64);
    count = wave_sum(count);
    if ((threadIdx.x & 63) == 0) {
        lds[threadIdx.x >> 6] = sum;
        lds[16 + (threadIdx.x >> 6)] = __int_as_float(count);
    }
    __syncthreads();
    if (threadIdx.x) return;
    sum = 0.f;
    count = 0;
    for (int w = 0; w < 16; ++w) {
        sum += lds[w];
        count += __float_as_int(lds[16 + w]);
    }
    const float n = p.mean ? (float)max(count, 1) : 1.f;
    *p.loss = sum / n;
    if (p.stats) p.stats[p.rows * kStats] = 1.f / n;
}

// Rows joined from their slices, a wave each; a lone workgroup also forms their sum.
template <typename DT, int KIND>
__global__ void __launch_bounds__(1024) distill_join_kernel(const DistillParams p) {
    __shared__ float lds[32];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t row = (int64_t)blockIdx.x * 16 + wave;
    if (row < p.rows) {
        const RowEnd<DT> end(p, row, lane);
        Running<KIND> run;
        const float *in = p.part + row * p.splits * 3;
        for (int i = lane; i < p.splits; i += 64) run.join(in[i * 3], in[i * 3 + 1], in[i * 3 + 2], p.c);
        run.join_wave(p.c);
        finish_row<DT, KIND>(p, row, run, end, lane);
    }
    if (gridDim.x == 1 && p.reduce) {
        __syncthreads();
        reduce_rows(p, lds);
    }
}

__global__ void __launch_bounds__(1024) distill_reduce_kernel(const DistillParams p) {
    __shared__ float lds[32];
    reduce_rows(p, lds);
}

// The gradient of a row (or slice): over the vocabulary first, then again at the teacher's ids and the
// label, whose values are formed whole (ids that repeat take the sum of their slots).
template <typename DT, int KIND, int NW>
__global__ void __launch_bounds__(256) distill_bwd_kernel(const DistillParams p) {
    constexpr int VE = Vec<DT>::N, NT = NW * 64, U = 4;
    extern __shared__ char dyn[];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int64_t item = (int64_t)blockIdx.x * (4 / NW) + (NW == 1 ? wave : 0);
    const int64_t row = item / p.splits;
    const int split = (int)(item - row * p.splits);
    const bool live = row < p.rows;  // dead waves keep the barriers
    const int t = NW == 1 ? lane : threadIdx.x;
    int *id = reinterpret_cast<int *>(dyn) + (NW == 1 ? wave : 0) * 2 * p.k;
    float *w = reinterpret_cast<float *>(id + p.k);
    const int label = live ? row_label(p, row) : -1;
    const char *base = static_cast<const char *>(p.logits) + row * p.logits_stride * elem_size<DT>();
    char *out = static_cast<char *>(p.d_logits) + row * p.vocab * elem_size<DT>();
    int first = 0, last = 0;
    if (live) slice_of(p, split, first, last);
    const Span sp = Span::of<DT>(base, first, last);
    const uint4 *body = reinterpret_cast<const uint4 *>(base + (int64_t)(first + sp.head) * elem_size<DT>());
    uint4 u[U];  // the first run's loads, ahead of what the row's statistics take
    if (label >= 0)
#pragma unroll
        for (int j = 0; j < U; ++j)
            if (t + j * NT < sp.vecs) u[j] = body[t + j * NT];
    int id0 = -1;
    float z0 = 0.f;
    if (label >= 0 && p.grad_w != 0.f && t < p.k) z0 = slot(p, row, t, id0);
    float m = 0.f, k0 = 0.f, k1 = 0.f, up = 0.f, kl = 0.f;
    if (label >= 0) {
        const float *st = p.stats + row * kStats;
        m = st[0];
        up = p.reduce ? *p.d_loss * p.stats[p.rows * kStats] : p.d_loss[row];
        kl = st[4] != 0.f ? up * p.grad_w : 0.f;
        k0 = kl * st[1];
        if (KIND != kOne) k1 = up * p.lam * st[2];
        else k0 += up * p.lam * st[2];
        if (kl != 0.f)  // the teacher's probabilities
            for (int k = t; k < p.k; k += NT) {
                int i = id0;
                const float z = k == t ? z0 : slot(p, row, k, i);
                id[k] = i;
                w[k] = i >= 0 ? expf((z - st[3]) * p.inv_tau) * st[4] : 0.f;
            }
    }
    const Reference ref(m, p.c);
    const auto value = [&](float v) {
        const float x = fast_exp2(ref.at(v, p.c));
        float g = k0 * x;
        if (KIND == kTwo) g = fmaf(k1, fast_exp2(ref.at1(v)), g);
        if (KIND == kSquare) g = fmaf(k1 * x, x, g);
        return g;
    };
    if (live && (label < 0 || (k0 == 0.f && k1 == 0.f))) {  // nothing of the row counts: zeros, whatever it holds
        for (int i = first + t; i < last; i += NT) Elem<DT>::st(out, i, 0.f);
    } else if (live) {
        if (t < sp.head + sp.tail) {
            const int i = t < sp.head ? first + t : sp.tail_at + t - sp.head;
            Elem<DT>::st(out, i, value(Elem<DT>::ld(base, i)));
        }
        const int at = first + sp.head;
        char *dst = out + (int64_t)at * elem_size<DT>();
        const bool whole = ((uintptr_t)dst & 15) == 0;  // else the gradient's rows lie otherwise than the logits'
        for (int i = t; i < sp.vecs; i += NT * U) {
            uint4 next[U];
#pragma unroll
            for (int j = 0; j < U; ++j)
                if (i + (U + j) * NT < sp.vecs) next[j] = body[i + (U + j) * NT];
#pragma unroll
            for (int j = 0; j < U; ++j) {
                const int at_vec = i + j * NT;
                if (at_vec >= sp.vecs) continue;
                float v[VE];
                Vec<DT>::get(u[j], v);
#pragma unroll
                for (int e = 0; e < VE; ++e) v[e] = value(v[e]);
                if (whole) reinterpret_cast<uint4 *>(dst)[at_vec] = Vec<DT>::put(v);
                else
#pragma unroll
                    for (int e = 0; e < VE; ++e) Elem<DT>::st(dst, at_vec * VE + e, v[e]);
            }
#pragma unroll
            for (int j = 0; j < U; ++j) u[j] = next[j];
        }
    }
    __syncthreads();  // the slots are in LDS, and the row's stores precede those that follow
    if (label < 0) return;
    const float one = up * p.lam;
    if (kl != 0.f)
        for (int k = t; k < p.k; k += NT) {
            const int i = id[k];
            if (i < first || i >= last) continue;
            float sum = 0.f;
            bool again = false;  // an earlier slot has this id and writes it
            for (int j = 0; j < p.k; ++j)
                if (id[j] == i) {
                    again |= j < k;
                    sum += w[j];
                }
            if (again) continue;
            Elem<DT>::st(out, i, value(Elem<DT>::ld(base, i)) - kl * sum - (i == label ? one : 0.f));
        }
    if (p.lam != 0.f && t == 0 && label >= first && label < last) {
        bool slotted = false;
        if (kl != 0.f)
            for (int j = 0; j < p.k; ++j) slotted |= id[j] == label;
        if (!slotted) Elem<DT>::st(out, label, value(Elem<DT>::ld(base, label)) - one);
    }
}

int distill_splits(int64_t rows, int vocab, bool bwd) {
    if (vocab <= kRowMax || rows <= 0 || (rows == 1 && !bwd && vocab <= kLoneMax)) return 1;
    const int64_t most = (vocab + kSlice - 1) / kSlice;
    return (int)std::max<int64_t>(1, std::min<int64_t>(most, kSliceGroups / rows));
}

DistillParams params(const dsalt_distill_args &a, bool bwd) {
    DistillParams p = {};
    p.logits = a.logits;
    p.teacher = a.teacher;
    p.ids = a.ids;
    p.labels = a.labels;
    p.rows = a.rows;
    p.logits_stride = a.logits_stride;
    p.teacher_stride = a.teacher_stride;
    p.ids_stride = a.ids_stride;
    p.ignore_index = a.ignore_index;
    p.vocab = a.vocab;
    p.k = a.k;
    p.teacher_dtype = a.teacher_dtype;
    p.ids64 = a.ids_int64;
    p.labels64 = a.labels_int64;
    p.splits = distill_splits(a.rows, a.vocab, bwd);
    const bool only_labels = a.label_weight == 1.f;  // then everything is at temperature 1
    p.inv_tau = only_labels ? 1.f : (float)(1.0 / (double)a.temperature);
    p.c = only_labels ? kLog2e : (float)(1.4426950408889634 / (double)a.temperature);
    p.lam = a.label_weight;
    p.kl_w = (1.f - a.label_weight) * a.temperature * a.temperature;
    p.grad_w = (1.f - a.label_weight) * a.temperature;
    p.stats = a.stats;
    p.loss = a.loss;
    p.reduce = a.reduction != DSALT_REDUCE_NONE;
    p.mean = a.reduction == DSALT_REDUCE_MEAN;
    p.lone = a.rows == 1 && p.splits == 1 && p.reduce;
    p.row_loss = p.reduce && !p.lone ? static_cast<float *>(a.workspace) : a.loss;
    p.part = static_cast<float *>(a.workspace) + (p.reduce ? a.rows : 0);
    p.d_loss = a.d_loss;
    p.d_logits = a.d_logits;
    return p;
}

template <typename DT, int KIND>
void launch_types(const DistillParams &p, bool bwd, hipStream_t stream) {
    const bool one_wave = p.vocab <= kRowMax;
    const dim3 grid((unsigned)(one_wave ? (p.rows + 3) / 4 : p.rows * p.splits)), block(256);
    const size_t lds = (size_t)(one_wave ? 4 : 1) * p.k * 8;
    if (bwd) {
        if (one_wave) hipLaunchKernelGGL((distill_bwd_kernel<DT, KIND, 1>), grid, block, lds, stream, p);
        else hipLaunchKernelGGL((distill_bwd_kernel<DT, KIND, 4>), grid, block, lds, stream, p);
        return;
    }
    if (one_wave) hipLaunchKernelGGL((distill_rows_kernel<DT, KIND, 1>), grid, block, 0, stream, p);
    else if (p.rows == 1 && p.splits == 1) hipLaunchKernelGGL((distill_rows_kernel<DT, KIND, 16>), grid, dim3(1024), 0, stream, p);
    else hipLaunchKernelGGL((distill_rows_kernel<DT, KIND, 4>), grid, block, 0, stream, p);
    const unsigned joins = (unsigned)((p.rows + 15) / 16);
    if (p.splits > 1) hipLaunchKernelGGL((distill_join_kernel<DT, KIND>), dim3(joins), dim3(1024), 0, stream, p);
    if (p.reduce && !p.lone && !(p.splits > 1 && joins == 1))
        hipLaunchKernelGGL(distill_reduce_kernel, dim3(1), dim3(1024), 0, stream, p);
}

hipError_t launch(const dsalt_distill_args &a, bool bwd, hipStream_t stream) {
    const DistillParams p = params(a, bwd);
    if (a.rows == 0) {
        if (!bwd && p.reduce) hipLaunchKernelGGL(distill_reduce_kernel, dim3(1), dim3(1024), 0, stream, p);
        return hipGetLastError();
    }
    const bool two = a.label_weight != 0.f && a.label_weight != 1.f && a.temperature != 1.f;
    const auto go = [&](auto dt) {
        if (!two) launch_types<decltype(dt), kOne>(p, bwd, stream);
        else if (a.temperature == 2.f) launch_types<decltype(dt), kSquare>(p, bwd, stream);
        else launch_types<decltype(dt), kTwo>(p, bwd, stream);
    };
    if (a.logits_dtype == DSALT_DTYPE_BF16) go(BF16());
    else if (a.logits_dtype == DSALT_DTYPE_F16) go(F16());
    else go(F32());
    return hipGetLastError();
}

}  // namespace

int64_t distill_workspace_bytes(int64_t rows, int vocab) {
    const int splits = distill_splits(rows, vocab, false);
    return rows == 1 && splits == 1 ? 0 : rows * 4 * (1 + (splits > 1 ? 3 * splits : 0));
}
int64_t distill_stats_count(int64_t rows) { return rows * kStats + 1; }
hipError_t launch_distill(const dsalt_distill_args &a, hipStream_t stream) { return launch(a, false, stream); }
hipError_t launch_distill_bwd(const dsalt_distill_args &a, hipStream_t stream) { return launch(a, true, stream); }

}  // namespace dsalt
