// Distillation from a teacher's top logits, beside the label loss, forward and backward.
//
//   q   = softmax(t / tau) over the entries that a row lists
//   p   = softmax(z / tau) over the whole vocabulary
//   row = alpha tau^2 sum_k q_k (log q_k - log p_{i_k}) + (1 - alpha) (lse(z) - z_y)
//   loss = weight * sum of rows / max(1, rows that list an entry or carry a label)
//   dz  = g weight / count * [alpha tau (p - q) + (1 - alpha) (softmax(z) - onehot_y)]
//
// The floor is one read of the logits and one write of their gradient.  A forward that will be
// differentiated meets it: a workgroup holds its row in registers (k_distill_row), so loss AND
// gradient come out of one read, written for the g = 1 that loss.backward() hands in; the
// backward launch looks at g on the device and leaves at once, or, for another g, computes the
// gradient anew from the logits (k_distill_bwd), rounded once either way.
//
// Both softmaxes share the maximum m (tau > 0 does not move it).  A statistic is kept as the
// pair (m, L = log2 of the sum relative to m), never as one number m c + L: logits of a thousand
// would cost that sum the digits that the loss is made of.  Exponents are (z - m) c, the
// difference first: m c alone would overflow where a mask holds the type's lowest value.
#include "lm_common.h"

namespace {

// How the two temperatures' exponentials are had.  With tau = 2 or 4 the label's is the
// teacher's squared once or twice: exp2 issues at a quarter of the rate of a product, and at two
// exponentials an element and pass the stream would wait for them.
enum { ONE = 0, GENERAL = 1, SQUARE = 2, FOURTH = 3 };

template <int MODE> DEVINL float second(float d, float e, float c1) {
    return MODE == GENERAL ? exp2_(d * c1) : MODE == SQUARE ? e * e : e * e * (e * e);
}

// The reference that exponents are taken from: a row of -inf alone keeps its sums at zero.
DEVINL float ref_of(float m) { return m == neg_inf() ? 0.f : m; }

struct Lists {
    const void* index;      // (N, K) int32 / int64, row stride is
    const void* teacher;    // (N, K) bf16 / fp16 / fp32, row stride ts
    const long* target;     // (N,) or null
    long is, ts;
    int K, index64, type;
};

// An entry is there when its index lies in the vocabulary and its logit is not -inf.
DEVINL bool entry(const Lists& l, long row, int k, int V, long& i, float& t) {
    i = load_index(l.index, row * l.is + k, l.index64);
    if (i < 0 || i >= V) return false;
    t = load_float(l.teacher, row * l.ts + k, l.type);
    return t != neg_inf();
}

// Per row: m, L of the label's and of the teacher's temperature, the teacher's own maximum and
// L, and whether the row counts.  A row without entries has the last L at -inf.
struct Stats {
    float m, l1, lt, rt, lq, counts, unused[2];
};

template <int TH> DEVINL float block_max(float v, float* lds) {
    v = wave_max(v);
    if ((threadIdx.x & 63) == 0) lds[__builtin_amdgcn_readfirstlane(threadIdx.x >> 6)] = v;
    __syncthreads();
    v = lds[threadIdx.x & (TH / 64 - 1)];
#pragma unroll
    for (int off = TH / 128; off > 0; off >>= 1) v = fmaxf(v, __shfl_xor(v, off, 64));
    __syncthreads();
    return v;
}
template <int TH> DEVINL float block_sum(float v, float* lds) {
    v = wave_sum(v);
    if ((threadIdx.x & 63) == 0) lds[__builtin_amdgcn_readfirstlane(threadIdx.x >> 6)] = v;
    __syncthreads();
    v = lds[threadIdx.x & (TH / 64 - 1)];
#pragma unroll
    for (int off = TH / 128; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
    __syncthreads();
    return v;
}

// ---------------------------------------------------------------------------
// The lists alone, a wave a row: the teacher's softmax, and which rows count.  It runs first
// because every gradient needs the count.  A single workgroup finishes the count itself.
// ---------------------------------------------------------------------------
__global__ __launch_bounds__(1024) void k_distill_lists(Lists l, Stats* __restrict__ stats, long N,
                                                        int V, float ct, float weight,
                                                        float* __restrict__ inv) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    float counted = 0.f;
    for (long row = blockIdx.x * 16l + wave; row < N; row += gridDim.x * 16l) {
        float mt = neg_inf(), any = 0.f, s = 0.f;
        for (int k = lane; k < l.K; k += 64) {
            long i;
            float t;
            if (entry(l, row, k, V, i, t)) {
                any = 1.f;
                mt = fmaxf(mt, t);
            }
        }
        any = wave_max(any);
        const float rt = ref_of(wave_max(mt));
        for (int k = lane; k < l.K; k += 64) {
            long i;
            float t;
            if (entry(l, row, k, V, i, t)) s += exp2_((t - rt) * ct);
        }
        s = wave_sum(s);
        const long y = l.target ? l.target[row] : -1;
        const float c = any != 0.f || (y >= 0 && y < V) ? 1.f : 0.f;
        counted += c;
        if (lane == 0) {
            stats[row].rt = rt;
            stats[row].lq = any != 0.f ? __log2f(s) : neg_inf();
            stats[row].counts = c;
        }
    }
    if (gridDim.x == 1) {           // counted is the wave's, below 2^24: exact
        __shared__ float sum[16];
        if (lane == 0) sum[wave] = counted;
        __syncthreads();
        if (threadIdx.x == 0) {
            for (int w = 1; w < 16; ++w) counted += sum[w];
            *inv = weight / fmaxf(counted, 1.f);
        }
    }
}

DEVINL double sum1024(double s, double* lds) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) s += __shfl_xor(s, off, 64);
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = s;
    __syncthreads();
    s = lds[0];
    for (int w = 1; w < 16; ++w) s += lds[w];
    return s;
}

// One workgroup in a fixed order (no atomics), 64-bit sums: a hundred thousand rows.
__global__ __launch_bounds__(1024) void k_distill_count(const Stats* __restrict__ stats,
                                                        float weight, float* __restrict__ inv,
                                                        long N) {
    __shared__ double lds[16];
    double c = 0;
#pragma unroll 4
    for (long i = threadIdx.x; i < N; i += 1024) c += stats[i].counts;
    c = sum1024(c, lds);
    if (threadIdx.x == 0) *inv = (float)(weight / (c > 1 ? c : 1));
}

// `counted`: inv is there; otherwise the rows are counted with their losses.
__global__ __launch_bounds__(1024) void k_distill_mean(const float* __restrict__ rows,
                                                       const Stats* __restrict__ stats,
                                                       int counted, float weight,
                                                       float* __restrict__ inv,
                                                       float* __restrict__ loss, long N) {
    __shared__ double ls[16], lc[16];
    double s = 0, c = 0;
#pragma unroll 4
    for (long i = threadIdx.x; i < N; i += 1024) {
        s += rows[i];
        if (!counted) c += stats[i].counts;
    }
    s = sum1024(s, ls);
    if (!counted) c = sum1024(c, lc);
    if (threadIdx.x == 0) {
        const float f = counted ? *inv : (float)(weight / (c > 1 ? c : 1));
        if (!counted) *inv = f;
        *loss = N > 0 ? (float)(s * f) : 0.f;
    }
}

// ---------------------------------------------------------------------------
// What a row adds to the loss besides its stream: the K listed logits and the label's.
// ---------------------------------------------------------------------------
template <typename T, int TH>
DEVINL void row_loss(const T* __restrict__ z, long row, int V, const Lists& l, float m, float l1,
                     float lt, float ct, float alpha, float tau, Stats* __restrict__ stats,
                     float* __restrict__ rows, float* lds) {
    const float rt = stats[row].rt, lq = stats[row].lq;
    float kl = 0.f;
    if (lq != neg_inf() && alpha != 0.f) {
        for (int k = threadIdx.x; k < l.K; k += TH) {
            long i;
            float t;
            if (!entry(l, row, k, V, i, t)) continue;
            const float a = (t - rt) * ct - lq, q = exp2_(a);       // log2 q
            if (q != 0.f) kl += q * (a - (((float)z[i] - m) * ct - lt));
        }
    }
    kl = block_sum<TH>(kl, lds);
    if (threadIdx.x == 0) {
        const long y = l.target ? l.target[row] : -1;
        float loss = alpha * tau * tau * LN2 * kl;
        if (lq == neg_inf() || alpha == 0.f) loss = 0.f;
        if (y >= 0 && y < V && alpha != 1.f)
            loss += (1.f - alpha) * (LN2 * l1 - ((float)z[y] - m));
        rows[row] = loss;
        stats[row].m = m;
        stats[row].l1 = l1;
        stats[row].lt = lt;
    }
}

// What the gradient of one row needs, for any of its columns.
template <int MODE> struct Grad {
    float m, c1, ct, lt, l1, ak, ac, pt, p1;    // pt, p1: the terms' factors before the exponential
    bool soft, label;
    DEVINL Grad(const Stats& s, const Lists& l, long row, int V, float g, float c1_, float ct_,
                float alpha, float tau)
        : m(s.m), c1(c1_), ct(ct_), lt(s.lt), l1(s.l1) {
        const long y = l.target ? l.target[row] : -1;
        label = y >= 0 && y < V && alpha != 1.f;
        soft = s.lq != neg_inf() && alpha != 0.f;
        ak = soft ? g * alpha * tau : 0.f;
        ac = label ? g * (1.f - alpha) : 0.f;
        pt = (MODE == ONE ? ak + ac : ak) * exp2_(-lt);     // the sums are at least 1
        p1 = ac * exp2_(-l1);
    }
    DEVINL float operator()(float x) const {
        const float d = x - m, e = exp2_(d * ct);
        return MODE == ONE ? pt * e : pt * e + p1 * second<MODE>(d, e, c1);
    }
};

// The listed columns and the label's in [lo, hi), written again after the stream (the caller has
// synchronised): computed anew in 32 bits and rounded once.  `bits` and `again` hold hi - lo zero
// bits, whole windows of 256.  Of an index that a row lists twice the entries are summed in the
// list's order: a wave walks the list once for a window of columns of its own, in `sums` (each
// entry's own walk to find its like took four rows of 20000, one of them twice, 141 ms; now 0.4).
constexpr int WINDOW = 256;
template <typename T, int TH, int MODE>
DEVINL void write_listed(const T* __restrict__ z, T* __restrict__ d, long row, int lo, int hi,
                         int V, const Lists& l, const Grad<MODE>& f, float rt, float lq,
                         unsigned* bits, unsigned* again, float* sums, int* seen_label,
                         int* twice) {
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));       // nothing of this is worked out before the stream
    const long y = l.target ? l.target[row] : -1;
    if (f.soft) {
        auto write = [&](long i, float q) {
            d[i] = (T)(f((float)z[i]) - f.ak * q - (i == y ? f.ac : 0.f));
        };
        auto repeated = [&](long i) { return again[(i - lo) >> 5] >> ((i - lo) & 31) & 1; };
        for (int k = tid; k < l.K; k += TH) {
            long i;
            float t;
            if (!entry(l, row, k, V, i, t) || i < lo || i >= hi) continue;
            const unsigned bit = 1u << ((i - lo) & 31);
            if (atomicOr(&bits[(i - lo) >> 5], bit) & bit) {
                atomicOr(&again[(i - lo) >> 5], bit);
                *twice = 1;
            }
            if (i == y) *seen_label = 1;
        }
        __syncthreads();
        for (int k = tid; k < l.K; k += TH) {
            long i;
            float t;
            if (!entry(l, row, k, V, i, t) || i < lo || i >= hi) continue;
            if (!repeated(i)) write(i, exp2_((t - rt) * f.ct - lq));
        }
        if (*twice) {
            const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
            sums += wave * WINDOW;
#pragma unroll 1
            for (int w0 = lo + wave * WINDOW; w0 < hi; w0 += TH / 64 * WINDOW) {
                if (!__any(again[((w0 - lo) >> 5) + (lane & 7)])) continue;
                wave_fence();
#pragma unroll 1
                for (int i = 0; i < WINDOW / 64; ++i) sums[i * 64 + lane] = 0.f;
                wave_fence();
#pragma unroll 1
                for (int k0 = 0; k0 < l.K; k0 += 64) {
                    long i = 0;
                    float t = 0.f;
                    const bool mine = k0 + lane < l.K && entry(l, row, k0 + lane, V, i, t) &&
                                      i >= w0 && i < min(w0 + WINDOW, hi) && repeated(i);
                    add_in_order(mine, (int)i - w0, exp2_((t - rt) * f.ct - lq), sums);
                }
                wave_fence();
#pragma unroll 1
                for (int i = w0 + lane; i < min(w0 + WINDOW, hi); i += 64)
                    if (repeated(i)) write(i, sums[i - w0]);
            }
        }
    }
    if (tid == 0 && f.label && !*seen_label && y >= lo && y < hi)
        d[y] = (T)(f((float)z[y]) - f.ac);
}

// Eight elements as the registers that hold them: four of 16-bit types, eight of fp32.
template <typename T> struct Raw {
    typedef int type __attribute__((ext_vector_type(sizeof(T) * 2)));
    typedef int loose __attribute__((ext_vector_type(sizeof(T) * 2), aligned(sizeof(T))));
};
template <typename T> DEVINL float element(const typename Raw<T>::type& v, int j) {
    return (float)__builtin_bit_cast(typename Vec8<T>::type, v)[j];
}
template <> DEVINL float element<bf16_t>(const Raw<bf16_t>::type& v, int j) {
    return __int_as_float(j & 1 ? v[j >> 1] & 0xffff0000 : v[j >> 1] << 16);
}
template <typename T> constexpr int minus_inf_word() {
    return sizeof(T) == 4 ? 0xff800000 : __is_same(T, bf16_t) ? 0xff80ff80 : 0xfc00fc00;
}

// The registers' contents as the compiler knows nothing about: without it, it keeps every value's
// 32-bit form and exponential from the sums to the gradient, four times the row's own registers.
// Tied to running values too, it also keeps the vectors' turns in order: interleaved, they spill.
template <typename R> DEVINL void forget(R& v, float& a, float& b) {
    asm volatile("" : "+v"(v), "+v"(a), "+v"(b)::"memory");
}

// ---------------------------------------------------------------------------
// A row in registers: TH threads hold NV vectors of eight each (50000 bf16 columns: 28 VGPRs of
// 1024 threads, two workgroups a CU).  One read gives the maximum, the sums, the loss and, GRAD,
// the gradient.
// More than 80 scalar registers, as 96 with what the system keeps, would leave a CU one workgroup
// of 1024 (1021 rows of 32001 fp32: 66 us instead of 56), a spilled one makes every wave wait for
// its stores.
// ---------------------------------------------------------------------------
template <typename T, int MODE, int TH, int NV, bool GRAD>
__global__ __launch_bounds__(TH, sizeof(T) * NV <= 14 ? 8 : 4)
__attribute__((amdgpu_num_sgpr(80))) void k_distill_row(
    const T* __restrict__ logits, long zs, Lists l, Stats* __restrict__ stats,
    float* __restrict__ rows, const float* __restrict__ inv, T* __restrict__ dz, int V, float c1,
    float ct, float alpha, float tau) {
    typedef typename Raw<T>::type Vec;
    __shared__ float lds[TH / 64];
    __shared__ int seen_label, twice;
    __shared__ unsigned bits[GRAD ? TH * NV / 4 : 1], again[GRAD ? TH * NV / 4 : 1];
    __shared__ float sums[GRAD ? TH / 64 * WINDOW : 1];
    const int tid = threadIdx.x;
    const long row = blockIdx.x;
    const T* z = logits + row * zs;
    Vec x[NV];
#pragma unroll
    for (int u = 0; u < NV; ++u) {
        const int v0 = (u * TH + tid) * 8;
        x[u] = v0 + 8 <= V ? *(const typename Raw<T>::loose*)(z + v0)
                           : (Vec)minus_inf_word<T>();
    }
    // what is left of a vocabulary that is no multiple of eight: one more for a few threads
    const int last = (V & ~7) + tid;
    const float rest = last < V && tid < 8 ? (float)z[last] : neg_inf();
    if (GRAD) {
        for (int i = tid; i < TH * NV / 4; i += TH) bits[i] = again[i] = 0;
        if (tid == 0) seen_label = twice = 0;
    }
    float m = rest, st = 0.f, s1 = 0.f;
#pragma unroll
    for (int u = 0; u < NV; ++u) {
#pragma unroll
        for (int j = 0; j < 8; ++j) m = fmaxf(m, element<T>(x[u], j));
        forget(x[u], m, s1);
    }
    m = ref_of(block_max<TH>(m, lds));
    {
        const float d = rest - m, e = exp2_(d * ct);
        st = e;
        if (MODE != ONE) s1 = second<MODE>(d, e, c1);
    }
#pragma unroll
    for (int u = 0; u < NV; ++u) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float d = element<T>(x[u], j) - m, e = exp2_(d * ct);
            st += e;
            if (MODE != ONE) s1 += second<MODE>(d, e, c1);
        }
        forget(x[u], st, s1);
    }
    const float lt = __log2f(block_sum<TH>(st, lds));
    const float l1 = MODE == ONE ? lt : __log2f(block_sum<TH>(s1, lds));
    if (!GRAD) {
        row_loss<T, TH>(z, row, V, l, m, l1, lt, ct, alpha, tau, stats, rows, lds);
        return;
    }
    T* d = dz + row * V;
    Stats s = stats[row];       // the teacher's part is there
    s.m = m;
    s.l1 = l1;
    s.lt = lt;
    const Grad<MODE> f(s, l, row, V, *inv, c1, ct, alpha, tau);
    const bool any = f.soft || f.label;     // padding: zero, whatever the logits hold
#pragma unroll
    for (int u = 0; u < NV; ++u) {
        const int v0 = (u * TH + tid) * 8;
        float o[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j] = any ? f(element<T>(x[u], j)) : 0.f;
        if (v0 + 8 <= V) store8(d + v0, o);
        if (u + 1 < NV) forget(x[u + 1], st, s1);
    }
    if (last < V && tid < 8) d[last] = (T)(any ? f(rest) : 0.f);
    // the row's registers are free from here on
    row_loss<T, TH>(z, row, V, l, m, l1, lt, ct, alpha, tau, stats, rows, lds);
    if (any)                                // row_loss has synchronised behind the stream
        write_listed<T, TH, MODE>(z, d, row, 0, V, V, l, f, s.rt, s.lq, bits, again, sums,
                                  &seen_label, &twice);
}

// ---------------------------------------------------------------------------
// The loss alone, of rows of any length: the running maximum and sums of one pass, rescaled when
// the maximum moves, which it may once per 32 values.
// ---------------------------------------------------------------------------
DEVINL float rescale(float m, float r, float c) {
    return m == neg_inf() ? 1.f : exp2_((m - r) * c);
}

template <typename T, int MODE, int TH>
__global__ __launch_bounds__(TH) void k_distill_long(
    const T* __restrict__ logits, long zs, Lists l, Stats* __restrict__ stats,
    float* __restrict__ rows, long N, int V, float c1, float ct, float alpha, float tau) {
    constexpr int U = 4;
    __shared__ float lds[TH / 64];
    for (long row = blockIdx.x; row < N; row += gridDim.x) {
        const T* z = logits + row * zs;
        float m = neg_inf(), st = 0.f, s1 = 0.f;
        for (long base = threadIdx.x * 8; base < V; base += TH * 8 * U) {
            float x[U][8];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const long v0 = base + u * TH * 8;
                if (v0 + 8 <= V) {
                    load8(z + v0, x[u]);
                } else {
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        x[u][j] = v0 + j < V ? (float)z[v0 + j] : neg_inf();
                }
            }
            float n = m;
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int j = 0; j < 8; ++j) n = fmaxf(n, x[u][j]);
            const float r = ref_of(n);
            st *= rescale(m, r, ct);
            if (MODE != ONE) s1 *= rescale(m, r, c1);
            m = n;
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float d = x[u][j] - r, e = exp2_(d * ct);
                    st += e;
                    if (MODE != ONE) s1 += second<MODE>(d, e, c1);
                }
        }
        const float r = ref_of(block_max<TH>(m, lds));
        const float lt = __log2f(block_sum<TH>(st * rescale(m, r, ct), lds));
        const float l1 = MODE == ONE
                             ? lt
                             : __log2f(block_sum<TH>(s1 * rescale(m, r, c1), lds));
        row_loss<T, TH>(z, row, V, l, r, l1, lt, ct, alpha, tau, stats, rows, lds);
    }
}

// ---------------------------------------------------------------------------
// The gradient from the logits and their statistics, `chunks` workgroups a row.  `done`: dz
// holds the gradient for g = 1 already.
// ---------------------------------------------------------------------------
template <typename T, int MODE>
__global__ __launch_bounds__(256) void k_distill_bwd(
    const T* __restrict__ logits, long zs, Lists l, const Stats* __restrict__ stats,
    const float* __restrict__ inv, const float* __restrict__ grad, T* __restrict__ dz, int done,
    long N, int V, int chunks, int width, float c1, float ct, float alpha, float tau) {
    __shared__ int seen_label, twice;
    __shared__ unsigned bits[512], again[512];      // width <= 16384 columns
    __shared__ float sums[4 * WINDOW];
    if (done && *grad == 1.f) return;
    const float g = *grad * *inv;
    for (long b = blockIdx.x; b < N * chunks; b += gridDim.x) {
        const long row = b / chunks;
        const int lo = (int)(b % chunks) * width, hi = min(V, lo + width);
        const T* z = logits + row * zs;
        T* d = dz + row * V;
        const Grad<MODE> f(stats[row], l, row, V, g, c1, ct, alpha, tau);
        const bool any = f.soft || f.label;
        for (int i = threadIdx.x; i < 512; i += 256) bits[i] = again[i] = 0;
        if (threadIdx.x == 0) seen_label = twice = 0;
        for (int v0 = lo + threadIdx.x * 8; v0 < hi; v0 += 256 * 8) {
            if (v0 + 8 <= hi) {
                float x[8] = {};
                if (any) {
                    load8(z + v0, x);
#pragma unroll
                    for (int j = 0; j < 8; ++j) x[j] = f(x[j]);
                }
                store8(d + v0, x);
            } else {
                for (int v = v0; v < hi; ++v) d[v] = (T)(any ? f((float)z[v]) : 0.f);
            }
        }
        __syncthreads();
        if (any)
            write_listed<T, 256, MODE>(z, d, row, lo, hi, V, l, f, stats[row].rt, stats[row].lq,
                                       bits, again, sums, &seen_label, &twice);
        __syncthreads();                // bits and flags are used again by the next chunk
    }
}

constexpr int LONGEST = 1024 * 8 * 7;   // columns that a workgroup's registers hold

template <typename T, int MODE, int TH, int NV>
void row_kernel(const void* z, long zs, const Lists& l, Stats* stats, float* rows,
                const float* inv, void* dz, long N, int V, float c1, float ct, float alpha,
                float tau, hipStream_t st) {
    const unsigned grid = (unsigned)N;
    if (dz)
        k_distill_row<T, MODE, TH, NV, true><<<grid, TH, 0, st>>>(
            (const T*)z, zs, l, stats, rows, inv, (T*)dz, V, c1, ct, alpha, tau);
    else
        k_distill_row<T, MODE, TH, NV, false><<<grid, TH, 0, st>>>(
            (const T*)z, zs, l, stats, rows, inv, (T*)dz, V, c1, ct, alpha, tau);
}

template <typename T, int MODE>
void fwd(const void* z, long zs, const Lists& l, Stats* stats, float* rows, const float* inv,
         void* dz, long N, int V, float c1, float ct, float alpha, float tau, hipStream_t st) {
    // Loss alone of many rows: small workgroups that keep loading while others reduce (8192 rows
    // of 50000 bf16: 165 us, 190 in registers); of few rows, the row's latency counts.
    const unsigned grid = (unsigned)(N < (1 << 20) ? N : (1 << 20));
    if (!dz && N >= 512)
        k_distill_long<T, MODE, 256><<<grid, 256, 0, st>>>((const T*)z, zs, l, stats, rows, N, V,
                                                           c1, ct, alpha, tau);
    else if (V > LONGEST)
        k_distill_long<T, MODE, 1024><<<grid, 1024, 0, st>>>((const T*)z, zs, l, stats, rows, N,
                                                             V, c1, ct, alpha, tau);
    // short rows: small workgroups, so that a CU's rows come and go one by one
    else if (V <= 256 * 8 * 4)
        row_kernel<T, MODE, 256, 4>(z, zs, l, stats, rows, inv, dz, N, V, c1, ct, alpha, tau, st);
    else if (V <= 1024 * 8 * 4)
        row_kernel<T, MODE, 1024, 4>(z, zs, l, stats, rows, inv, dz, N, V, c1, ct, alpha, tau, st);
    else
        row_kernel<T, MODE, 1024, 7>(z, zs, l, stats, rows, inv, dz, N, V, c1, ct, alpha, tau, st);
}

template <typename T, int MODE>
void bwd(const void* z, long zs, const Lists& l, const Stats* stats, const float* inv,
         const float* grad, void* dz, int done, long N, int V, float c1, float ct, float alpha,
         float tau, hipStream_t st) {
    int chunks = (V + 16383) / 16384;
    while (N * chunks < 1024 && V / chunks > 4096) chunks *= 2;     // few rows: fill the chip
    const int width = ((V + chunks - 1) / chunks + 7) / 8 * 8;
    const long blocks = N * chunks;
    // eight a CU; where the work is done already they only have to come and go
    k_distill_bwd<T, MODE><<<(unsigned)(blocks < 2048 ? blocks : 2048), 256, 0, st>>>(
        (const T*)z, zs, l, stats, inv, grad, (T*)dz, done, N, V, chunks, width, c1, ct, alpha,
        tau);
}

// One temperature serves both terms when it is 1, or when one of the terms is absent.
int mode_of(const Lists& l, float alpha, float tau) {
    if (tau == 1.f || !l.target || alpha == 1.f) return ONE;
    return tau == 2.f ? SQUARE : tau == 4.f ? FOURTH : GENERAL;
}

}  // namespace

extern "C" {

// Whether a forward can leave the gradient too.
int distill_in_registers(int V) { return V <= LONGEST; }

void launch_distill_fwd(int type, const void* z, long zs, const void* index, long is, int index64,
                        const void* teacher, long ts, int ttype, const long* target, int K,
                        void* stats, float* rows, float* loss, float* inv, void* dz, long N,
                        int V, float alpha, float tau, float weight, hipStream_t st) {
    const Lists l{index, teacher, target, is, ts, K, index64, ttype};
    const float c1 = LOG2E, ct = LOG2E / tau;
    Stats* s = (Stats*)stats;
    if (N > 0) {
        // one workgroup up to four rows a wave; the count of more is a launch of its own where
        // gradients wait for it
        const long wanted = N <= 64 ? 1 : (N + 15) / 16;
        k_distill_lists<<<(unsigned)(wanted < (1 << 20) ? wanted : (1 << 20)), 1024, 0, st>>>(
            l, s, N, V, ct, weight, inv);
        if (wanted > 1 && dz) k_distill_count<<<1, 1024, 0, st>>>(s, weight, inv, N);
#define MODES(T)                                                                                 \
    switch (mode_of(l, alpha, tau)) {                                                            \
        case ONE: fwd<T, ONE>(z, zs, l, s, rows, inv, dz, N, V, c1, ct, alpha, tau, st); break;  \
        case SQUARE:                                                                             \
            fwd<T, SQUARE>(z, zs, l, s, rows, inv, dz, N, V, c1, ct, alpha, tau, st);            \
            break;                                                                               \
        case FOURTH:                                                                             \
            fwd<T, FOURTH>(z, zs, l, s, rows, inv, dz, N, V, c1, ct, alpha, tau, st);            \
            break;                                                                               \
        default: fwd<T, GENERAL>(z, zs, l, s, rows, inv, dz, N, V, c1, ct, alpha, tau, st);      \
    }
        if (type == LM_BF16) {
            MODES(bf16_t)
        } else if (type == LM_F16) {
            MODES(f16_t)
        } else {
            MODES(float)
        }
#undef MODES
    }
    k_distill_mean<<<1, 1024, 0, st>>>(rows, s, N > 0 && (N <= 64 || dz), weight, inv, loss, N);
}

void launch_distill_bwd(int type, const void* z, long zs, const void* index, long is, int index64,
                        const void* teacher, long ts, int ttype, const long* target, int K,
                        const void* stats, const float* inv, const float* grad, void* dz,
                        int done, long N, int V, float alpha, float tau, hipStream_t st) {
    const Lists l{index, teacher, target, is, ts, K, index64, ttype};
    const float c1 = LOG2E, ct = LOG2E / tau;
    const Stats* s = (const Stats*)stats;
#define MODES(T)                                                                                 \
    switch (mode_of(l, alpha, tau)) {                                                            \
        case ONE: bwd<T, ONE>(z, zs, l, s, inv, grad, dz, done, N, V, c1, ct, alpha, tau, st);   \
            break;                                                                               \
        case SQUARE:                                                                             \
            bwd<T, SQUARE>(z, zs, l, s, inv, grad, dz, done, N, V, c1, ct, alpha, tau, st);      \
            break;                                                                               \
        case FOURTH:                                                                             \
            bwd<T, FOURTH>(z, zs, l, s, inv, grad, dz, done, N, V, c1, ct, alpha, tau, st);      \
            break;                                                                               \
        default: bwd<T, GENERAL>(z, zs, l, s, inv, grad, dz, done, N, V, c1, ct, alpha, tau,     \
                                 st);                                                            \
    }
    if (type == LM_BF16) {
        MODES(bf16_t)
    } else if (type == LM_F16) {
        MODES(f16_t)
    } else {
        MODES(float)
    }
#undef MODES
}

}  // extern "C"
