// Distillation from a teacher's top logits, beside the label loss, forward and backward.
//
//   q   = softmax(t / tau) over the entries that a row lists
//   p   = softmax(z / tau) over the whole vocabulary
//   row = alpha tau^2 sum_k q_k (log q_k - log p_{i_k}) + (1 - alpha) (lse(z) - z_y)
//   loss = sum of rows / max(1, rows that list an entry or carry a label)
//   dz  = g / count * [alpha tau (p - q) + (1 - alpha) (softmax(z) - onehot_y)]
//
// Both softmaxes share ONE pass over the row: tau > 0 does not move the maximum, so the running
// state is (m, sum 2^((z-m) c1), sum 2^((z-m) ctau)), c = log2(e) / temperature.  A statistic is
// kept as the pair (m, L = log2 of the sum), never as one number m c + L: logits of a thousand
// would cost that sum the digits that the loss is made of.
#include "lm_common.h"

namespace {

struct Stat {       // running maximum and the two sums relative to it
    float m, s1, st;
};

// The reference that the exponents are taken from.  A row (or part of one) that has seen nothing
// above -inf keeps its sums at zero and takes part in no rescaling.
DEVINL float ref_of(float m) { return m == neg_inf() ? 0.f : m; }

// A difference first, then the temperature: m c alone would overflow where a mask holds the
// type's lowest value.
DEVINL float rescale(float m, float r, float c) {
    return m == neg_inf() ? 1.f : exp2_((m - r) * c);
}

template <bool TWO>
DEVINL void merge(Stat& a, float m, float s1, float st, float c1, float ct) {
    const float n = fmaxf(a.m, m), r = ref_of(n);
    a.st = a.st * rescale(a.m, r, ct) + st * rescale(m, r, ct);
    if (TWO) a.s1 = a.s1 * rescale(a.m, r, c1) + s1 * rescale(m, r, c1);
    a.m = n;
}

// Running statistics of columns [lo, hi) of one row by 256 threads, in four 8-wide loads a step:
// the maximum is settled once per 32 values, so an element costs a max and a difference, and a
// product, an exp2 and an add per temperature -- at two bytes an element the exp2 rate is next to the memory's.
template <typename T, bool TWO>
DEVINL Stat scan(const T* __restrict__ z, int lo, int hi, float c1, float ct) {
    constexpr int U = 4;
    Stat a{neg_inf(), 0.f, 0.f};
    for (int base = lo + threadIdx.x * 8; base < hi; base += 256 * 8 * U) {
        float x[U][8];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int v0 = base + u * 256 * 8;
            if (v0 + 8 <= hi) {
                load8(z + v0, x[u]);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) x[u][j] = v0 + j < hi ? (float)z[v0 + j] : neg_inf();
            }
        }
        float n = a.m;
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int j = 0; j < 8; ++j) n = fmaxf(n, x[u][j]);
        const float r = ref_of(n);
        a.st *= rescale(a.m, r, ct);
        if (TWO) a.s1 *= rescale(a.m, r, c1);
        a.m = n;
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float d = x[u][j] - r;
                a.st += exp2_(d * ct);
                if (TWO) a.s1 += exp2_(d * c1);
            }
    }
    return a;
}

template <bool TWO>
DEVINL Stat block_merge(Stat a, float c1, float ct, float* lds) {
#pragma unroll 1
    for (int off = 32; off > 0; off >>= 1) {
        const float m = __shfl_xor(a.m, off, 64), s1 = __shfl_xor(a.s1, off, 64),
                    st = __shfl_xor(a.st, off, 64);
        merge<TWO>(a, m, s1, st, c1, ct);
    }
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) {
        lds[wave * 3] = a.m;
        lds[wave * 3 + 1] = a.s1;
        lds[wave * 3 + 2] = a.st;
    }
    __syncthreads();
    a = Stat{lds[0], lds[1], lds[2]};
    for (int w = 1; w < 4; ++w) merge<TWO>(a, lds[w * 3], lds[w * 3 + 1], lds[w * 3 + 2], c1, ct);
    __syncthreads();
    return a;
}

DEVINL float block_max(float v, float* lds) {
    v = wave_max(v);
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    v = fmaxf(fmaxf(lds[0], lds[1]), fmaxf(lds[2], lds[3]));
    __syncthreads();
    return v;
}
DEVINL float block_sum(float v, float* lds) {
    v = wave_sum(v);
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    v = (lds[0] + lds[1]) + (lds[2] + lds[3]);
    __syncthreads();
    return v;
}

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

// What a row's loss needs besides the stream: the K listed logits and the label's.
template <typename T>
DEVINL void finish_row(const T* __restrict__ z, long row, int V, const Lists& l, float m, float l1,
                       float lt, float ct, float alpha, float tau, float* __restrict__ stats,
                       float* __restrict__ rows, long N, float* lds) {
    float mt = neg_inf(), any = 0.f;
    for (int k = threadIdx.x; k < l.K; k += 256) {
        long i;
        float t;
        if (entry(l, row, k, V, i, t)) {
            any = 1.f;
            mt = fmaxf(mt, t);
        }
    }
    mt = block_max(mt, lds);
    any = block_max(any, lds);
    const float rt = ref_of(mt);
    float s = 0.f;
    for (int k = threadIdx.x; k < l.K; k += 256) {
        long i;
        float t;
        if (entry(l, row, k, V, i, t)) s += exp2_((t - rt) * ct);
    }
    s = block_sum(s, lds);
    const float lq = __log2f(s);
    float kl = 0.f;
    for (int k = threadIdx.x; k < l.K; k += 256) {
        long i;
        float t;
        if (!entry(l, row, k, V, i, t)) continue;
        const float a = (t - rt) * ct - lq, q = exp2_(a);       // log2 q
        if (q != 0.f) kl += q * (a - (((float)z[i] - ref_of(m)) * ct - lt));
    }
    kl = block_sum(kl, lds);
    if (threadIdx.x == 0) {
        const long y = l.target ? l.target[row] : -1;
        const bool label = y >= 0 && y < V;
        float loss = any != 0.f && alpha != 0.f ? alpha * tau * tau * LN2 * kl : 0.f;
        if (label && alpha != 1.f)
            loss += (1.f - alpha) * (LN2 * l1 - ((float)z[y] - ref_of(m)));
        rows[row] = loss;
        rows[N + row] = any != 0.f || label ? 1.f : 0.f;
        float* st = stats + row * 8;
        st[0] = ref_of(m);
        st[1] = l1;
        st[2] = lt;
        st[3] = rt;
        st[4] = any != 0.f ? lq : neg_inf();    // no entries: no teacher term
    }
}

// One workgroup a row: with thousands of rows the grid fills the chip and the row's stream is the
// whole cost.
template <typename T, bool TWO>
__global__ __launch_bounds__(256) void k_distill_fwd(
    const T* __restrict__ logits, long zs, Lists l, float* __restrict__ stats,
    float* __restrict__ rows, long N, int V, float c1, float ct, float alpha, float tau) {
    __shared__ float lds[12];
    for (long row = blockIdx.x; row < N; row += gridDim.x) {
        const T* z = logits + row * zs;
        const Stat a = block_merge<TWO>(scan<T, TWO>(z, 0, V, c1, ct), c1, ct, lds);
        const float lt = __log2f(a.st);
        const float l1 = TWO ? __log2f(a.s1) : lt;
        finish_row(z, row, V, l, a.m, l1, lt, ct, alpha, tau, stats, rows, N, lds);
    }
}

// Few rows: `splits` workgroups share a row's columns, a second launch joins them.
template <typename T, bool TWO>
__global__ __launch_bounds__(256) void k_distill_part(const T* __restrict__ logits, long zs,
                                                      float* __restrict__ part, int V, int splits,
                                                      int width, float c1, float ct) {
    __shared__ float lds[12];
    const long row = blockIdx.x / splits;
    const int sp = blockIdx.x % splits, lo = sp * width, hi = min(V, lo + width);
    const Stat a =
        block_merge<TWO>(scan<T, TWO>(logits + row * zs, lo, hi, c1, ct), c1, ct, lds);
    if (threadIdx.x == 0) {
        float* p = part + (row * splits + sp) * 3;
        p[0] = a.m;
        p[1] = a.s1;
        p[2] = a.st;
    }
}

template <typename T, bool TWO>
__global__ __launch_bounds__(256) void k_distill_join(
    const T* __restrict__ logits, long zs, Lists l, const float* __restrict__ part,
    float* __restrict__ stats, float* __restrict__ rows, long N, int V, int splits, float c1,
    float ct, float alpha, float tau) {
    __shared__ float lds[12];
    const long row = blockIdx.x;
    Stat a{neg_inf(), 0.f, 0.f};
    for (int s = threadIdx.x; s < splits; s += 256) {
        const float* p = part + (row * splits + s) * 3;
        merge<TWO>(a, p[0], p[1], p[2], c1, ct);
    }
    a = block_merge<TWO>(a, c1, ct, lds);
    const float lt = __log2f(a.st);
    const float l1 = TWO ? __log2f(a.s1) : lt;
    finish_row(logits + row * zs, row, V, l, a.m, l1, lt, ct, alpha, tau, stats, rows, N, lds);
}

// The mean over the rows that carry anything, and 1 / their count.  One workgroup in a
// fixed order (no atomics), 64-bit sums: a hundred thousand rows.
__global__ __launch_bounds__(1024) void k_distill_mean(const float* __restrict__ rows,
                                                       float* __restrict__ loss,
                                                       float* __restrict__ inv, long N) {
    __shared__ double ls[16], lc[16];
    double s = 0, c = 0;
    for (long i = threadIdx.x; i < N; i += 1024) {
        s += rows[i];
        c += rows[N + i];
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
        s += __shfl_xor(s, off, 64);
        c += __shfl_xor(c, off, 64);
    }
    if ((threadIdx.x & 63) == 0) {
        ls[threadIdx.x >> 6] = s;
        lc[threadIdx.x >> 6] = c;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < 16; ++w) {
            s += ls[w];
            c += lc[w];
        }
        const double n = c > 1 ? c : 1;
        *loss = (float)(s / n);
        *inv = (float)(1 / n);
    }
}

// Gradient: `chunks` workgroups a row.  The stream writes a p for every column of the chunk; then
// the few listed columns and the label's are written again, computed anew in 32 bits and rounded
// once.  An index that a row lists twice is summed by its first entry.
template <typename T, bool TWO>
__global__ __launch_bounds__(256) void k_distill_bwd(
    const T* __restrict__ logits, long zs, Lists l, const float* __restrict__ stats,
    const float* __restrict__ inv, const float* __restrict__ grad, T* __restrict__ dz, long N,
    int V, int chunks, int width, float c1, float ct, float alpha, float tau) {
    __shared__ int seen_label, twice;
    __shared__ unsigned bits[512];      // width <= 16384 columns
    const float g = *grad * *inv;
    for (long b = blockIdx.x; b < N * chunks; b += gridDim.x) {
        const long row = b / chunks;
        const int lo = (int)(b % chunks) * width, hi = min(V, lo + width);
        const T* z = logits + row * zs;
        T* d = dz + row * V;
        const float* st = stats + row * 8;
        const float m = st[0], l1 = st[1], lt = st[2], rt = st[3], lq = st[4];
        const long y = l.target ? l.target[row] : -1;
        const bool label = y >= 0 && y < V && alpha != 1.f, soft = lq != neg_inf() && alpha != 0.f;
        const float ak = soft ? g * alpha * tau : 0.f, ac = label ? g * (1.f - alpha) : 0.f;
        auto value = [&](float x) {
            if (TWO)
                return ak * exp2_((x - m) * ct - lt) + ac * exp2_((x - m) * c1 - l1);
            return (ak + ac) * exp2_((x - m) * ct - lt);
        };
        if (!soft && !label) {          // padding: zero, whatever the logits hold
            for (int v0 = lo + threadIdx.x * 8; v0 < hi; v0 += 256 * 8) {
                const float zero[8] = {};
                if (v0 + 8 <= hi) store8(d + v0, zero);
                else
                    for (int v = v0; v < hi; ++v) d[v] = (T)0.f;
            }
            continue;                   // the same for all threads of the workgroup
        }
        for (int i = threadIdx.x; i < 512; i += 256) bits[i] = 0;
        if (threadIdx.x == 0) seen_label = twice = 0;
        for (int v0 = lo + threadIdx.x * 8; v0 < hi; v0 += 256 * 8) {
            if (v0 + 8 <= hi) {
                float x[8];
                load8(z + v0, x);
#pragma unroll
                for (int j = 0; j < 8; ++j) x[j] = value(x[j]);
                store8(d + v0, x);
            } else {
                for (int v = v0; v < hi; ++v) d[v] = (T)value((float)z[v]);
            }
        }
        __syncthreads();
        if (soft) {
            for (int k = threadIdx.x; k < l.K; k += 256) {
                long i;
                float t;
                if (!entry(l, row, k, V, i, t) || i < lo || i >= hi) continue;
                const unsigned bit = 1u << ((i - lo) & 31);
                if (atomicOr(&bits[(i - lo) >> 5], bit) & bit) twice = 1;
                if (i == y) seen_label = 1;
            }
            __syncthreads();
            for (int k = threadIdx.x; k < l.K; k += 256) {
                long i;
                float t;
                if (!entry(l, row, k, V, i, t) || i < lo || i >= hi) continue;
                float q = exp2_((t - rt) * ct - lq);
                bool first = true;
                if (twice) {
                    for (int j = 0; j < l.K; ++j) {
                        long i2;
                        float t2;
                        if (j == k || !entry(l, row, j, V, i2, t2) || i2 != i) continue;
                        if (j < k) first = false;
                        else q += exp2_((t2 - rt) * ct - lq);
                    }
                }
                if (first) d[i] = (T)(value((float)z[i]) - ak * q - (i == y ? ac : 0.f));
            }
        }
        if (threadIdx.x == 0 && label && !seen_label && y >= lo && y < hi)
            d[y] = (T)(value((float)z[y]) - ac);
        __syncthreads();                // bits and flags are used again by the next chunk
    }
}

template <typename T, bool TWO>
void fwd(const void* z, long zs, const Lists& l, float* part, float* stats, float* rows,
         float* loss, float* inv, long N, int V, int splits, float c1, float ct, float alpha, float tau,
         hipStream_t stream) {
    if (N == 0) {           // the mean of nothing is zero
    } else if (splits <= 1) {
        const unsigned grid = (unsigned)(N < (1 << 20) ? N : (1 << 20));
        k_distill_fwd<T, TWO><<<grid, 256, 0, stream>>>((const T*)z, zs, l, stats, rows, N, V, c1,
                                                        ct, alpha, tau);
    } else {
        const int width = ((V + splits - 1) / splits + 7) / 8 * 8;
        k_distill_part<T, TWO><<<(unsigned)(N * splits), 256, 0, stream>>>(
            (const T*)z, zs, part, V, splits, width, c1, ct);
        k_distill_join<T, TWO><<<(unsigned)N, 256, 0, stream>>>(
            (const T*)z, zs, l, part, stats, rows, N, V, splits, c1, ct, alpha, tau);
    }
    k_distill_mean<<<1, 1024, 0, stream>>>(rows, loss, inv, N);
}

template <typename T, bool TWO>
void bwd(const void* z, long zs, const Lists& l, const float* stats, const float* inv,
         const float* grad, void* dz, long N, int V, float c1, float ct, float alpha, float tau,
         hipStream_t stream) {
    int chunks = (V + 16383) / 16384;
    while (N * chunks < 1024 && V / chunks > 4096) chunks *= 2;     // few rows: fill the chip
    const int width = ((V + chunks - 1) / chunks + 7) / 8 * 8;
    const long blocks = N * chunks;
    const unsigned grid = (unsigned)(blocks < (1 << 22) ? blocks : (1 << 22));
    k_distill_bwd<T, TWO><<<grid, 256, 0, stream>>>((const T*)z, zs, l, stats, inv, grad, (T*)dz,
                                                    N, V, chunks, width, c1, ct, alpha, tau);
}

}  // namespace

extern "C" {

// Workgroups that share a row's columns in the forward pass: about two a CU, no part shorter
// than one step of the scan.
int distill_splits(long N, int V) {
    if (N >= 512) return 1;
    const long want = (512 + N - 1) / (N > 0 ? N : 1), most = (V + 2047) / 2048;
    return (int)(want < most ? want : most);
}

// One temperature serves both terms when it is 1, or when one of the terms is absent.
void launch_distill_fwd(int type, const void* z, long zs, const void* index, long is, int index64,
                        const void* teacher, long ts, int ttype, const long* target, int K,
                        float* part, float* stats, float* rows, float* loss, float* inv,
                        long N, int V, float alpha, float tau, hipStream_t stream) {
    const Lists l{index, teacher, target, is, ts, K, index64, ttype};
    const bool two = tau != 1.f && target && alpha != 1.f;
    const float c1 = LOG2E, ct = LOG2E / tau;
    const int splits = distill_splits(N, V);
#define GO(T)                                                                                    \
    two ? fwd<T, true>(z, zs, l, part, stats, rows, loss, inv, N, V, splits, c1, ct, alpha, tau, \
                       stream)                                                                   \
        : fwd<T, false>(z, zs, l, part, stats, rows, loss, inv, N, V, splits, c1, ct, alpha, tau,\
                        stream)
    if (type == LM_BF16) GO(bf16_t);
    else if (type == LM_F16) GO(f16_t);
    else GO(float);
#undef GO
}

void launch_distill_bwd(int type, const void* z, long zs, const void* index, long is, int index64,
                        const void* teacher, long ts, int ttype, const long* target, int K,
                        const float* stats, const float* inv, const float* grad, void* dz, long N,
                        int V, float alpha, float tau, hipStream_t stream) {
    const Lists l{index, teacher, target, is, ts, K, index64, ttype};
    const bool two = tau != 1.f && target && alpha != 1.f;
    const float c1 = LOG2E, ct = LOG2E / tau;
#define GO(T)                                                                                    \
    two ? bwd<T, true>(z, zs, l, stats, inv, grad, dz, N, V, c1, ct, alpha, tau, stream)         \
        : bwd<T, false>(z, zs, l, stats, inv, grad, dz, N, V, c1, ct, alpha, tau, stream)
    if (type == LM_BF16) GO(bf16_t);
    else if (type == LM_F16) GO(f16_t);
    else GO(float);
#undef GO
}

}  // extern "C"
