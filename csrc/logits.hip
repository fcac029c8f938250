// Penalties for repeated tokens, biases and grammar masks on the logits of a decode step.
//
//   seen  : the token stands anywhere in the row's history
//   count : how often it stands behind the prompt, in what the row has generated
//   z1 = seen ? (z > 0 ? z / rho : z rho) : z
//   z2 = z1 - frequency count - presence [count > 0]
//   z3 = z2 + sum of the biases that the row lists for the token
//   out = allowed ? z3 : -inf
//
// ONE launch without state between steps: a workgroup owns 2048 (8192) neighbouring columns of a
// row, counts the history's tokens that fall into them in LDS (whole-number atomics, so the
// order does not matter), and streams its columns once.  Each workgroup of a row reads the row's
// history again, from L2: a few KB beside its own columns.
#include "lm_common.h"

namespace {

struct Row {            // one per-request number: a tensor, or the same for all
    const float* p;
    float all;
    DEVINL float operator()(long b) const { return p ? p[b] : all; }
};

struct Adjust {
    const void *history, *lengths, *prompts, *bias_index;
    const float* bias;
    const unsigned* allowed;
    long hs, bis, bs, as;       // row strides
    int L, NB, history64, lengths64, prompts64, index64;
    Row repetition, presence, frequency;
};

constexpr unsigned PROMPT = 1u << 31;   // seen in the prompt; the bits below count the rest

template <typename T, int TH>
__global__ __launch_bounds__(TH) void k_adjust(const T* __restrict__ logits, long zs,
                                                T* __restrict__ out, Adjust a, int V, int chunks) {
    constexpr int C = TH * 8, U = TH > 256 ? 4 : 8;     // columns; tokens a thread at once
    __shared__ unsigned count[C];
    __shared__ float bias[C];
    __shared__ unsigned bits[C / 32], again[C / 32];   // tokens that the biases list, and repeat
    __shared__ int twice;
    const int tid = threadIdx.x;
    const bool past = a.history, some = a.bias_index;
    const long b = blockIdx.x / chunks;
    const int lo = (int)(blockIdx.x % chunks) * C, n = min(C, V - lo);
    const T* z = logits + b * zs + lo;
    // The columns and what the row is made of are all asked for before the first is needed.
    float x[8];
    const int i0 = tid * 8;
    if (i0 + 8 <= n) load8(z + i0, x);
    unsigned ok = 0xff;
    if (a.allowed && i0 < n) ok = a.allowed[b * a.as + ((lo + i0) >> 5)] >> ((lo + i0) & 31);
    long t[U];
    auto load = [&](long j0, long end) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const long j = j0 + u * TH + tid;
            t[u] = load_index(a.history, b * a.hs + (j < end ? j : end - 1), a.history64) - lo;
        }
    };
    if (past) load(0, a.L);     // the length is still on its way
    const float rho = a.repetition(b), pres = a.presence(b), freq = a.frequency(b);
    long len = 0, prompt = 0;
    if (past) {
        len = a.lengths ? load_index(a.lengths, b, a.lengths64) : a.L;
        len = len < 0 ? 0 : len > a.L ? a.L : len;
        prompt = a.prompts ? load_index(a.prompts, b, a.prompts64) : 0;
#pragma unroll
        for (int i = 0; i < C / TH; ++i) count[i * TH + tid] = 0;
    }
    if (some) {
#pragma unroll
        for (int i = 0; i < C / TH; ++i) bias[i * TH + tid] = 0.f;
        if (tid < C / 32) bits[tid] = again[tid] = 0;
        if (tid == 0) twice = 0;
    }
    __syncthreads();
    for (long j0 = 0; j0 < len; j0 += TH * U) {
        if (j0) load(j0, len);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const long j = j0 + u * TH + tid;
            if (j >= len || t[u] < 0 || t[u] >= n) continue;
            if (j < prompt) atomicOr(&count[t[u]], PROMPT);
            else atomicAdd(&count[t[u]], 1u);
        }
    }
    if (some) {
        for (int k = tid; k < a.NB; k += TH) {
            const long v = load_index(a.bias_index, b * a.bis + k, a.index64) - lo;
            const float f = a.bias[b * a.bs + k];
            if (v < 0 || v >= n) continue;
            const unsigned bit = 1u << (v & 31);
            if (atomicOr(&bits[v >> 5], bit) & bit) {
                atomicOr(&again[v >> 5], bit);
                twice = 1;
            } else {
                bias[v] = f;            // stands unless the token comes again
            }
        }
        __syncthreads();
        // Repeated tokens' biases, in the list's own order: a wave walks the list once for 512
        // columns of its own (20000 biases, one of them twice: 0.1 ms; each entry's own walk to
        // find its like took 158).
        if (twice) {
            const int lane = tid & 63, w0 = (tid & ~63) * 8;
            if (__any(lane < 16 && again[w0 / 32 + (lane & 15)])) {
                auto repeated = [&](int v) { return again[v >> 5] >> (v & 31) & 1; };
                for (int i = 0; i < 8; ++i)
                    if (repeated(w0 + i * 64 + lane)) bias[w0 + i * 64 + lane] = 0.f;
                wave_fence();
                for (int k0 = 0; k0 < a.NB; k0 += 64) {
                    const int k = min(k0 + lane, a.NB - 1);
                    const long v = load_index(a.bias_index, b * a.bis + k, a.index64) - lo;
                    const bool mine = k0 + lane < a.NB && v >= w0 && v < min(w0 + 512, n) &&
                                      repeated((int)v);
                    add_in_order(mine, (int)v, a.bias[b * a.bs + k], bias);
                }
            }
        }
    }
    __syncthreads();
    T* o = out + b * V + lo;
    auto value = [&](float x, int i) {
        if (past) {
            const unsigned c = count[i];
            if (c) {
                x = x > 0.f ? x / rho : x * rho;
                const unsigned fresh = c & ~PROMPT;
                if (fresh) x = x - freq * (float)fresh - pres;
            }
        }
        return some ? x + bias[i] : x;
    };
    if (i0 + 8 <= n) {
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = ok >> j & 1 ? value(x[j], i0 + j) : neg_inf();
        store8(o + i0, x);
    } else {
        for (int j = 0; i0 + j < n; ++j)
            o[i0 + j] = (T)(ok >> j & 1 ? value((float)z[i0 + j], i0 + j) : neg_inf());
    }
}

template <typename T>
void go(const void* z, long zs, void* out, const Adjust& a, long B, int V, hipStream_t stream) {
    // Every workgroup of a row reads its whole history: a long one by a quarter as many (columns of
    // 2048 and of 8192, 64 rows of 50000: 16384 tokens 27 and 16 us, 4096 12.7 and 10.4, 1024 10.3
    // and 10.0; 1024 rows: 4096 tokens 105 and 97, 1024 75 and 92).
    const int small = (V + 2047) / 2048, large = (V + 8191) / 8192;
    // A launch holds fewer than 2^32 threads: more rows than fit the large ones take the small.
    if (a.L >= 4096 && B * large * 1024 < (1l << 32))
        k_adjust<T, 1024><<<(unsigned)(B * large), 1024, 0, stream>>>((const T*)z, zs, (T*)out, a,
                                                                      V, large);
    else
        k_adjust<T, 256><<<(unsigned)(B * small), 256, 0, stream>>>((const T*)z, zs, (T*)out, a, V,
                                                                    small);
}

}  // namespace

extern "C" void launch_adjust(int type, const void* z, long zs, void* out, const void* history,
                              long hs, int L, int history64, const void* lengths, int lengths64,
                              const void* prompts, int prompts64, const float* repetition,
                              float repetition_all, const float* presence, float presence_all,
                              const float* frequency, float frequency_all, const void* bias_index,
                              long bis, int index64, const float* bias, long bs, int NB,
                              const unsigned* allowed, long as, long B, int V,
                              hipStream_t stream) {
    const Adjust a{history, lengths, prompts, bias_index, bias, allowed, hs, bis, bs, as, L, NB,
                   history64, lengths64, prompts64, index64, {repetition, repetition_all},
                   {presence, presence_all}, {frequency, frequency_all}};
    if (type == LM_BF16) go<bf16_t>(z, zs, out, a, B, V, stream);
    else if (type == LM_F16) go<f16_t>(z, zs, out, a, B, V, stream);
    else go<float>(z, zs, out, a, B, V, stream);
}
