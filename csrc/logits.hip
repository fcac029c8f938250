// Penalties for repeated tokens, biases and grammar masks on the logits of a decode step.
//
//   seen  : the token stands anywhere in the row's history
//   count : how often it stands behind the prompt, in what the row has generated
//   z1 = seen ? (z > 0 ? z / rho : z rho) : z
//   z2 = z1 - frequency count - presence [count > 0]
//   z3 = z2 + sum of the biases that the row lists for the token
//   out = allowed ? z3 : -inf
//
// ONE launch without state between steps: a workgroup owns `C` neighbouring columns of a row,
// counts the history's tokens that fall into them in LDS (whole-number atomics, so the order
// does not matter), and streams its columns once.  Each workgroup of a row reads the row's
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

template <typename T, int C>
__global__ __launch_bounds__(256) void k_adjust(const T* __restrict__ logits, long zs,
                                                T* __restrict__ out, Adjust a, long B, int V,
                                                int chunks) {
    __shared__ unsigned count[C];
    __shared__ float bias[C];
    __shared__ unsigned bits[C / 32];
    __shared__ int twice;
    const int tid = threadIdx.x;
    const bool past = a.history, some = a.bias_index;
    for (long blk = blockIdx.x; blk < B * chunks; blk += gridDim.x) {
        const long b = blk / chunks;
        const int lo = (int)(blk % chunks) * C, n = min(C, V - lo);
        if (past)
            for (int i = tid; i < C; i += 256) count[i] = 0;
        if (some) {
            for (int i = tid; i < C; i += 256) bias[i] = 0.f;
            for (int i = tid; i < C / 32; i += 256) bits[i] = 0;
            if (tid == 0) twice = 0;
        }
        __syncthreads();
        if (past) {
            long len = a.lengths ? load_index(a.lengths, b, a.lengths64) : a.L;
            len = len < 0 ? 0 : len > a.L ? a.L : len;
            const long prompt = a.prompts ? load_index(a.prompts, b, a.prompts64) : 0;
            for (long j = tid; j < len; j += 256) {
                const long v = load_index(a.history, b * a.hs + j, a.history64) - lo;
                if (v < 0 || v >= n) continue;
                if (j < prompt) atomicOr(&count[v], PROMPT);
                else atomicAdd(&count[v], 1u);
            }
        }
        if (some) {
            for (int k = tid; k < a.NB; k += 256) {
                const long v = load_index(a.bias_index, b * a.bis + k, a.index64) - lo;
                if (v < 0 || v >= n) continue;
                const unsigned bit = 1u << (v & 31);
                if (atomicOr(&bits[v >> 5], bit) & bit) twice = 1;
            }
            __syncthreads();
            for (int k = tid; k < a.NB; k += 256) {
                const long v = load_index(a.bias_index, b * a.bis + k, a.index64) - lo;
                if (v < 0 || v >= n) continue;
                float s = a.bias[b * a.bs + k];
                bool first = true;
                if (twice) {            // in the list's own order, so that the sum is one sum
                    for (int j = 0; j < a.NB; ++j) {
                        if (j == k ||
                            load_index(a.bias_index, b * a.bis + j, a.index64) - lo != v)
                            continue;
                        if (j < k) first = false;
                        else s += a.bias[b * a.bs + j];
                    }
                }
                if (first) bias[v] = s;
            }
        }
        __syncthreads();
        const float rho = a.repetition(b), pres = a.presence(b), freq = a.frequency(b);
        const T* z = logits + b * zs + lo;
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
        for (int i = tid * 8; i < n; i += 256 * 8) {
            unsigned ok = 0xff;
            if (a.allowed) ok = a.allowed[b * a.as + ((lo + i) >> 5)] >> ((lo + i) & 31);
            if (i + 8 <= n) {
                float x[8];
                load8(z + i, x);
#pragma unroll
                for (int j = 0; j < 8; ++j) x[j] = ok >> j & 1 ? value(x[j], i + j) : neg_inf();
                store8(o + i, x);
            } else {
                for (int j = 0; i + j < n; ++j)
                    o[i + j] = (T)(ok >> j & 1 ? value((float)z[i + j], i + j) : neg_inf());
            }
        }
        __syncthreads();                // the counts are cleared again for the next columns
    }
}

template <typename T, int C>
void go(const void* z, long zs, void* out, const Adjust& a, long B, int V, hipStream_t stream) {
    const int chunks = (V + C - 1) / C;
    const long blocks = B * chunks;
    k_adjust<T, C><<<(unsigned)(blocks < (1 << 22) ? blocks : (1 << 22)), 256, 0, stream>>>(
        (const T*)z, zs, (T*)out, a, B, V, chunks);
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
    if (type == LM_BF16) go<bf16_t, 2048>(z, zs, out, a, B, V, stream);
    else if (type == LM_F16) go<f16_t, 2048>(z, zs, out, a, B, V, stream);
    else go<float, 2048>(z, zs, out, a, B, V, stream);
}
