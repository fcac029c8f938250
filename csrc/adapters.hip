// Low-rank adapters of many requests at once beside a shared projection:
//
//   v_i   = s_l x_i A_l              (K -> R)        l = adapter of row i, or none
//   out_i = y_i + v_i B_l            (R -> M)
//   u_i   = s_l dy_i B_l^T           (M -> R)        backward
//   dx_i  = u_i A_l^T                (R -> K)
//   dA_l  = sum_i x_i^T u_i,   dB_l = sum_i v_i^T dy_i
//
// R is 4 to 128 where K and M are thousands, so every product streams one wide matrix past a
// narrow one and is bound by that stream: `shrink` reads rows (x, dy), `expand` reads and writes
// them (y, dx), `outer` reads them again for the weights' gradients.  MFMA feeds on 32 of the
// contraction at a time in the stream's own layout; accumulation, split sums and partial
// gradients are fp32, v and u are rounded once to the type (they are MFMA operands).
//
// Rows come grouped by adapter.  Sequences are time-major, row = t * Bn + column, and an adapter
// belongs to a column, so only the Bn columns are grouped: segment s lists its columns in
// `order[start, start + count)`, and its T * count rows are enumerated time-major.
#include "lm_common.h"

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef bf16_t bf16x8 __attribute__((ext_vector_type(8)));
typedef f16_t f16x8 __attribute__((ext_vector_type(8)));
template <typename T> struct Frag;
template <> struct Frag<bf16_t> { typedef bf16x8 type; };
template <> struct Frag<f16_t> { typedef f16x8 type; };

// A: lane holds row lane & 15, contraction (lane >> 4) * 8 + [0, 8); B: column lane & 15, the
// same; D: column lane & 15, rows (lane >> 4) * 4 + [0, 4).
DEVINL f32x4 mfma(bf16x8 a, bf16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
DEVINL f32x4 mfma(f16x8 a, f16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// Eight neighbours of which `left` exist; the others are zero.
template <typename T> DEVINL typename Frag<T>::type load_frag(const T* p, int left) {
    typename Frag<T>::type v;
    if (left >= 8) {
        const auto u = *(const typename Vec8<T>::type*)p;
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = u[j];
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = j < left ? p[j] : (T)0.f;
    }
    return v;
}

struct Rows {
    const int* order;       // (Bn,) columns, grouped by adapter
    const int4* segs;       // (S,) adapter (-1: none), start, count, 0
    const int* adapter;     // (Bn,) adapter of a column
    int S, Bn;
    long T;
};

struct Scale {              // one number an adapter, or one for all
    const float* p;
    float all;
    DEVINL float operator()(int l) const { return p ? p[l] : all; }
};

struct Tile {               // up to 1 << shift rows of one segment, from its row j0 on
    int adapter, start, count;
    long j0, n;             // n: rows of the segment
    int first;              // number of the segment's first tile
};

// Which rows tile number `tile` holds.  A wave sums up the segments' tiles, 64 at a time.
DEVINL Tile find_tile(const Rows& r, int tile, int shift) {
    const int lane = threadIdx.x & 63;
    int base = 0;
    Tile f{-1, 0, 0, 0, 0, 0};
    for (int s0 = 0; s0 < r.S; s0 += 64) {
        const int s = s0 + lane;
        const int4 g = s < r.S ? r.segs[s] : make_int4(-1, 0, 0, 0);
        const int t = (int)((r.T * g.z + (1l << shift) - 1) >> shift);
        int sum = t;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const int o = __shfl_up(sum, off, 64);
            if (lane >= off) sum += o;
        }
        const unsigned long long hit = __ballot(base + sum > tile);
        if (hit) {
            const int at = __ffsll(hit) - 1;
            f.adapter = __shfl(g.x, at, 64);
            f.start = __shfl(g.y, at, 64);
            f.count = __shfl(g.z, at, 64);
            f.first = base + __shfl(sum - t, at, 64);
            f.n = r.T * f.count;
            f.j0 = (long)(tile - f.first) << shift;
            return f;
        }
        base += __shfl(sum, 63, 64);
    }
    return f;
}

DEVINL long row_of(const Rows& r, const Tile& f, long j) {
    if (f.count == r.Bn) return j;                  // every column: grouping keeps their order
    if (r.T == 1) return r.order[f.start + j];
    const unsigned c = f.count, t = (unsigned)j / c;    // j < 2^31 (checked on the host)
    return (long)t * r.Bn + r.order[f.start + ((unsigned)j - t * c)];
}

// ---------------------------------------------------------------------------
// shrink: V[row] = s_l X[row] W_l.  A workgroup takes 128 rows of one adapter and `kper` of the
// contraction; its four waves hold 32 rows each and share W's 128-step panel, which lies in LDS
// with the contraction contiguous (transposed on the way in where W is (K, R)).
// ---------------------------------------------------------------------------
constexpr int S_TM = 7;     // log2 rows a workgroup
constexpr int S_KC = 128;   // contraction a step

template <typename T, int RT, bool KCONT>
__global__ __launch_bounds__(256) void k_shrink(const T* __restrict__ X, long xs,
                                                const T* __restrict__ W, int K, int R, Rows rows,
                                                Scale scale, T* __restrict__ V, int RP,
                                                float* __restrict__ part, long N, int splits,
                                                int kper) {
    typedef typename Frag<T>::type F;
    constexpr int LD = S_KC + 8;
    __shared__ __attribute__((aligned(16))) T w[RT * 16 * LD];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int split = blockIdx.x % splits;
    const Tile f = find_tile(rows, blockIdx.x / splits, S_TM);
    if (f.adapter < 0) return;
    const T* Wl = W + (long)f.adapter * K * R;
    const int kend = min(K, (split + 1) * kper);
    long row[2];
    bool ok[2];
    const T* xp[2];
#pragma unroll
    for (int m = 0; m < 2; ++m) {
        const long j = f.j0 + wave * 32 + m * 16 + (lane & 15);
        ok[m] = j < f.n;
        row[m] = row_of(rows, f, ok[m] ? j : f.n - 1);
        xp[m] = X + row[m] * xs;
    }
    f32x4 acc[2][RT];
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int t = 0; t < RT; ++t) acc[m][t] = f32x4{0, 0, 0, 0};

    for (int k0 = split * kper; k0 < kend; k0 += S_KC) {
        F x[2][4];
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                const int k = k0 + s * 32 + (lane >> 4) * 8;
                x[m][s] = load_frag(xp[m] + k, kend - k);
            }
        __syncthreads();
        if (KCONT) {
            for (int u = tid; u < RT * 16 * (S_KC / 8); u += 256) {
                const int r = u / (S_KC / 8), k = u % (S_KC / 8) * 8;
                *(F*)(w + r * LD + k) =
                    load_frag(Wl + (long)r * K + k0 + k, r < R ? kend - k0 - k : 0);
            }
        } else {
            for (int u = tid; u < RT * 2 * S_KC; u += 256) {
                const int k = u / (RT * 2), r = u % (RT * 2) * 8;
                const F v = load_frag(Wl + (long)(k0 + k) * R + r, k0 + k < kend ? R - r : 0);
#pragma unroll
                for (int j = 0; j < 8; ++j) w[(r + j) * LD + k] = v[j];
            }
        }
        __syncthreads();
#pragma unroll
        for (int s = 0; s < 4; ++s)
#pragma unroll
            for (int t = 0; t < RT; ++t) {
                const F b = *(const F*)(w + (t * 16 + (lane & 15)) * LD + s * 32 + (lane >> 4) * 8);
#pragma unroll
                for (int m = 0; m < 2; ++m) acc[m][t] = mfma(x[m][s], b, acc[m][t]);
            }
    }
    const float sc = scale(f.adapter);
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int src = (lane >> 4) * 4 + i;
            const long r = __shfl(row[m], src, 64);
            const int good = __shfl((int)ok[m], src, 64);
            if (!good) continue;
            if (splits > 1) {
                float* p = part + ((long)split * N + r) * (RT * 16) + (lane & 15);
#pragma unroll
                for (int t = 0; t < RT; ++t) p[t * 16] = acc[m][t][i];
            } else {
                T* v = V + r * RP + (lane & 15);
#pragma unroll
                for (int t = 0; t < RT; ++t) v[t * 16] = (T)(acc[m][t][i] * sc);
                if (RT == 1) v[16] = (T)0.f;        // expand contracts 32 at a time
            }
        }
}

template <typename T>
__global__ __launch_bounds__(256) void k_shrink_sum(const float* __restrict__ part, long N, int R16,
                                                    int splits, Rows rows, Scale scale,
                                                    T* __restrict__ V, int RP) {
    const long i = (long)blockIdx.x * 256 + threadIdx.x;
    if (i >= N * RP) return;
    const long row = i / RP;
    const int r = (int)(i % RP), l = rows.adapter[row % rows.Bn];
    if (l < 0) return;
    float s = 0.f;
    if (r < R16)
        for (int k = 0; k < splits; ++k) s += part[((long)k * N + row) * R16 + r];
    V[i] = (T)(s * scale(l));
}

// ---------------------------------------------------------------------------
// expand: out[row] = base[row] + V[row] W_l (base may be out itself, or absent: zero).  A wave
// keeps W for 64 columns in registers and streams the workgroup's rows past it, 16 at a time.
// W is the A operand and the rows are B's columns, so that a lane ends up with neighbouring
// columns of one row; columns are dealt to the tiles' rows such that two tiles make eight of
// them: column of tile t, MFMA row i = (t >> 1) * 32 + (i >> 2) * 8 + (t & 1) * 4 + (i & 3).
// ---------------------------------------------------------------------------
constexpr int E_TM = 7;

template <typename T, int RK, bool RCONT>
__global__ __launch_bounds__(256) void k_expand(const T* base, long bs, T* out, long os,
                                                const T* __restrict__ V, int RP,
                                                const T* __restrict__ W, int M, int R, Rows rows,
                                                int strips) {
    typedef typename Frag<T>::type F;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 4;
    const Tile f = find_tile(rows, blockIdx.x / strips, E_TM);
    const int m0 = blockIdx.x % strips * 256 + wave * 64;
    if (m0 >= M) return;
    F w[RK][4];
    if (f.adapter >= 0) {
        const T* Wl = W + (long)f.adapter * M * R;
#pragma unroll
        for (int k = 0; k < RK; ++k)
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const int i = lane & 15;
                const int m = m0 + (t >> 1) * 32 + (i >> 2) * 8 + (t & 1) * 4 + (i & 3);
                const int r = k * 32 + g * 8;
                if (RCONT) {
                    w[k][t] = load_frag(Wl + (long)m * R + r, m < M ? R - r : 0);
                } else {
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        w[k][t][j] =
                            m < M && r + j < R ? Wl[(long)(r + j) * M + m] : (T)0.f;
                }
            }
    }
    const long jend = min(f.n, f.j0 + (1l << E_TM));
    for (long j0 = f.j0; j0 < jend; j0 += 16) {
        const long j = j0 + (lane & 15);
        const bool ok = j < jend;
        const long row = row_of(rows, f, ok ? j : jend - 1);
        f32x4 acc[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) acc[t] = f32x4{0, 0, 0, 0};
        if (f.adapter >= 0) {
#pragma unroll
            for (int k = 0; k < RK; ++k) {
                const F v = *(const F*)(V + row * RP + k * 32 + g * 8);
#pragma unroll
                for (int t = 0; t < 4; ++t) acc[t] = mfma(w[k][t], v, acc[t]);
            }
        }
        if (!ok) continue;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int m = m0 + h * 32 + g * 8;
            float o[8] = {};
            if (m + 8 <= M) {
                if (base) load8(base + row * bs + m, o);
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    o[q] += acc[2 * h][q];
                    o[4 + q] += acc[2 * h + 1][q];
                }
                store8(out + row * os + m, o);
            } else {
#pragma unroll
                for (int q = 0; q < 8; ++q)
                    if (m + q < M) {
                        const float b = base ? (float)base[row * bs + m + q] : 0.f;
                        out[row * os + m + q] = (T)(b + acc[2 * h + (q >> 2)][q & 3]);
                    }
            }
        }
    }
}

// ---------------------------------------------------------------------------
// outer: part[tile][r][p] = sum over the tile's rows of P[row][p] Q[row][r].  The contraction
// runs over rows, so both operands are transposed on their way into LDS: a thread takes two
// rows' eight neighbours and writes eight row pairs.  LDS rows hold 64 of the contraction (128
// bytes, all banks); the 16-byte chunk is XORed with the row so that neither the writes (16
// column groups at once) nor the 16-byte reads (16 rows at once) meet in a bank.
// ---------------------------------------------------------------------------
DEVINL int swz(int p, int chunk) { return p * 64 + ((chunk ^ (p ^ (p >> 3))) & 7) * 8; }

template <typename T>
DEVINL void stage_pair(T* lds, int p0, int pair, typename Frag<T>::type a,
                       typename Frag<T>::type b) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        typedef T two __attribute__((ext_vector_type(2)));
        *(two*)(lds + swz(p0 + j, pair >> 2) + (pair & 3) * 2) = two{a[j], b[j]};
    }
}

template <typename T, int RT>
__global__ __launch_bounds__(256) void k_outer(const T* __restrict__ P, long ps, int NP,
                                               const T* __restrict__ Q, int RP,
                                               float* __restrict__ part, Rows rows, int strips,
                                               int shift) {
    typedef typename Frag<T>::type F;
    __shared__ __attribute__((aligned(16))) T pt[128 * 64];
    __shared__ __attribute__((aligned(16))) T qt[RT * 16 * 64];
    __shared__ long at[64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int tile = blockIdx.x / strips, p0 = blockIdx.x % strips * 128;
    const Tile f = find_tile(rows, tile, shift);
    if (f.adapter < 0) return;
    f32x4 acc[2][RT];
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int t = 0; t < RT; ++t) acc[m][t] = f32x4{0, 0, 0, 0};
    const long jend = min(f.n, f.j0 + (1l << shift));
    for (long j0 = f.j0; j0 < jend; j0 += 64) {
        __syncthreads();
        if (tid < 64) at[tid] = j0 + tid < jend ? row_of(rows, f, j0 + tid) : -1;
        __syncthreads();
        for (int u = tid; u < 32 * 16; u += 256) {
            const int c = u & 15, pair = u >> 4, p = p0 + c * 8;
            const long a = at[pair * 2], b = at[pair * 2 + 1];
            stage_pair(pt, c * 8, pair, load_frag(P + a * ps + p, a < 0 ? 0 : NP - p),
                       load_frag(P + b * ps + p, b < 0 ? 0 : NP - p));
        }
        for (int u = tid; u < 32 * RT * 2; u += 256) {
            const int c = u % (RT * 2), pair = u / (RT * 2);
            const long a = at[pair * 2], b = at[pair * 2 + 1];
            stage_pair(qt, c * 8, pair, load_frag(Q + a * RP + c * 8, a < 0 ? 0 : 8),
                       load_frag(Q + b * RP + c * 8, b < 0 ? 0 : 8));
        }
        __syncthreads();
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            F a[2];
#pragma unroll
            for (int m = 0; m < 2; ++m)
                a[m] = *(const F*)(pt + swz(wave * 32 + m * 16 + (lane & 15), s * 4 + (lane >> 4)));
#pragma unroll
            for (int t = 0; t < RT; ++t) {
                const F b = *(const F*)(qt + swz(t * 16 + (lane & 15), s * 4 + (lane >> 4)));
#pragma unroll
                for (int m = 0; m < 2; ++m) acc[m][t] = mfma(a[m], b, acc[m][t]);
            }
        }
    }
    const int LP = strips * 128;
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int t = 0; t < RT; ++t)
            *(f32x4*)(part + ((long)tile * RT * 16 + t * 16 + (lane & 15)) * LP + p0 + wave * 32 +
                      m * 16 + (lane >> 4) * 4) = acc[m][t];
}

// The weights' gradient: an adapter's tiles in their order, rounded once.  An adapter without
// rows gets zeros.  out is (L, R, NP) or, RCONT, (L, NP, R).
template <typename T, bool RCONT>
__global__ __launch_bounds__(256) void k_outer_sum(const float* __restrict__ part, int R16, int LP,
                                                   Rows rows, int shift, T* __restrict__ out,
                                                   int NP, int R, int blocks) {
    const int l = blockIdx.x / blocks, lane = threadIdx.x & 63;
    int first = 0, tiles = 0, base = 0;
    for (int s0 = 0; s0 < rows.S; s0 += 64) {
        const int s = s0 + lane;
        const int4 g = s < rows.S ? rows.segs[s] : make_int4(-1, 0, 0, 0);
        const int t = (int)((rows.T * g.z + (1l << shift) - 1) >> shift);
        int sum = t;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const int o = __shfl_up(sum, off, 64);
            if (lane >= off) sum += o;
        }
        const unsigned long long hit = __ballot(g.x == l && t > 0);
        if (hit) {
            const int k = __ffsll(hit) - 1;
            first = base + __shfl(sum - t, k, 64);
            tiles = __shfl(t, k, 64);
            break;
        }
        base += __shfl(sum, 63, 64);
    }
    const long i = (long)(blockIdx.x % blocks) * 256 + threadIdx.x;
    if (i >= (long)NP * R) return;
    const int p = (int)(i % NP), r = (int)(i / NP);
    float s = 0.f;
    for (int t = first; t < first + tiles; ++t) s += part[((long)t * R16 + r) * LP + p];
    out[(long)l * NP * R + (RCONT ? (long)p * R + r : i)] = (T)s;
}

int tiles_of(const long* counts, int S, long T, int shift) {
    long n = 0;
    for (int s = 0; s < S; ++s) n += (T * counts[s] + (1l << shift) - 1) >> shift;
    return (int)n;
}

template <typename T, int RT, bool KCONT>
void shrink_rt(const void* X, long xs, const void* W, int K, int R, const Rows& rows, int tiles,
               const Scale& scale, void* V, int RP, float* part, long N, int splits, int kper,
               hipStream_t st) {
    k_shrink<T, RT, KCONT><<<(unsigned)(tiles * splits), 256, 0, st>>>(
        (const T*)X, xs, (const T*)W, K, R, rows, scale, (T*)V, RP, part, N, splits, kper);
}

template <typename T, bool KCONT>
void shrink(const void* X, long xs, const void* W, int K, int R, const Rows& rows, int tiles,
            const Scale& scale, void* V, int RP, float* part, long N, int splits, int kper,
            hipStream_t st) {
#define GO(RT)                                                                                   \
    shrink_rt<T, RT, KCONT>(X, xs, W, K, R, rows, tiles, scale, V, RP, part, N, splits, kper, st)
    const int R16 = R <= 16 ? 16 : R <= 32 ? 32 : R <= 64 ? 64 : 128;
    if (R16 == 16) GO(1);
    else if (R16 == 32) GO(2);
    else if (R16 == 64) GO(4);
    else GO(8);
#undef GO
    if (splits > 1) {
        const long n = N * RP;
        k_shrink_sum<T><<<(unsigned)((n + 255) / 256), 256, 0, st>>>(part, N, R16, splits, rows,
                                                                     scale, (T*)V, RP);
    }
}

template <typename T, bool RCONT>
void expand(const void* base, long bs, void* out, long os, const void* V, int RP, const void* W,
            int M, int R, const Rows& rows, int tiles, hipStream_t st) {
    const int strips = (M + 255) / 256;
#define GO(RK)                                                                                   \
    k_expand<T, RK, RCONT><<<(unsigned)tiles * strips, 256, 0, st>>>(                            \
        (const T*)base, bs, (T*)out, os, (const T*)V, RP, (const T*)W, M, R, rows, strips)
    if (RP == 32) GO(1);
    else if (RP == 64) GO(2);
    else GO(4);
#undef GO
}

template <typename T, bool RCONT>
void outer(const void* P, long ps, int NP, const void* Q, int RP, float* part, const Rows& rows,
           int tiles, int shift, void* out, int R, int L, hipStream_t st) {
    const int strips = (NP + 127) / 128, R16 = R <= 16 ? 16 : RP;
#define GO(RT)                                                                                   \
    k_outer<T, RT><<<(unsigned)tiles * strips, 256, 0, st>>>((const T*)P, ps, NP, (const T*)Q,   \
                                                             RP, part, rows, strips, shift)
    if (tiles == 0) {           // no row has an adapter: the sum below writes zeros
    } else if (R16 == 16) GO(1);
    else if (R16 == 32) GO(2);
    else if (R16 == 64) GO(4);
    else GO(8);
#undef GO
    const int blocks = (int)(((long)NP * R + 255) / 256);
    k_outer_sum<T, RCONT><<<(unsigned)L * blocks, 256, 0, st>>>(
        part, R16, strips * 128, rows, shift, (T*)out, NP, R, blocks);
}

}  // namespace

extern "C" {

// Row length of v and u: the contraction of expand, in steps of 32.
int lowrank_rp(int R) { return R <= 32 ? 32 : R <= 64 ? 64 : 128; }

// Workgroups that share a row tile's contraction: about two a CU, no share below two steps.
int lowrank_splits(const long* counts, int S, long T, int K) {
    const int tiles = tiles_of(counts, S, T, S_TM), most = (K + 2 * S_KC - 1) / (2 * S_KC);
    int want = tiles > 0 ? (512 + tiles - 1) / tiles : 1;
    return want < 1 ? 1 : want > most ? most : want;
}

void launch_shrink(int type, int kcont, const void* X, long xs, const void* W, int K, int R,
                   const int* order, const int* segs, const int* adapter, const long* counts,
                   int S, int Bn, long T, const float* scale, float scale_all, void* V,
                   float* part, hipStream_t st) {
    const Rows rows{order, (const int4*)segs, adapter, S, Bn, T};
    const Scale sc{scale, scale_all};
    const int tiles = tiles_of(counts, S, T, S_TM), splits = lowrank_splits(counts, S, T, K);
    if (tiles == 0) return;
    const int kper = ((K + splits - 1) / splits + S_KC - 1) / S_KC * S_KC;
    const long N = T * Bn;
    const int RP = lowrank_rp(R);
    if (type == LM_BF16)
        kcont ? shrink<bf16_t, true>(X, xs, W, K, R, rows, tiles, sc, V, RP, part, N, splits,
                                     kper, st)
              : shrink<bf16_t, false>(X, xs, W, K, R, rows, tiles, sc, V, RP, part, N, splits,
                                      kper, st);
    else
        kcont ? shrink<f16_t, true>(X, xs, W, K, R, rows, tiles, sc, V, RP, part, N, splits, kper,
                                    st)
              : shrink<f16_t, false>(X, xs, W, K, R, rows, tiles, sc, V, RP, part, N, splits,
                                     kper, st);
}

void launch_expand(int type, int rcont, const void* base, long bs, void* out, long os,
                   const void* V, const void* W, int M, int R, const int* order, const int* segs,
                   const int* adapter, const long* counts, int S, int Bn, long T,
                   hipStream_t st) {
    const Rows rows{order, (const int4*)segs, adapter, S, Bn, T};
    const int tiles = tiles_of(counts, S, T, E_TM), RP = lowrank_rp(R);
    if (tiles == 0) return;
    if (type == LM_BF16)
        rcont ? expand<bf16_t, true>(base, bs, out, os, V, RP, W, M, R, rows, tiles, st)
              : expand<bf16_t, false>(base, bs, out, os, V, RP, W, M, R, rows, tiles, st);
    else
        rcont ? expand<f16_t, true>(base, bs, out, os, V, RP, W, M, R, rows, tiles, st)
              : expand<f16_t, false>(base, bs, out, os, V, RP, W, M, R, rows, tiles, st);
}

// log2 of the rows that one partial gradient sums: about two workgroups a CU over the strips,
// never fewer than 64 rows (a step) nor more than 4096.
int lowrank_outer_shift(const long* counts, int S, long T, int NP) {
    const int strips = (NP + 127) / 128;
    int shift = 12;
    while (shift > 6 && (long)tiles_of(counts, S, T, shift) * strips < 1024) --shift;
    return shift;
}
int lowrank_outer_tiles(const long* counts, int S, long T, int shift) {
    return tiles_of(counts, S, T, shift);
}

void launch_outer(int type, int rcont, const void* P, long ps, int NP, const void* Q, float* part,
                  const int* order, const int* segs, const int* adapter, const long* counts,
                  int S, int Bn, long T, int shift, void* out, int R, int L, hipStream_t st) {
    const Rows rows{order, (const int4*)segs, adapter, S, Bn, T};
    const int tiles = tiles_of(counts, S, T, shift), RP = lowrank_rp(R);
    if (type == LM_BF16)
        rcont ? outer<bf16_t, true>(P, ps, NP, Q, RP, part, rows, tiles, shift, out, R, L, st)
              : outer<bf16_t, false>(P, ps, NP, Q, RP, part, rows, tiles, shift, out, R, L, st);
    else
        rcont ? outer<f16_t, true>(P, ps, NP, Q, RP, part, rows, tiles, shift, out, R, L, st)
              : outer<f16_t, false>(P, ps, NP, Q, RP, part, rows, tiles, shift, out, R, L, st);
}

}  // extern "C"
