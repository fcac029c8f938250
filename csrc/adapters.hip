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

// An operand whose contraction runs down the rows of an LDS tile: column c (lane & 15) of rows
// k0 + (lane >> 4) * 8 + [0, 8).  The hardware's transposing read takes 4 rows x 16 columns a
// group of 16 lanes: lane L names row L >> 2 and four columns, lane i receives column i's four.
// `c` is the address of that lane's four columns; tile rows are multiples of 8 bytes.
template <typename T> DEVINL typename Frag<T>::type column_frag(const T* tile, int ld, int k0,
                                                                int c) {
    typedef short s4 __attribute__((ext_vector_type(4)));
    typedef short s8 __attribute__((ext_vector_type(8)));
    typedef __attribute__((address_space(3))) s4 lds4;
    const int lane = threadIdx.x & 63;
    const T* p = tile + (k0 + (lane >> 4) * 8 + ((lane & 15) >> 2)) * ld + c;
    const s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)p);
    const s4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(p + 4 * ld));
    return __builtin_bit_cast(typename Frag<T>::type,
                              __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
}
DEVINL int own_columns() { return (threadIdx.x & 3) * 4; }     // of a lane, in 16 neighbours

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
// contraction; its four waves hold 32 rows each, straight from memory in the operand's layout,
// and share W's 128-step panel in LDS.  The next step's rows and panel are on their way while
// this one is multiplied.
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
    // rows of the panel: R of the contraction each (KCONT), or 128 of R each
    constexpr int LD = KCONT ? S_KC + 8 : RT * 16 + (RT >= 4 ? 16 : 0);
    __shared__ __attribute__((aligned(16))) T w[(KCONT ? RT * 16 : S_KC) * LD];
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

    F x[2][4], wv[RT];      // RT * 16 * 128 elements of the panel: RT vectors a thread
    auto load = [&](int k0) {
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                const int k = k0 + s * 32 + (lane >> 4) * 8;
                x[m][s] = load_frag(xp[m] + k, kend - k);
            }
#pragma unroll
        for (int i = 0; i < RT; ++i) {
            const int u = i * 256 + tid;
            if (KCONT) {
                const int r = u / (S_KC / 8), k = k0 + u % (S_KC / 8) * 8;
                wv[i] = load_frag(Wl + (long)r * K + k, r < R ? kend - k : 0);
            } else {
                const int k = k0 + u / (RT * 2), r = u % (RT * 2) * 8;
                wv[i] = load_frag(Wl + (long)k * R + r, k < kend ? R - r : 0);
            }
        }
    };
    int k0 = split * kper;
    if (k0 < kend) load(k0);
    for (; k0 < kend; k0 += S_KC) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < RT; ++i) {
            const int u = i * 256 + tid, n = KCONT ? S_KC / 8 : RT * 2;
            *(F*)(w + u / n * LD + u % n * 8) = wv[i];
        }
        F now[2][4];
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int s = 0; s < 4; ++s) now[m][s] = x[m][s];
        __syncthreads();
        if (k0 + S_KC < kend) load(k0 + S_KC);
#pragma unroll
        for (int s = 0; s < 4; ++s)
#pragma unroll
            for (int t = 0; t < RT; ++t) {
                const F b = KCONT ? *(const F*)(w + (t * 16 + (lane & 15)) * LD + s * 32 +
                                                (lane >> 4) * 8)
                                  : column_frag(w, LD, s * 32, t * 16 + own_columns());
#pragma unroll
                for (int m = 0; m < 2; ++m) acc[m][t] = mfma(now[m][s], b, acc[m][t]);
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
// keeps W for 64 columns in registers and streams the workgroup's rows past it, 32 at a time and
// 32 ahead.  W is the A operand and the rows are B's columns, so that a lane ends up with
// neighbouring columns of one row; columns are dealt to the tiles' rows such that two tiles make
// eight of them: column of tile t, MFMA row i = (t >> 1) * 32 + (i >> 2) * 8 + (t & 1) * 4 + (i & 3).
// ---------------------------------------------------------------------------
template <typename T, int RK, bool RCONT>
__global__ __launch_bounds__(256) void k_expand(const T* base, long bs, T* out, long os,
                                                const T* __restrict__ V, int RP,
                                                const T* __restrict__ W, int M, int R, Rows rows,
                                                int strips, int shift) {
    typedef typename Frag<T>::type F;
    typedef typename Vec8<T>::type U8;
    constexpr int LD = 256 + 16;
    __shared__ __attribute__((aligned(16))) T wt[RCONT ? 8 : RK * 32 * LD];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 4;
    const Tile f = find_tile(rows, blockIdx.x / strips, shift);
    const int strip = blockIdx.x % strips * 256, m0 = strip + wave * 64;
    const bool mine = f.adapter >= 0;
    if (!mine && base == out) return;           // nothing to add in place
    F w[RK][4];
    if (mine) {
        const T* Wl = W + (long)f.adapter * M * R;
        if (RCONT) {
#pragma unroll
            for (int k = 0; k < RK; ++k)
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    const int i = lane & 15, r = k * 32 + g * 8;
                    const int m = m0 + (t >> 1) * 32 + (i >> 2) * 8 + (t & 1) * 4 + (i & 3);
                    w[k][t] = load_frag(Wl + (long)m * R + r, m < M ? R - r : 0);
                }
        } else {
#pragma unroll
            for (int i = 0; i < RK * 4; ++i) {
                const int u = i * 256 + tid, r = u / 32, m = strip + u % 32 * 8;
                *(F*)(wt + r * LD + u % 32 * 8) =
                    load_frag(Wl + (long)r * M + m, r < R ? M - m : 0);
            }
            __syncthreads();
#pragma unroll
            for (int k = 0; k < RK; ++k)
#pragma unroll
                for (int t = 0; t < 4; ++t)
                    w[k][t] = column_frag(wt, LD, k * 32, wave * 64 + (t >> 1) * 32 +
                                                              (lane & 3) * 8 + (t & 1) * 4);
        }
    }
    if (m0 >= M) return;
    const long jend = min(f.n, f.j0 + (1l << shift));
    F v[2][RK];
    U8 y[2][2];
    long row[2];
    auto load = [&](long j0) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const long j = j0 + h * 16 + (lane & 15);
            row[h] = row_of(rows, f, j < jend ? j : jend - 1);
            if (mine)
#pragma unroll
                for (int k = 0; k < RK; ++k) v[h][k] = *(const F*)(V + row[h] * RP + k * 32 + g * 8);
            if (base)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const int m = m0 + c * 32 + g * 8;
                    if (m + 8 <= M) y[h][c] = *(const U8*)(base + row[h] * bs + m);
                }
        }
    };
    load(f.j0);
    for (long j0 = f.j0; j0 < jend; j0 += 32) {
        f32x4 acc[2][4];
        U8 b[2][2];
        long at[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            at[h] = row[h];
#pragma unroll
            for (int c = 0; c < 2; ++c) b[h][c] = y[h][c];
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                acc[h][t] = f32x4{0, 0, 0, 0};
                if (mine)
#pragma unroll
                    for (int k = 0; k < RK; ++k) acc[h][t] = mfma(w[k][t], v[h][k], acc[h][t]);
            }
        }
        if (j0 + 32 < jend) load(j0 + 32);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            if (j0 + h * 16 + (lane & 15) >= jend) continue;
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const int m = m0 + c * 32 + g * 8;
                if (m + 8 <= M) {
                    U8 o;
#pragma unroll
                    for (int q = 0; q < 8; ++q)
                        o[q] = (T)((base ? (float)b[h][c][q] : 0.f) + acc[h][2 * c + (q >> 2)][q & 3]);
                    *(U8*)(out + at[h] * os + m) = o;
                } else {
#pragma unroll
                    for (int q = 0; q < 8; ++q)
                        if (m + q < M) {
                            const float was = base ? (float)base[at[h] * bs + m + q] : 0.f;
                            out[at[h] * os + m + q] = (T)(was + acc[h][2 * c + (q >> 2)][q & 3]);
                        }
                }
            }
        }
    }
}

// ---------------------------------------------------------------------------
// outer: part[tile][r][p] = sum over the tile's rows of P[row][p] Q[row][r].  A workgroup owns 64
// CT columns and walks the tile's rows 64 at a time: they pass through LDS as they are, and both
// operands are read from there with their columns' rows side by side.
//
// DV: the rows meet W on the way too, partv[strip][row][r] = sum over the strip's columns of
// P[row][p] W_l[r][p] -- the backward pass's u, in shares of 256 columns.  dy is then read once
// for both; the shares cost 8 R bytes a row and strip (written, read again) beside the 512 of a
// second reading of dy.
// ---------------------------------------------------------------------------
template <typename T, int RT, int CT, bool DV>
__global__ __launch_bounds__(256) void k_outer(const T* __restrict__ P, long ps, int NP,
                                               const T* __restrict__ Q, int RP,
                                               float* __restrict__ part,
                                               const T* __restrict__ W, int R,
                                               float* __restrict__ partv, long N, Rows rows,
                                               int strips, int shift) {
    typedef typename Frag<T>::type F;
    constexpr int PC = 64 * CT, S = PC / 32, LP = PC + 16, LQ = RT * 16 + (RT >= 4 ? 16 : 0);
    constexpr int LW = PC + 8;
    __shared__ __attribute__((aligned(16))) T pt[64 * LP];
    __shared__ __attribute__((aligned(16))) T qt[64 * LQ];
    __shared__ __attribute__((aligned(16))) T wt[DV ? RT * 16 * LW : 8];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 4;
    const int tile = blockIdx.x / strips, strip = blockIdx.x % strips, p0 = strip * PC;
    const Tile f = find_tile(rows, tile, shift);
    if (f.adapter < 0) return;
    if (DV) {
        const T* Wl = W + (long)f.adapter * NP * R;
        for (int u = tid; u < RT * 16 * (PC / 8); u += 256) {
            const int r = u / (PC / 8), c = u % (PC / 8) * 8;
            *(F*)(wt + r * LW + c) = load_frag(Wl + (long)r * NP + p0 + c, r < R ? NP - p0 - c : 0);
        }
    }
    f32x4 acc[CT][RT];
#pragma unroll
    for (int c = 0; c < CT; ++c)
#pragma unroll
        for (int t = 0; t < RT; ++t) acc[c][t] = f32x4{0, 0, 0, 0};
    const long jend = min(f.n, f.j0 + (1l << shift));
    constexpr int QV = (64 * RT * 2 + 255) / 256;       // vectors of Q a thread
    F x[S], q[QV];
    long row = 0;
    bool ok = false;
    auto load = [&](long j0) {
        const long j = j0 + wave * 16 + (lane & 15);
        ok = j < jend;
        row = row_of(rows, f, ok ? j : jend - 1);
        const T* xp = P + row * ps + p0 + g * 8;
#pragma unroll
        for (int s = 0; s < S; ++s) x[s] = load_frag(xp + s * 32, ok ? NP - p0 - s * 32 - g * 8 : 0);
#pragma unroll
        for (int i = 0; i < QV; ++i) {
            const int u = i * 256 + tid, n = u / (RT * 2);
            if (n >= 64) continue;
            const long k = j0 + n;
            const long r = row_of(rows, f, k < jend ? k : jend - 1);
            q[i] = load_frag(Q + r * RP + u % (RT * 2) * 8, k < jend ? 8 : 0);
        }
    };
    load(f.j0);
    for (long j0 = f.j0; j0 < jend; j0 += 64) {
        __syncthreads();
        F now[S];
#pragma unroll
        for (int s = 0; s < S; ++s) {
            now[s] = x[s];
            *(F*)(pt + (wave * 16 + (lane & 15)) * LP + s * 32 + g * 8) = x[s];
        }
#pragma unroll
        for (int i = 0; i < QV; ++i) {
            const int u = i * 256 + tid, n = u / (RT * 2);
            if (n < 64) *(F*)(qt + n * LQ + u % (RT * 2) * 8) = q[i];
        }
        const long at = row;
        const bool good = ok;
        __syncthreads();
        if (j0 + 64 < jend) load(j0 + 64);
        if (DV) {
            f32x4 u[RT];
#pragma unroll
            for (int t = 0; t < RT; ++t) {
                u[t] = f32x4{0, 0, 0, 0};
#pragma unroll
                for (int s = 0; s < S; ++s)
                    u[t] = mfma(now[s], *(const F*)(wt + (t * 16 + (lane & 15)) * LW + s * 32 +
                                                    g * 8), u[t]);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const long r = __shfl(at, g * 4 + i, 64);
                if (__shfl((int)good, g * 4 + i, 64))
#pragma unroll
                    for (int t = 0; t < RT; ++t)
                        partv[((long)strip * N + r) * (RT * 16) + t * 16 + (lane & 15)] = u[t][i];
            }
        }
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            F b[RT];
#pragma unroll
            for (int t = 0; t < RT; ++t) b[t] = column_frag(qt, LQ, s * 32, t * 16 + own_columns());
#pragma unroll
            for (int c = 0; c < CT; ++c) {
                const F a = column_frag(pt, LP, s * 32, (wave * CT + c) * 16 + own_columns());
#pragma unroll
                for (int t = 0; t < RT; ++t) acc[c][t] = mfma(a, b[t], acc[c][t]);
            }
        }
    }
#pragma unroll
    for (int c = 0; c < CT; ++c)
#pragma unroll
        for (int t = 0; t < RT; ++t)
            *(f32x4*)(part + ((long)tile * RT * 16 + t * 16 + (lane & 15)) * (strips * PC) + p0 +
                      (wave * CT + c) * 16 + g * 4) = acc[c][t];
}

// The weights' gradient: an adapter's tiles in a fixed order, rounded once.  An adapter without
// rows gets zeros.  out is (L, R, NP) or, RCONT, (L, NP, R).  32 lanes take 128 columns of one r,
// eight groups share the tiles.
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
    __shared__ f32x4 sums[256];
    const int b = blockIdx.x % blocks, cols = (NP + 127) / 128;
    const int r = b / cols, p = b % cols * 128 + (threadIdx.x & 31) * 4, group = threadIdx.x >> 5;
    f32x4 s = f32x4{0, 0, 0, 0};
    const float* q = part + (long)r * LP + p;       // LP is a multiple of 128
#pragma unroll 4
    for (int t = first + group; t < first + tiles; t += 8)
        s += *(const f32x4*)(q + (long)t * R16 * LP);
    sums[threadIdx.x] = s;
    __syncthreads();
    if (group) return;
#pragma unroll
    for (int k = 1; k < 8; ++k) s += sums[k * 32 + threadIdx.x];
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (p + j < NP)
            out[(long)l * NP * R + (RCONT ? (long)(p + j) * R + r : (long)r * NP + p + j)] =
                (T)s[j];
}

int tiles_of(const long* counts, int S, long T, int shift) {
    long n = 0;
    for (int s = 0; s < S; ++s) n += (T * counts[s] + (1l << shift) - 1) >> shift;
    return (int)n;
}

int r16_of(int R) { return R <= 16 ? 16 : R <= 32 ? 32 : R <= 64 ? 64 : 128; }

template <typename T, bool KCONT>
void shrink(const void* X, long xs, const void* W, int K, int R, const Rows& rows, int tiles,
            const Scale& scale, void* V, int RP, float* part, long N, int splits, int kper,
            hipStream_t st) {
#define GO(RT)                                                                                   \
    k_shrink<T, RT, KCONT><<<(unsigned)(tiles * splits), 256, 0, st>>>(                          \
        (const T*)X, xs, (const T*)W, K, R, rows, scale, (T*)V, RP, part, N, splits, kper)
    const int R16 = r16_of(R);
    if (R16 == 16) GO(1);
    else if (R16 == 32) GO(2);
    else if (R16 == 64) GO(4);
    else GO(8);
#undef GO
}

template <typename T, bool RCONT>
void expand(const void* base, long bs, void* out, long os, const void* V, int RP, const void* W,
            int M, int R, const Rows& rows, int tiles, int shift, hipStream_t st) {
    const int strips = (M + 255) / 256;
#define GO(RK)                                                                                   \
    k_expand<T, RK, RCONT><<<(unsigned)tiles * strips, 256, 0, st>>>(                            \
        (const T*)base, bs, (T*)out, os, (const T*)V, RP, (const T*)W, M, R, rows, strips, shift)
    if (RP == 32) GO(1);
    else if (RP == 64) GO(2);
    else GO(4);
#undef GO
}

// Columns that a workgroup of outer owns: 256, or 128 where a rank of 128 fills the registers.
int outer_columns(int R) { return R > 64 ? 128 : 256; }

template <typename T, bool RCONT>
void outer(const void* P, long ps, int NP, const void* Q, int RP, float* part, const void* W,
           float* partv, long N, const Rows& rows, int tiles, int shift, void* out, int R, int L,
           hipStream_t st) {
    const int PC = outer_columns(R), strips = (NP + PC - 1) / PC, R16 = r16_of(R);
#define GO(RT, CT, DV)                                                                           \
    k_outer<T, RT, CT, DV><<<(unsigned)tiles * strips, 256, 0, st>>>(                            \
        (const T*)P, ps, NP, (const T*)Q, RP, part, (const T*)W, R, partv, N, rows, strips, shift)
    if (tiles == 0) {           // no row has an adapter: the sum below writes zeros
    } else if (R16 == 16) {
        if (W) GO(1, 4, true);
        else GO(1, 4, false);
    } else if (R16 == 32) {
        if (W) GO(2, 4, true);
        else GO(2, 4, false);
    } else if (R16 == 64) GO(4, 4, false);
    else GO(8, 2, false);
#undef GO
    const int blocks = (NP + 127) / 128 * R;
    k_outer_sum<T, RCONT><<<(unsigned)L * blocks, 256, 0, st>>>(
        part, R16, strips * PC, rows, shift, (T*)out, NP, R, blocks);
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

// `part` (splits, N, R16) is left unsummed for launch_shrink_sum where splits > 1.
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

void launch_shrink_sum(int type, int R, const int* order, const int* segs, const int* adapter,
                       int S, int Bn, long T, const float* scale, float scale_all, void* V,
                       const float* part, int splits, hipStream_t st) {
    const Rows rows{order, (const int4*)segs, adapter, S, Bn, T};
    const Scale sc{scale, scale_all};
    const int RP = lowrank_rp(R), R16 = r16_of(R);
    const long N = T * Bn, blocks = (N * RP + 255) / 256;
    if (type == LM_BF16)
        k_shrink_sum<bf16_t><<<(unsigned)blocks, 256, 0, st>>>(part, N, R16, splits, rows, sc,
                                                               (bf16_t*)V, RP);
    else
        k_shrink_sum<f16_t><<<(unsigned)blocks, 256, 0, st>>>(part, N, R16, splits, rows, sc,
                                                              (f16_t*)V, RP);
}

void launch_expand(int type, int rcont, const void* base, long bs, void* out, long os,
                   const void* V, const void* W, int M, int R, const int* order, const int* segs,
                   const int* adapter, const long* counts, int S, int Bn, long T,
                   hipStream_t st) {
    const Rows rows{order, (const int4*)segs, adapter, S, Bn, T};
    // rows a workgroup: as many as leave four workgroups a CU, 256 at most, 32 at least
    const long strips = (M + 255) / 256;
    int shift = 8;
    while (shift > 5 && tiles_of(counts, S, T, shift) * strips < 1024) --shift;
    const int tiles = tiles_of(counts, S, T, shift), RP = lowrank_rp(R);
    if (tiles == 0) return;
    if (type == LM_BF16)
        rcont ? expand<bf16_t, true>(base, bs, out, os, V, RP, W, M, R, rows, tiles, shift, st)
              : expand<bf16_t, false>(base, bs, out, os, V, RP, W, M, R, rows, tiles, shift, st);
    else
        rcont ? expand<f16_t, true>(base, bs, out, os, V, RP, W, M, R, rows, tiles, shift, st)
              : expand<f16_t, false>(base, bs, out, os, V, RP, W, M, R, rows, tiles, shift, st);
}

int lowrank_strips(int NP, int R) { return (NP + outer_columns(R) - 1) / outer_columns(R); }
// log2 of the rows that one partial gradient sums: about four workgroups a CU over the strips,
// never fewer than 64 rows (a step) nor more than 4096.
int lowrank_outer_shift(const long* counts, int S, long T, int NP, int R) {
    const long strips = lowrank_strips(NP, R);
    int shift = 12;
    while (shift > 6 && tiles_of(counts, S, T, shift) * strips < 1024) --shift;
    return shift;
}
int lowrank_outer_tiles(const long* counts, int S, long T, int shift) {
    return tiles_of(counts, S, T, shift);
}
// Whether the backward pass reads dy once for u and dB (k_outer's DV): not where the shares of u
// would be as many bytes as dy.
int lowrank_one_reading(int R) { return R <= 32; }

void launch_outer(int type, int rcont, const void* P, long ps, int NP, const void* Q, float* part,
                  const void* W, float* partv, const int* order, const int* segs,
                  const int* adapter, const long* counts, int S, int Bn, long T, int shift,
                  void* out, int R, int L, hipStream_t st) {
    const Rows rows{order, (const int4*)segs, adapter, S, Bn, T};
    const int tiles = tiles_of(counts, S, T, shift), RP = lowrank_rp(R);
    const long N = T * Bn;
    if (type == LM_BF16)
        rcont ? outer<bf16_t, true>(P, ps, NP, Q, RP, part, W, partv, N, rows, tiles, shift, out,
                                    R, L, st)
              : outer<bf16_t, false>(P, ps, NP, Q, RP, part, W, partv, N, rows, tiles, shift, out,
                                     R, L, st);
    else
        rcont ? outer<f16_t, true>(P, ps, NP, Q, RP, part, W, partv, N, rows, tiles, shift, out,
                                   R, L, st)
              : outer<f16_t, false>(P, ps, NP, Q, RP, part, W, partv, N, rows, tiles, shift, out,
                                    R, L, st);
}

}  // extern "C"
