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
// contraction at a time in the stream's own layout; accumulation, split sums, partial gradients,
// v and u are fp32.  v and u meet the matrix instructions in parts of the type that add up to them
// (`in_parts`): of 16-bit v the products would carry 2^-8 of error, and an fp16 v beyond 65504 is
// an infinity where the result need not be.  Each result is rounded once.
//
// Rows come grouped by adapter.  Sequences are time-major, row = t * Bn + column, and an adapter
// belongs to a column, so only the Bn columns are grouped: segment s lists its columns in
// `order[start, start + count)`, and its T * count rows are enumerated time-major.
#include "lm_common.h"

#include <algorithm>

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

// Eight neighbours from element e of a matrix that has `limit` elements, without a branch: near
// the very end the last eight are taken, and `trim` shifts them into place.  Loads that differ
// from lane to lane in their form would wait for each other at the point where they join.
template <typename T> DEVINL typename Frag<T>::type eight(const T* p, long e, long limit) {
    return __builtin_bit_cast(typename Frag<T>::type,
                              *(const typename Vec8<T>::type*)(p + min(e, limit - 8)));
}
// The same of a matrix that is read once in whole lines and need not stay in the caches: outer's
// P (65536 rows of 4096: 129 -> 104 us).  Not of base or x, whose lines several loads share, nor
// of the distilled logits, which are written next (all three slower).
template <typename T>
DEVINL typename Frag<T>::type eight_once(const T* p, long e, long limit) {
    return __builtin_bit_cast(
        typename Frag<T>::type,
        __builtin_nontemporal_load((const typename Vec8<T>::type*)(p + min(e, limit - 8))));
}
// What `eight` gave for element e, with zeros for all but the first `left`.
template <typename F> DEVINL F trim(F v, long e, long limit, int left) {
    typedef unsigned long long u2 __attribute__((ext_vector_type(2)));
    u2 u = __builtin_bit_cast(u2, v);
    const int over = (int)(e - min(e, limit - 8)), s = over * 16;
    if (over >= 8) u = u2{0, 0};
    else if (s >= 64) u = u2{u[1] >> (s - 64), 0};
    else if (s > 0) u = u2{u[0] >> s | u[1] << (64 - s), u[1] >> s};
    const int keep = min(max(left, 0), 8) * 16;
    if (keep < 64) u = u2{u[0] & ((1ull << keep) - 1), 0};
    else if (keep < 128) u = u2{u[0], u[1] & ((1ull << (keep - 64)) - 1)};
    return __builtin_bit_cast(F, u);
}

// An fp32 number as the sum of a 16-bit type's, operands of as many matrix instructions.  All parts
// have the number's sign, and none is zero unless it is: an infinity in the other operand then
// gives that infinity, where plus and minus or zero times infinity would give NaN.
//
// bf16 has fp32's range and a third of its digits: three parts, each but the last cut off, and the
// last one's digits fit.  Where nothing is left, 2^-30 of the first.
constexpr int parts_of(bool fp16) { return fp16 ? 2 : 3; }
DEVINL void in_parts(float v, bf16_t (&p)[3]) {
    auto cut = [](float x) { return __int_as_float(__float_as_int(x) & 0xffff0000); };
    const float a = cut(v), least = a * 0x1p-30f;
    const float r = v - a, b = fabsf(r) > 0.f ? cut(r) : least;         // of infinity r is NaN
    const float q = r - b, c = fabsf(q) > 0.f ? q : least;
    p[0] = __builtin_bit_cast(bf16_t, (short)(__float_as_int(a) >> 16));
    p[1] = __builtin_bit_cast(bf16_t, (short)(__float_as_int(b) >> 16));
    p[2] = __builtin_bit_cast(bf16_t, (short)(__float_as_int(c) >> 16));
}
// fp16 has not the range: a row's numbers come scaled by a power of two that brings the largest to
// [2^14, 2^15).  Two parts: 22 digits, and an error of 2^-37 of the largest at most.
DEVINL void in_parts(float v, f16_t (&p)[2]) {
    const f16_t least = (f16_t)(v > 0.f ? 0x1p-24f : v < 0.f ? -0x1p-24f : 0.f);
    f16_t a = (f16_t)__builtin_amdgcn_cvt_pkrtz(v, 0.f)[0];
    if (a == (f16_t)0.f) a = least;
    const float r = v - (float)a;
    const f16_t b = (f16_t)r;
    p[0] = a;
    p[1] = fabsf(r) > 0.f && b != (f16_t)0.f && (r > 0.f) == (v > 0.f) ? b : least;
}
// The exponent of that power's inverse for numbers of which m is the largest finite one; of zeros
// alone -120, so that both powers are normal numbers.
DEVINL int shift_of(float m) { return max((__float_as_int(m) >> 23) - 127 - 14, -120); }
DEVINL float two_to(int e) { return __int_as_float((127 + e) << 23); }
DEVINL float finite_size(float x) { return fabsf(x) < __builtin_huge_valf() ? fabsf(x) : 0.f; }

// Eight parts times two to e <= 0, none of them zero that was not: 1, as bits, is 2^-24.
DEVINL bf16x8 shifted(bf16x8 v, int) { return v; }
DEVINL f16x8 shifted(f16x8 v, int e) {
    typedef unsigned short u16x8 __attribute__((ext_vector_type(8)));
    const u16x8 was = __builtin_bit_cast(u16x8, v);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = __builtin_amdgcn_ldexph(v[j], (short)e);
    const u16x8 least = __builtin_elementwise_min(was & (unsigned short)0x7fff, (u16x8)1);
    const u16x8 size = __builtin_bit_cast(u16x8, v) & (unsigned short)0x7fff;
    return __builtin_bit_cast(f16x8, __builtin_elementwise_max(size, least) |
                                         was & (unsigned short)0x8000);
}

// A row of v or u in memory: its parts one behind the other, R16 numbers each, and fp16's shift.
__host__ __device__ constexpr int row_length(bool fp16, int R16) {
    return fp16 ? 2 * R16 + 8 : 3 * R16;
}
template <typename T> DEVINL int row_shift(const T* row, int R16) {
    return *(const int*)(row + 2 * R16);
}

// The bits of a vector's first `left` elements, and the vector without the others.
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
DEVINL u32x4 first_bits(int left) {
    u32x4 m;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        m[i] = left >= 2 * i + 2 ? ~0u : left == 2 * i + 1 ? 0xffffu : 0u;
    return m;
}
template <typename F> DEVINL F keep(F v, u32x4 m) {
    return __builtin_bit_cast(F, __builtin_bit_cast(u32x4, v) & m);
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

// Workgroups go round the eight XCDs by their number, each with an L2 of its own.  This order
// hands an XCD neighbouring work: strips that share a line at their border (rows of an odd width
// have no aligned ones) meet in one L2, also half-written.
DEVINL int by_xcd() {
    const int n = gridDim.x, b = blockIdx.x, x = b & 7, q = n >> 3, r = n & 7;
    return x * q + (x < r ? x : r) + (b >> 3);
}

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

// The sum over a wave's lanes up to one's own: by shifts in rows of 16 lanes, then from the last
// lane of a row to the next ones (every lane of the wave has to be there).
DEVINL int running_sum(int x) {
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);     // row_shr:1
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);     // row_shr:2
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);     // row_shr:4
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);     // row_shr:8
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);     // row_bcast:15
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);     // row_bcast:31
    return x;
}

// The largest of a wave's numbers, none below `least`, the same way.
DEVINL int wave_largest(int x, int least) {
    x = max(x, __builtin_amdgcn_update_dpp(least, x, 0x111, 0xf, 0xf, false));
    x = max(x, __builtin_amdgcn_update_dpp(least, x, 0x112, 0xf, 0xf, false));
    x = max(x, __builtin_amdgcn_update_dpp(least, x, 0x114, 0xf, 0xf, false));
    x = max(x, __builtin_amdgcn_update_dpp(least, x, 0x118, 0xf, 0xf, false));
    x = max(x, __builtin_amdgcn_update_dpp(least, x, 0x142, 0xa, 0xf, false));
    x = max(x, __builtin_amdgcn_update_dpp(least, x, 0x143, 0xc, 0xf, false));
    return __builtin_amdgcn_readlane(x, 63);
}

// Which rows tile number `tile` holds.  A wave sums up the segments' tiles, 64 at a time.
DEVINL Tile find_tile(const Rows& r, int tile, int shift) {
    const int lane = threadIdx.x & 63;
    int base = 0;
    Tile f{-1, 0, 0, 0, 0, 0};
    for (int s0 = 0; s0 < r.S; s0 += 64) {
        const int s = s0 + lane;
        const int4 g = s < r.S ? r.segs[s] : make_int4(-1, 0, 0, 0);
        const int t = (int)((r.T * g.z + (1l << shift) - 1) >> shift);
        const int sum = running_sum(t);
        const unsigned long long hit = __ballot(base + sum > tile);
        if (hit) {
            const int at = __ffsll(hit) - 1;
            f.adapter = __builtin_amdgcn_readlane(g.x, at);
            f.start = __builtin_amdgcn_readlane(g.y, at);
            f.count = __builtin_amdgcn_readlane(g.z, at);
            f.first = base + __builtin_amdgcn_readlane(sum - t, at);
            f.n = r.T * f.count;
            f.j0 = (long)(tile - f.first) << shift;
            return f;
        }
        base += __builtin_amdgcn_readlane(sum, 63);
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
// shrink: V[row] = s_l X[row] W_l.  A workgroup takes 64 rows of one adapter and `kper` of the
// contraction, 256 a step: rows come in 512 neighbouring bytes each (in the operand's own layout,
// 64 at a time, 65536 rows of 1024 took 48 us from memory, now 26) and pass through LDS with W's
// panel, the next step's on their way meanwhile; a wave multiplies 16 of the rows.
// ---------------------------------------------------------------------------
constexpr int S_TM = 6;     // log2 rows a workgroup
constexpr int S_KC = 256;   // contraction a step

template <typename T, int RT, bool KCONT>
__global__ __launch_bounds__(256) void k_shrink(const T* __restrict__ X, long xs, long xlimit,
                                                const T* __restrict__ W, long wlimit, int K, int R,
                                                Rows rows, Scale scale, T* __restrict__ V,
                                                float* __restrict__ part, long N, int splits,
                                                int kper) {
    typedef typename Frag<T>::type F;
    // rows of the panel: R of the contraction each (KCONT), or 256 of R each
    constexpr int LX = S_KC + 8, LD = KCONT ? S_KC + 8 : RT * 16 + (RT >= 4 ? 16 : 0);
    __shared__ __attribute__((aligned(16))) T xt[64 * LX];
    __shared__ __attribute__((aligned(16))) T w[(KCONT ? RT * 16 : S_KC) * LD];
    __shared__ int at[64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 4;
    const int split = blockIdx.x % splits;
    const Tile f = find_tile(rows, blockIdx.x / splits, S_TM);
    if (f.adapter < 0) return;
    if (tid < 64) at[tid] = (int)row_of(rows, f, min(f.j0 + tid, f.n - 1));
    const long wl = (long)f.adapter * K * R;
    const int kend = min(K, (split + 1) * kper);
    f32x4 acc[RT];
#pragma unroll
    for (int t = 0; t < RT; ++t) acc[t] = f32x4{0, 0, 0, 0};
    __syncthreads();

    constexpr int XV = 64 * S_KC / 8 / 256, WV = RT * 2;    // vectors a thread
    F x[XV], wv[WV];
    // element of W that vector i starts with, and how many of it belong to the panel
    auto of_panel = [&](int i, int k0, int& left) {
        const int u = i * 256 + tid;
        if (KCONT) {
            const int r = u / (S_KC / 8), k = k0 + u % (S_KC / 8) * 8;
            left = r < R ? kend - k : 0;
            return wl + (long)r * K + k;
        }
        const int k = k0 + u / (RT * 2), r = u % (RT * 2) * 8;
        left = k < kend ? R - r : 0;
        return wl + (long)k * R + r;
    };
    auto of_rows = [&](int i, int k0) { return at[i * 8 + tid / 32] * xs + k0 + tid % 32 * 8; };
    auto load = [&](int k0) {
#pragma unroll
        for (int i = 0; i < XV; ++i) x[i] = eight_once(X, of_rows(i, k0), xlimit);
#pragma unroll
        for (int i = 0; i < WV; ++i) {
            int left;
            wv[i] = eight(W, of_panel(i, k0, left), wlimit);
        }
    };
    int k0 = split * kper;
    if (k0 < kend) load(k0);
    for (; k0 < kend; k0 += S_KC) {
        const bool tail = k0 + S_KC > kend;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < XV; ++i) {
            if (tail) x[i] = trim(x[i], of_rows(i, k0), xlimit, kend - k0 - tid % 32 * 8);
            *(F*)(xt + (i * 8 + tid / 32) * LX + tid % 32 * 8) = x[i];
        }
#pragma unroll
        for (int i = 0; i < WV; ++i) {
            const int u = i * 256 + tid, n = KCONT ? S_KC / 8 : RT * 2;
            if (tail || R != RT * 16) {
                int left;
                const long e = of_panel(i, k0, left);
                wv[i] = trim(wv[i], e, wlimit, left);
            }
            *(F*)(w + u / n * LD + u % n * 8) = wv[i];
        }
        __syncthreads();
        if (k0 + S_KC < kend) load(k0 + S_KC);
#pragma unroll
        for (int s = 0; s < S_KC / 32; ++s) {
            const F a = *(const F*)(xt + (wave * 16 + (lane & 15)) * LX + s * 32 + g * 8);
#pragma unroll
            for (int t = 0; t < RT; ++t)
                acc[t] = mfma(a,
                              KCONT ? *(const F*)(w + (t * 16 + (lane & 15)) * LD + s * 32 + g * 8)
                                       : column_frag(w, LD, s * 32, t * 16 + own_columns()),
                              acc[t]);
        }
    }
    const float sc = scale(f.adapter);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int n = wave * 16 + g * 4 + i;
        if (f.j0 + n >= f.n) continue;
        const long r = at[n];
        if (part) {
            float* p = part + ((long)split * N + r) * (RT * 16) + (lane & 15);
#pragma unroll
            for (int t = 0; t < RT; ++t) p[t * 16] = acc[t][i];
        } else {
            constexpr bool SCALED = __is_same(T, f16_t);
            constexpr int NQ = parts_of(SCALED);
            float x[RT], m = 0.f;
#pragma unroll
            for (int t = 0; t < RT; ++t) {      // zeros behind R, where an infinity left NaN
                x[t] = t * 16 + (lane & 15) < R ? acc[t][i] * sc : 0.f;
                m = fmaxf(m, finite_size(x[t]));
            }
            T* v = V + r * row_length(SCALED, RT * 16);
            int e = 0;
            if (SCALED) {
#pragma unroll
                for (int off = 8; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor(m, off, 64));
                e = shift_of(m);
                if ((lane & 15) == 0) *(int*)(v + 2 * RT * 16) = e;
            }
#pragma unroll
            for (int t = 0; t < RT; ++t) {
                T p[NQ];
                in_parts(SCALED ? x[t] * two_to(-e) : x[t], p);
#pragma unroll
                for (int j = 0; j < NQ; ++j) v[(j * RT + t) * 16 + (lane & 15)] = p[j];
            }
        }
    }
}

// The shares summed in a fixed order and scaled; four of a row's R a thread.  GR groups of threads
// take every GR-th share where there are many (98 of 8192 rows, rank 32).
template <typename T, int GR>
__global__ __launch_bounds__(256) void k_shrink_sum(const float* __restrict__ part, long N, int R,
                                                    int R16, int splits, Rows rows, Scale scale,
                                                    T* __restrict__ V) {
    typedef T out4 __attribute__((ext_vector_type(4)));
    constexpr bool SCALED = __is_same(T, f16_t);
    constexpr int TH = 256 / GR, NQ = parts_of(SCALED);
    __shared__ f32x4 sums[GR > 1 ? 256 : 1];
    const int group = threadIdx.x / TH;
    const long i = (long)blockIdx.x * TH + threadIdx.x % TH;
    const long row = i / (R16 / 4);
    const int r = (int)(i % (R16 / 4)) * 4;
    const int l = row < N ? rows.adapter[(unsigned)row % (unsigned)rows.Bn] : -1;
    f32x4 s = f32x4{0, 0, 0, 0};
    if (l >= 0) {
        const float* p = part + row * R16 + r;
#pragma unroll 8
        for (int k = group; k < splits; k += GR) s += *(const f32x4*)(p + (long)k * N * R16);
    }
    if (GR > 1) {
        sums[threadIdx.x] = s;
        __syncthreads();
        if (group) return;
#pragma unroll
        for (int k = 1; k < GR; ++k) s += sums[k * TH + threadIdx.x];
    }
    if (l < 0) return;
    const float sc = scale(l);
    T* v = V + row * row_length(SCALED, R16);
    float m = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        s[j] = r + j < R ? s[j] * sc : 0.f;
        m = fmaxf(m, finite_size(s[j]));
    }
    if (SCALED) {               // a row's threads are neighbours in a wave
        for (int off = R16 / 8; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor(m, off, 64));
        const int e = shift_of(m);
        if (r == 0) *(int*)(v + 2 * R16) = e;
        s *= two_to(-e);
    }
    out4 o[NQ];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        T p[NQ];
        in_parts(s[j], p);
#pragma unroll
        for (int k = 0; k < NQ; ++k) o[k][j] = p[k];
    }
#pragma unroll
    for (int k = 0; k < NQ; ++k) *(out4*)(v + k * R16 + r) = o[k];
}

// ---------------------------------------------------------------------------
// expand: out[row] = base[row] + V[row] W_l (base may be out itself, or absent: zero).  A wave
// keeps W for 64 columns in registers and multiplies 32 of the workgroup's rows at a time.  W is
// the A operand and the rows are B's columns, so that a lane holds four neighbouring columns of
// one row; the products pass through LDS in fp32 to the lanes that hold base for whole rows of
// 256 columns: read and written as 512 neighbouring bytes (in the operand's layout, 64 at a time,
// rows of 50000 ran at 3.5 TB/s), loaded one step ahead.  V's parts pass through LDS too, a step
// ahead and read once a workgroup: every wave needs all of them, and in registers they cost rank
// 128 half of its waves (16384 rows of 4096: 137 us, now 74).  dx, a stream of stores alone, runs
// with a fourth workgroup a CU (65536 rows of 1024: 42 -> 36 us; with base 203 -> 205).
// ---------------------------------------------------------------------------
template <typename T, int RK, bool RCONT>
__global__ __launch_bounds__(256, RCONT && RK == 1 ? 4 : 1)
void k_expand(const T* base, long bs, long blimit, T* out, long os, const T* __restrict__ V,
              int R16, const T* __restrict__ W, long wlimit, int M, int R, Rows rows, int strips,
              int shift) {
    typedef typename Frag<T>::type F;
    typedef typename Vec8<T>::type U8;
    constexpr bool SCALED = __is_same(T, f16_t);
    constexpr int LD = 256 + 16, LS = 256 + 4, NQ = parts_of(SCALED);
    // V's rows of a step, part by part; eight more keep neighbouring rows in other banks
    constexpr int VR = RK * 4, VL = NQ * RK * 32 + 8, NV = (32 * NQ * VR + 255) / 256;
    constexpr int WB = RCONT ? 0 : RK * 32 * LD * 2, SB = 32 * LS * 4, STEP = SB + 32 * VL * 2;
    __shared__ __attribute__((aligned(16))) char lds[WB > STEP ? WB : STEP];
    __shared__ int at[256];                     // the tile's rows, divided out once
    T* const wt = (T*)lds;                      // W, and when it is in registers
    float* const sums = (float*)lds;            // the products
    T* const vt = (T*)(lds + SB);               // and V
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 4;
    const int block = by_xcd();
    const Tile f = find_tile(rows, block / strips, shift);
    const int strip = block % strips * 256, m0 = strip + wave * 64;
    const long LV = row_length(SCALED, R16);
    const bool mine = f.adapter >= 0;
    if (!mine && base == out) return;           // nothing to add in place
    const long jend = min(f.n, f.j0 + (1l << shift));
    if (f.j0 + tid < jend) at[tid] = (int)row_of(rows, f, f.j0 + tid);
    F w[RK][4];
    if (mine) {
        const long wl = (long)f.adapter * M * R;
        if (RCONT) {
#pragma unroll
            for (int k = 0; k < RK; ++k)
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    const int m = m0 + t * 16 + (lane & 15), r = k * 32 + g * 8;
                    const long e = wl + (long)m * R + r;
                    w[k][t] = trim(eight(W, e, wlimit), e, wlimit, m < M ? R - r : 0);
                }
        } else {
            F v[RK * 4];
#pragma unroll
            for (int i = 0; i < RK * 4; ++i) {
                const int u = i * 256 + tid;
                v[i] = eight(W, wl + (long)(u / 32) * M + strip + u % 32 * 8, wlimit);
            }
#pragma unroll
            for (int i = 0; i < RK * 4; ++i) {
                const int u = i * 256 + tid, r = u / 32, m = strip + u % 32 * 8;
                if (R != RK * 32 || strip + 256 > M)
                    v[i] = trim(v[i], wl + (long)r * M + m, wlimit, r < R ? M - m : 0);
                *(F*)(wt + r * LD + u % 32 * 8) = v[i];
            }
        }
    }
    __syncthreads();
    // a lane's share of base and out: eight columns of every eighth row
    const int m = strip + (tid & 31) * 8;
    const bool whole = m + 8 <= M;
    F y[4], v[NV];
    int shifts[2], next_shifts[2];
    auto load_base = [&](long j0) {
        if (!base) return;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const long j = j0 + i * 8 + (tid >> 5);
            y[i] = eight(base, at[(j < jend ? j : jend - 1) - f.j0] * bs + m, blimit);
        }
    };
    auto load_rows = [&](long j0) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int u = i * 256 + tid, n = u / VR % 32, c = u % VR * 8;
            const long j = j0 + n, row = at[(j < jend ? j : jend - 1) - f.j0];
            const bool there = RK > 1 || c < R16;       // zeros up to a contraction of 32
            v[i] = *(const F*)(V + row * LV + min(u / VR / 32, NQ - 1) * R16 + (there ? c : 0));
            if (!there) v[i] = F{};
        }
        if (SCALED)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const long j = j0 + h * 16 + (lane & 15);
                next_shifts[h] = row_shift(V + at[(j < jend ? j : jend - 1) - f.j0] * LV, R16);
            }
    };
    auto store_rows = [&]() {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int u = i * 256 + tid;
            if (u < 32 * NQ * VR)
                *(F*)(vt + u / VR % 32 * VL + u / VR / 32 * RK * 32 + u % VR * 8) = v[i];
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) shifts[h] = next_shifts[h];
    };
    if (mine) load_rows(f.j0);
    load_base(f.j0);
    if (mine && !RCONT) {
#pragma unroll
        for (int k = 0; k < RK; ++k)
#pragma unroll
            for (int t = 0; t < 4; ++t)
                w[k][t] = column_frag(wt, LD, k * 32, wave * 64 + t * 16 + own_columns());
    }
    __syncthreads();                            // W is read
    if (mine) {
        store_rows();
        load_rows(f.j0 + 32);
    }
    __syncthreads();
    auto multiply = [&](f32x4 (&acc)[2][4]) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const T* row = vt + (h * 16 + (lane & 15)) * VL + g * 8;
#pragma unroll
            for (int t = 0; t < 4; ++t) acc[h][t] = f32x4{0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < NQ; ++i)
#pragma unroll
                for (int k = 0; k < RK; ++k) {
                    const F p = *(const F*)(row + (i * RK + k) * 32);
#pragma unroll
                    for (int t = 0; t < 4; ++t) acc[h][t] = mfma(w[k][t], p, acc[h][t]);
                }
            if (SCALED)                         // a lane's column of D is a row
#pragma unroll
                for (int t = 0; t < 4; ++t) acc[h][t] *= two_to(shifts[h]);
        }
    };
    auto to_lds = [&](const f32x4 (&acc)[2][4]) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int t = 0; t < 4; ++t)
                *(f32x4*)(sums + (h * 16 + (lane & 15)) * LS + wave * 64 + t * 16 + g * 4) =
                    acc[h][t];
    };
    long j0 = f.j0;
    // Whole steps: loads and stores without a condition, so that a wait for a load counts exactly
    // the younger ones and does not drain the stores.
    if (mine && strip + 256 <= M) {
        for (; j0 + 32 <= jend; j0 += 32) {
            f32x4 acc[2][4];
            multiply(acc);
            __syncthreads();                    // V and the last step's products are read
            to_lds(acc);
            store_rows();
            load_rows(j0 + 64);
            __syncthreads();
            U8 o[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int n = i * 8 + (tid >> 5);
                const f32x4 lo = *(const f32x4*)(sums + n * LS + (tid & 31) * 8);
                const f32x4 hi = *(const f32x4*)(sums + n * LS + (tid & 31) * 8 + 4);
#pragma unroll
                for (int q = 0; q < 8; ++q)
                    o[i][q] = (T)((base ? (float)y[i][q] : 0.f) + (q < 4 ? lo[q & 3] : hi[q & 3]));
            }
            load_base(j0 + 32);
#pragma unroll
            for (int i = 0; i < 4; ++i)
                *(U8*)(out + at[j0 + i * 8 + (tid >> 5) - f.j0] * os + m) = o[i];
        }
    }
    for (; j0 < jend; j0 += 32) {
        f32x4 acc[2][4];
        if (mine) multiply(acc);
        __syncthreads();
        if (mine) {
            to_lds(acc);
            store_rows();
            load_rows(j0 + 64);
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int n = i * 8 + (tid >> 5);
            if (j0 + n >= jend || m >= M) continue;
            const long row = at[j0 + n - f.j0];
            f32x4 lo = f32x4{0, 0, 0, 0}, hi = lo;
            if (mine) {
                lo = *(const f32x4*)(sums + n * LS + (tid & 31) * 8);
                hi = *(const f32x4*)(sums + n * LS + (tid & 31) * 8 + 4);
            }
            if (whole) {
                U8 o;
#pragma unroll
                for (int q = 0; q < 8; ++q)
                    o[q] = (T)((base ? (float)y[i][q] : 0.f) + (q < 4 ? lo[q & 3] : hi[q & 3]));
                *(U8*)(out + row * os + m) = o;
            } else {
                const F was = trim(y[i], row * bs + m, blimit, M - m);
#pragma unroll
                for (int q = 0; q < 8; ++q)
                    if (m + q < M)
                        out[row * os + m + q] =
                            (T)((base ? (float)was[q] : 0.f) + (q < 4 ? lo[q & 3] : hi[q & 3]));
            }
        }
        if (j0 + 32 < jend) load_base(j0 + 32);
    }
}

// ---------------------------------------------------------------------------
// The same for a decode step, where an adapter has a row or a few and its weights are most of
// what is read: a wave takes 512 columns, eight a lane, and up to four rows, and multiplies W as
// it comes, whole lines of one r, without staging.  The shares of V are summed here, which saves
// the launch that does it elsewhere.
// ---------------------------------------------------------------------------
constexpr int FEW = 2;      // log2 rows a wave

// v = s x A of the rows `at`, from the shares of x A.
DEVINL void sum_shares(const float* __restrict__ part, const int* at, int n, long N, int R16,
                       int splits, float scale, float* v) {
    for (int u = threadIdx.x; u < n * R16; u += 64) {
        const int i = u / R16, r = u - i * R16;
        const float* p = part + (long)at[i] * R16 + r;
        float s = 0.f;
#pragma unroll 8
        for (int k = 0; k < splits; ++k) s += p[(long)k * N * R16];
        v[i * 128 + r] = s * scale;
    }
    __syncthreads();
}

template <typename T>
__global__ __launch_bounds__(64) void k_expand_few(const T* base, long bs, T* out, long os,
                                                   const float* __restrict__ part, long N, int R16,
                                                   int splits, Scale scale,
                                                   const T* __restrict__ W, int M, int R,
                                                   Rows rows, int strips) {
    constexpr int NR = 1 << FEW, U = 16;
    typedef typename Vec8<T>::type U8;
    __shared__ float v[NR * 128];
    __shared__ int at[NR];
    const int lane = threadIdx.x;
    const Tile f = find_tile(rows, blockIdx.x / strips, FEW);
    const bool mine = f.adapter >= 0;
    if (!mine && base == out) return;
    const int n = (int)min((long)NR, f.n - f.j0), own = blockIdx.x % strips * 512 + lane * 8;
    // The last lane of an odd width takes the last eight columns, and stores those that are its
    // own; lanes behind it take them too and store nothing.
    const bool whole = M >= 8;
    const int m = whole && own > M - 8 ? M - 8 : own;
    // What is read goes out without conditions (a row behind the last is the first again), the
    // rows' numbers first: W is on its way while they come, base and V while W does.
    const unsigned j = (unsigned)f.j0 + (lane < n ? lane : 0), c = f.count, t = j / c;
    const int column = rows.order[f.start + (j - t * c)];
    const T* Wl = W + (long)(mine ? f.adapter : 0) * M * R + m;
    U8 w[U];
    auto load = [&](int r0) {
#pragma unroll
        for (int u = 0; u < U; ++u) w[u] = *(const U8*)(Wl + (long)min(r0 + u, R - 1) * M);
    };
    if (whole) {
        load(0);
        if (lane < NR) at[lane] = (int)t * rows.Bn + column;
        __syncthreads();
        long row[NR];
        U8 y[NR];
#pragma unroll
        for (int i = 0; i < NR; ++i) {
            row[i] = at[i];
            y[i] = *(const U8*)(base + row[i] * bs + m);
        }
        float acc[NR][8] = {};
        if (mine) {
            sum_shares(part, at, n, N, R16, splits, scale(f.adapter), v);
            for (int r0 = 0; r0 < R; r0 += U) {
                if (r0) load(r0);
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (r0 + u < R)
#pragma unroll
                        for (int i = 0; i < NR; ++i)
                            if (i < n)
#pragma unroll
                                for (int q = 0; q < 8; ++q)
                                    acc[i][q] += v[i * 128 + r0 + u] * (float)w[u][q];
            }
        }
#pragma unroll
        for (int i = 0; i < NR; ++i) {
            if (i >= n) continue;
            float o[8];
#pragma unroll
            for (int q = 0; q < 8; ++q) o[q] = (float)y[i][q] + acc[i][q];
            if (m == own) store8(out + row[i] * os + m, o);
            else
#pragma unroll
                for (int q = 0; q < 8; ++q)
                    if (m + q >= own) out[row[i] * os + m + q] = (T)o[q];
        }
        return;
    }
    if (lane < NR) at[lane] = (int)t * rows.Bn + column;
    __syncthreads();
    if (mine) sum_shares(part, at, n, N, R16, splits, scale(f.adapter), v);
    for (int i = 0; i < n; ++i)
        for (int q = lane; q < M; q += 64) {            // fewer than eight columns
            float s = (float)base[at[i] * bs + q];
            if (mine)
                for (int r = 0; r < R; ++r) s += v[i * 128 + r] * (float)Wl[(long)r * M + q - m];
            out[at[i] * os + q] = (T)s;
        }
}

// ---------------------------------------------------------------------------
// outer: part[tile][r][p] = sum over the tile's rows of P[row][p] Q[row][r].  A workgroup owns 64
// CT columns and walks the tile's rows 64 at a time: they pass through LDS as they are, and both
// operands are read from there with their columns' rows side by side.
//
// fp16's rows of Q have shifts of their own, and a sum over rows has to have one: the largest so
// far.  A row's parts are scaled to it on the way into LDS, and the sums when it grows.
//
// NS > 0: the rows meet W on the way too, partv[share][row][r] = sum over the workgroup's columns
// of P[row][p] W_l[r][p] -- the backward pass's u, in shares of NS times as many columns.  dy is
// then read once for both; a share costs 8 R bytes a row (written, read again), a second reading
// of dy 128 CT NS.
// ---------------------------------------------------------------------------
template <typename T, int RT, int CT, int NS>
__global__ __launch_bounds__(256) void k_outer(const T* __restrict__ P, long ps, long plimit,
                                               int NP, const T* __restrict__ Q,
                                               float* __restrict__ part,
                                               const T* __restrict__ W, long wlimit, int R,
                                               float* __restrict__ partv, long N,
                                               T* __restrict__ whole, int rcont, Rows rows,
                                               int shares, int shift) {
    typedef typename Frag<T>::type F;
    constexpr bool DV = NS > 0;
    constexpr int C = DV ? NS : 1;                  // strips of PC columns
    constexpr bool SCALED = __is_same(T, f16_t);
    constexpr int PC = 64 * CT, S = PC / 32, LP = PC + 16, LQ = RT * 16 + (RT >= 4 ? 16 : 0);
    constexpr int LW = C * PC + 8, NQ = parts_of(SCALED);
    constexpr int R16 = RT * 16;
    constexpr long LV = row_length(SCALED, R16);
    __shared__ __attribute__((aligned(16))) T pt[64 * LP];
    __shared__ __attribute__((aligned(16))) T qt[NQ][64 * LQ];
    __shared__ __attribute__((aligned(16))) T wt[DV ? RT * 16 * LW : 8];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 4;
    const int block = by_xcd(), tile = block / shares, share = block % shares;
    const int p0 = share * C * PC;
    const Tile f = find_tile(rows, tile, shift);
    if (f.adapter < 0) return;
    if (DV) {
#pragma unroll 4
        for (int u = tid; u < RT * 16 * (C * PC / 8); u += 256) {
            const int r = u / (C * PC / 8), c = u % (C * PC / 8) * 8;
            const long e = (long)f.adapter * NP * R + (long)r * NP + p0 + c;
            *(F*)(wt + r * LW + c) = trim(eight(W, e, wlimit), e, wlimit, r < R ? NP - p0 - c : 0);
        }
    }
    // A wave takes all of the ranks and a fourth of the columns; of many ranks a part and more of
    // the columns, so that fewer operands are read from LDS (rank 128: 28 a step instead of 52).
    constexpr int WR = RT == 8 ? 4 : RT == 4 ? 2 : 1, RW = RT / WR, CW = CT * WR;
    const int ct0 = wave / WR * CW, rt0 = wave % WR * RW;
    f32x4 acc[C][CW][RW];
#pragma unroll
    for (int k = 0; k < C; ++k)
#pragma unroll
        for (int c = 0; c < CW; ++c)
#pragma unroll
            for (int t = 0; t < RW; ++t) acc[k][c][t] = f32x4{0, 0, 0, 0};
    const long jend = min(f.n, f.j0 + (1l << shift));
    constexpr int QV = (64 * RT * 2 + 255) / 256;       // vectors of Q a thread
    constexpr int PV = 64 * PC / 8 / 256, PW = PC / 8;  // of P; a row's
    constexpr int D = C > 1 ? 2 : 1;                    // strips of P ahead
    F x[D][PV], q[QV][NQ];
    int shifts[QV], shift_of_lane = -120, shift_q = -120;   // of a vector's row; the sums'
    // Loads and stores end in the order they went out, and a wait for a load has to know how many
    // are younger: so nothing in the loop goes out on a condition (rows behind the last are the
    // last again), or the wait would drain all of them (8192 rows of 50000 in one group, a
    // workgroup a CU: 280 us, now 215).
    // Rows of this step (for u), the next (loading) and the one behind it: row t Bn + column.
    __shared__ int at[3][64];
    auto find_row = [&](long j0, int& tb) {
        const long k = j0 + lane;
        const unsigned j = (unsigned)(k < jend ? k : jend - 1), c = f.count, t = j / c;
        tb = t * rows.Bn;
        return rows.order[f.start + (j - t * c)];
    };
    int tb, column;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        column = find_row(f.j0 + i * 64, tb);
        if (wave == 3) at[i][lane] = tb + column;
    }
    __syncthreads();
    int slot = 0;
    // a row's columns side by side over the lanes: rows of an odd width straddle few lines
    auto load = [&](F (&x)[PV], long j0, int slot, int first) {
#pragma unroll
        for (int i = 0; i < PV; ++i) {
            const int n = i * (256 / PW) + tid / PW, c = first + tid % PW * 8;
            x[i] = eight_once(P, at[slot][n] * ps + c, plimit);
        }
    };
    auto load_q = [&](long j0, int slot) {
#pragma unroll
        for (int i = 0; i < QV; ++i) {
            const int u = i * 256 + tid, n = u / (RT * 2);
            if (n >= 64) continue;
            const T* row = Q + at[slot][n] * LV;
#pragma unroll
            for (int j = 0; j < NQ; ++j) q[i][j] = *(const F*)(row + j * R16 + u % (RT * 2) * 8);
            if (SCALED) shifts[i] = row_shift(row, R16);
        }
        if (SCALED) shift_of_lane = row_shift(Q + at[slot][lane] * LV, R16);
    };
    // u of a step goes out in the next one, before its loads; rows behind the last, and the first
    // time all, to a row behind the shares that nobody reads.
    f32x4 u[RT];
    long to[4];
#pragma unroll
    for (int t = 0; t < RT; ++t) u[t] = f32x4{0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 4; ++i) to[i] = (long)shares * N;
    auto store_u = [&]() {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float* v = partv + to[i] * (RT * 16) + (lane & 15);
#pragma unroll
            for (int t = 0; t < RT; ++t) {
                v[t * 16] = u[t][i];
                u[t][i] = 0.f;
            }
        }
    };
    load_q(f.j0, 0);
    load(x[0], f.j0, 0, p0);
    __builtin_amdgcn_sched_barrier(0);
    if (D > 1) load(x[D - 1], f.j0, 0, p0 + PC);
    for (long j0 = f.j0; j0 < jend; j0 += 64) {
        const int next = slot == 2 ? 0 : slot + 1, behind = next == 2 ? 0 : next + 1;
#pragma unroll
        for (int k = 0; k < C; ++k) {
            __syncthreads();
            // Columns behind the last and rows behind the tile's are zero.  A strip that ends early
            // masks its columns (trimming them held its workgroups, and with them the launch, up by
            // half); the last rows of the tile, and of the matrix, are trimmed.
            const bool tail = j0 + 64 > jend;
            const bool close = tail || __builtin_amdgcn_readfirstlane(at[slot][63]) * ps + p0 +
                                               (k + 1) * PC > plimit;
            const u32x4 mask = first_bits(NP - p0 - k * PC - tid % PW * 8);
#pragma unroll
            for (int i = 0; i < PV; ++i) {
                const int n = i * (256 / PW) + tid / PW, c = p0 + k * PC + tid % PW * 8;
                F v = x[k % D][i];
                if (close) v = trim(v, at[slot][n] * ps + c, plimit, j0 + n < jend ? NP - c : 0);
                else if (p0 + (k + 1) * PC > NP) v = keep(v, mask);
                *(F*)(pt + n * LP + tid % PW * 8) = v;
            }
            if (SCALED && k == 0) {
                const int e = wave_largest(shift_of_lane, -120);
                if (e > shift_q) {
                    const float f = ldexpf(1.f, shift_q - e);
#pragma unroll
                    for (int l = 0; l < C; ++l)
#pragma unroll
                        for (int c = 0; c < CW; ++c)
#pragma unroll
                            for (int t = 0; t < RW; ++t) acc[l][c][t] *= f;
                    shift_q = e;
                }
            }
            if (k == 0)
#pragma unroll
                for (int i = 0; i < QV; ++i) {
                    const int u = i * 256 + tid, n = u / (RT * 2);
                    if (n >= 64) continue;
#pragma unroll
                    for (int j = 0; j < NQ; ++j) {
                        F v = j0 + n < jend ? q[i][j] : F{};
                        if (SCALED) v = shifted(v, shifts[i] - shift_q);
                        *(F*)(qt[j] + n * LQ + u % (RT * 2) * 8) = v;
                    }
                }
            __syncthreads();
            if (k == 0) {
                if (DV) store_u();
                column = find_row(j0 + 128, tb);
                load_q(j0 + 64, next);
            }
            if (k + D < C) load(x[k % D], j0, slot, p0 + (k + D) * PC);
            else load(x[k % D], j0 + 64, next, p0 + (k + D - C) * PC);
            if (DV) {           // a wave takes 16 of the rows
#pragma unroll
                for (int s = 0; s < S; ++s) {
                    const F a = *(const F*)(pt + (wave * 16 + (lane & 15)) * LP + s * 32 + g * 8);
#pragma unroll
                    for (int t = 0; t < RT; ++t)
                        u[t] = mfma(a, *(const F*)(wt + (t * 16 + (lane & 15)) * LW + k * PC +
                                                   s * 32 + g * 8), u[t]);
                }
            }
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                F b[NQ][RW];
#pragma unroll
                for (int i = 0; i < NQ; ++i)
#pragma unroll
                    for (int t = 0; t < RW; ++t)
                        b[i][t] = column_frag(qt[i], LQ, s * 32, (rt0 + t) * 16 + own_columns());
#pragma unroll
                for (int c = 0; c < CW; ++c) {
                    const F a = column_frag(pt, LP, s * 32, (ct0 + c) * 16 + own_columns());
#pragma unroll
                    for (int i = 0; i < NQ; ++i)
#pragma unroll
                        for (int t = 0; t < RW; ++t)
                            acc[k][c][t] = mfma(a, b[i][t], acc[k][c][t]);
                }
            }
        }
        if (DV) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int n = wave * 16 + g * 4 + i;
                to[i] = j0 + n < jend ? (long)share * N + at[slot][n] : (long)shares * N;
            }
        }
        if (wave == 3) at[behind][lane] = tb + column;
        slot = next;
    }
    if (DV) store_u();
    if (SCALED)
#pragma unroll
        for (int t = 0; t < RW; ++t)
#pragma unroll
            for (int k = 0; k < C; ++k)
#pragma unroll
                for (int c = 0; c < CW; ++c) acc[k][c][t] *= two_to(shift_q);
    if (whole) {                // the adapter's only tile: its gradient, rounded here
        T* o = whole + (long)f.adapter * NP * R;
#pragma unroll
        for (int k = 0; k < C; ++k)
#pragma unroll
            for (int c = 0; c < CW; ++c)
#pragma unroll
                for (int t = 0; t < RW; ++t) {
                    typedef T out4 __attribute__((ext_vector_type(4), aligned(2)));
                    const int p = p0 + k * PC + (ct0 + c) * 16 + g * 4;
                    const int r = (rt0 + t) * 16 + (lane & 15);
                    const f32x4 v = acc[k][c][t];
                    if (r >= R) continue;
                    if (!rcont && p + 4 <= NP) {
                        *(out4*)(o + (long)r * NP + p) = out4{(T)v[0], (T)v[1], (T)v[2], (T)v[3]};
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (p + i < NP)
                                o[rcont ? (long)(p + i) * R + r : (long)r * NP + p + i] = (T)v[i];
                    }
                }
        return;
    }
    const int LO = shares * C * PC;
#pragma unroll
    for (int k = 0; k < C; ++k)
#pragma unroll
        for (int c = 0; c < CW; ++c)
#pragma unroll
            for (int t = 0; t < RW; ++t)
                *(f32x4*)(part + ((long)tile * R16 + (rt0 + t) * 16 + (lane & 15)) * LO + p0 +
                          k * PC + (ct0 + c) * 16 + g * 4) = acc[k][c][t];
}

// The weights' gradient: an adapter's tiles in a fixed order, rounded once.  An adapter without
// rows gets zeros.  out is (L, R, NP) or, RCONT, (L, NP, R).  A thread takes four columns of one
// r; GR groups of threads share the tiles where there are many.
template <typename T, bool RCONT, int GR>
__global__ __launch_bounds__(256) void k_outer_sum(const float* __restrict__ part, int R16, int LP,
                                                   Rows rows, int shift, T* __restrict__ out,
                                                   int NP, int R, int blocks) {
    const int l = blockIdx.x / blocks, lane = threadIdx.x & 63;
    int first = 0, tiles = 0, base = 0;
    for (int s0 = 0; s0 < rows.S; s0 += 64) {
        const int s = s0 + lane;
        const int4 g = s < rows.S ? rows.segs[s] : make_int4(-1, 0, 0, 0);
        const int t = (int)((rows.T * g.z + (1l << shift) - 1) >> shift);
        const int sum = running_sum(t);
        const unsigned long long hit = __ballot(g.x == l && t > 0);
        if (hit) {
            const int k = __ffsll(hit) - 1;
            first = base + __builtin_amdgcn_readlane(sum - t, k);
            tiles = __builtin_amdgcn_readlane(t, k);
            break;
        }
        base += __builtin_amdgcn_readlane(sum, 63);
    }
    constexpr int TH = 256 / GR;
    __shared__ f32x4 sums[GR > 1 ? 256 : 1];
    const int b = blockIdx.x % blocks, cols = (NP + TH * 4 - 1) / (TH * 4);
    const int r = b / cols, group = threadIdx.x / TH;
    const int p = (b % cols * TH + threadIdx.x % TH) * 4;
    f32x4 s = f32x4{0, 0, 0, 0};
    const float* q = part + (long)r * LP + p;       // LP >= NP is a multiple of four
    if (p < NP)
#pragma unroll 4
        for (int t = first + group; t < first + tiles; t += GR)
            s += *(const f32x4*)(q + (long)t * R16 * LP);
    if (GR > 1) {
        sums[threadIdx.x] = s;
        __syncthreads();
        if (group) return;
#pragma unroll
        for (int k = 1; k < GR; ++k) s += sums[k * TH + threadIdx.x];
    }
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
void shrink(const void* X, long xs, long xlimit, const void* W, long wlimit, int K, int R,
            const Rows& rows, int tiles, const Scale& scale, void* V, float* part, long N,
            int splits, int kper, hipStream_t st) {
#define GO(RT)                                                                                   \
    k_shrink<T, RT, KCONT><<<(unsigned)(tiles * splits), 256, 0, st>>>(                          \
        (const T*)X, xs, xlimit, (const T*)W, wlimit, K, R, rows, scale, (T*)V, part, N,         \
        splits, kper)
    const int R16 = r16_of(R);
    if (R16 == 16) GO(1);
    else if (R16 == 32) GO(2);
    else if (R16 == 64) GO(4);
    else GO(8);
#undef GO
}

template <typename T, bool RCONT>
void expand(const void* base, long bs, long blimit, void* out, long os, const void* V,
            const void* W, long wlimit, int M, int R, const Rows& rows, int tiles, int shift,
            hipStream_t st) {
    const int strips = (M + 255) / 256, R16 = r16_of(R);
#define GO(RK)                                                                                   \
    k_expand<T, RK, RCONT><<<(unsigned)tiles * strips, 256, 0, st>>>(                            \
        (const T*)base, bs, blimit, (T*)out, os, (const T*)V, R16, (const T*)W, wlimit, M, R,    \
        rows, strips, shift)
    if (R16 <= 32) GO(1);
    else if (R16 == 64) GO(2);
    else GO(4);
#undef GO
}

// Columns that a workgroup of outer owns: 256, or 128 where a rank of 128 fills the registers.
// With u 1024 or 512, as many as the accumulators leave room for (65536 rows of 4096, rank 16: u's
// shares 9 us to sum, 17 at 256 columns), but 256 where that would leave CUs without work (1073
// rows of 2049: 9 us, 20 at 1024).
int outer_columns(int R, int with_u, long row_tiles, int NP) {
    if (R > 64) return 128;
    const int wide = R <= 16 ? 1024 : 512;
    return with_u && row_tiles * ((NP + wide - 1) / wide) >= 512 ? wide : 256;
}

// `whole`: every adapter's rows are one tile, and out holds zeros for those without rows.
template <typename T, bool RCONT>
void outer(const void* P, long ps, long plimit, int NP, const void* Q, float* part,
           const void* W, long wlimit, float* partv, long N, const Rows& rows, int tiles,
           int shift, int columns, int whole, void* out, int R, int L, hipStream_t st) {
    const int PC = columns, strips = (NP + PC - 1) / PC, R16 = r16_of(R);
#define GO(RT, CT, NS)                                                                           \
    k_outer<T, RT, CT, NS><<<(unsigned)tiles * strips, 256, 0, st>>>(                            \
        (const T*)P, ps, plimit, NP, (const T*)Q, part, (const T*)W, wlimit, R, partv, N,        \
        whole ? (T*)out : nullptr, RCONT, rows, strips, shift)
    if (tiles == 0) {           // no row has an adapter: the sum below writes zeros
    } else if (R16 == 16) {
        if (!W) GO(1, 4, 0);
        else if (PC > 256) GO(1, 4, 4);
        else GO(1, 4, 1);
    } else if (R16 == 32) {
        if (!W) GO(2, 4, 0);
        else if (PC > 256) GO(2, 4, 2);
        else GO(2, 4, 1);
    } else if (R16 == 64) GO(4, 4, 0);
    else GO(8, 2, 0);
#undef GO
    if (whole) return;
    const long many = (NP + 127) / 128 * (long)R;
    if (tiles > 16 * L && L * many * 256 < (1l << 32)) {    // many tiles an adapter
        const int blocks = (int)many;
        k_outer_sum<T, RCONT, 8><<<(unsigned)L * blocks, 256, 0, st>>>(
            part, R16, strips * PC, rows, shift, (T*)out, NP, R, blocks);
    } else {
        const int blocks = (NP + 1023) / 1024 * R;
        k_outer_sum<T, RCONT, 1><<<(unsigned)L * blocks, 256, 0, st>>>(
            part, R16, strips * PC, rows, shift, (T*)out, NP, R, blocks);
    }
}

}  // namespace

extern "C" {

// Numbers of a row of v's and u's shares, and 16-bit words of a row of v or u.
int lowrank_width(int R) { return r16_of(R); }
int lowrank_row(int type, int R) { return row_length(type == LM_F16, r16_of(R)); }

// Workgroups that share a row tile's contraction: about two a CU, no share below a step.  Up to
// `alone` steps stay with one: where the sum is a launch of its own, four do (8192 rows of 1024,
// rank 32: 10.4 us, 8.2 + 5.2 in four shares; eight take 11.9, and 6.4 + 3.8 in eight).
int lowrank_splits(const long* counts, int S, long T, int K, int alone) {
    const int tiles = tiles_of(counts, S, T, S_TM), steps = (K + S_KC - 1) / S_KC;
    const int want = tiles > 0 ? (512 + tiles - 1) / tiles : 1;
    return steps <= alone ? 1 : want > steps ? steps : want;
}

// With `part` (splits, N, R16) the shares are left there unscaled and V is not written.
void launch_shrink(int type, int kcont, const void* X, long xs, long xlimit, const void* W,
                   long wlimit, int K, int R, const int* order, const int* segs,
                   const int* adapter, const long* counts, int S, int Bn, long T,
                   const float* scale, float scale_all, void* V, float* part, int splits,
                   hipStream_t st) {
    const Rows rows{order, (const int4*)segs, adapter, S, Bn, T};
    const Scale sc{scale, scale_all};
    const int tiles = tiles_of(counts, S, T, S_TM);
    if (tiles == 0) return;
    const int kper = ((K + splits - 1) / splits + S_KC - 1) / S_KC * S_KC;
    const long N = T * Bn;
#define GO(T, KCONT)                                                                             \
    shrink<T, KCONT>(X, xs, xlimit, W, wlimit, K, R, rows, tiles, sc, V, part, N, splits, kper, st)
    if (type == LM_BF16) {
        if (kcont) GO(bf16_t, true);
        else GO(bf16_t, false);
    } else {
        if (kcont) GO(f16_t, true);
        else GO(f16_t, false);
    }
#undef GO
}

void launch_shrink_sum(int type, int R, const int* order, const int* segs, const int* adapter,
                       int S, int Bn, long T, const float* scale, float scale_all, void* V,
                       const float* part, int splits, hipStream_t st) {
    const Rows rows{order, (const int4*)segs, adapter, S, Bn, T};
    const Scale sc{scale, scale_all};
    const int R16 = r16_of(R);
    const long N = T * Bn, threads = N * (R16 / 4);
#define GO(T, GR)                                                                                \
    k_shrink_sum<T, GR><<<(unsigned)((threads + 256 / GR - 1) / (256 / GR)), 256, 0, st>>>(      \
        part, N, R, R16, splits, rows, sc, (T*)V)
    if (type == LM_BF16) {
        if (splits < 32) GO(bf16_t, 1);
        else GO(bf16_t, 8);
    } else {
        if (splits < 32) GO(f16_t, 1);
        else GO(f16_t, 8);
    }
#undef GO
}

void launch_expand(int type, int rcont, const void* base, long bs, long blimit, void* out,
                   long os, const void* V, const void* W, long wlimit, int M, int R,
                   const int* order, const int* segs, const int* adapter, const long* counts,
                   int S, int Bn, long T, hipStream_t st) {
    const Rows rows{order, (const int4*)segs, adapter, S, Bn, T};
    // rows a workgroup: as many as leave four workgroups a CU, 256 at most, 32 at least
    const long strips = (M + 255) / 256;
    int shift = 8;
    while (shift > 5 && tiles_of(counts, S, T, shift) * strips < 1024) --shift;
    const int tiles = tiles_of(counts, S, T, shift);
    if (tiles == 0) return;
#define GO(T, RCONT)                                                                             \
    expand<T, RCONT>(base, bs, blimit, out, os, V, W, wlimit, M, R, rows, tiles, shift, st)
    if (type == LM_BF16) {
        if (rcont) GO(bf16_t, true);
        else GO(bf16_t, false);
    } else {
        if (rcont) GO(f16_t, true);
        else GO(f16_t, false);
    }
#undef GO
}

// A decode step: W passes twice on the average at most, four rows a pass.  16 adapters at the
// head (50000 columns, rank 16): 4 rows each 22 us, 29 through shrink, its sum and expand; 8 rows
// 33 and 31, 16 rows 49 and 33.  A row alone takes as long either way, with a launch less here.
int lowrank_few(const long* counts, int S, long T) {
    return tiles_of(counts, S, T, FEW) <= 2 * S;
}

void launch_expand_few(int type, const void* base, long bs, void* out, long os, const float* part,
                       const void* W, int M, int R, const int* order, const int* segs,
                       const int* adapter, const long* counts, int S, int Bn, long T,
                       const float* scale, float scale_all, int splits, hipStream_t st) {
    const Rows rows{order, (const int4*)segs, adapter, S, Bn, T};
    const Scale sc{scale, scale_all};
    const int tiles = tiles_of(counts, S, T, FEW), strips = (M + 511) / 512, R16 = r16_of(R);
    const long N = T * Bn;
    if (type == LM_BF16)
        k_expand_few<bf16_t><<<(unsigned)tiles * strips, 64, 0, st>>>(
            (const bf16_t*)base, bs, (bf16_t*)out, os, part, N, R16, splits, sc,
            (const bf16_t*)W, M, R, rows, strips);
    else
        k_expand_few<f16_t><<<(unsigned)tiles * strips, 64, 0, st>>>(
            (const f16_t*)base, bs, (f16_t*)out, os, part, N, R16, splits, sc, (const f16_t*)W, M,
            R, rows, strips);
}

int lowrank_outer_columns(const long* counts, int S, long T, int NP, int R, int with_u) {
    return outer_columns(R, with_u, tiles_of(counts, S, T, 6), NP);
}
// Whether every group of rows is one tile: its gradient is written without a sum of partial ones.
int lowrank_outer_whole(const long* counts, int S, long T, int shift) {
    return tiles_of(counts, S, T, shift) == S;
}
// log2 of the rows that one partial gradient sums, 64 (a step) to 4096: the least time by what
// was measured, in us.  A workgroup takes 6 to come and go, and a step of 64 rows 1.2, or what it
// reads at 25 GB/s by itself, or at its share of 5 TB/s; rounds of the workgroups that fit the
// chip count whole; the partial gradients are written and read again by a launch of 4, which one
// tile an adapter does without.  65536 rows of 4096 columns, rank 16: 1024 rows; 8192 of 50000,
// rank 32, in four groups, and 1073 of 2049 in seven: one tile each.
int lowrank_outer_shift(const long* counts, int S, long T, int strips, int columns, int R) {
    const double fit = columns > 256 ? 512 : 1024, R16 = r16_of(R);
    int best = 6;
    double least = 1e300;
    long most = 0;              // rows of an adapter
    for (int s = 0; s < S; ++s) most = std::max(most, T * counts[s]);
    for (int shift = 12; shift >= 6; --shift) {
        const double blocks = (double)tiles_of(counts, S, T, shift) * strips;
        const double at_once = blocks < fit ? blocks : fit;
        const double alone = columns * 128 / 2.5e4 > 1.2 ? columns * 128 / 2.5e4 : 1.2;
        const double steps = (double)((std::min(1l << shift, most) + 63) >> 6);
        const double step = columns * 128 * at_once / 5e6;
        double us = (double)(long)((blocks + fit - 1) / fit) *
                    (6 + steps * (step > alone ? step : alone));
        if (!lowrank_outer_whole(counts, S, T, shift)) us += 4 + blocks * columns * R16 * 8 / 5e6;
        if (us < least) {
            least = us;
            best = shift;
        }
    }
    return best;
}
int lowrank_outer_tiles(const long* counts, int S, long T, int shift) {
    return tiles_of(counts, S, T, shift);
}
// Whether the backward pass reads dy once for u and dB (k_outer's DV): not where the shares of u
// would be as many bytes as dy.
int lowrank_one_reading(int R) { return R <= 32; }

void launch_outer(int type, int rcont, const void* P, long ps, long plimit, int NP,
                  const void* Q, float* part, const void* W, long wlimit, float* partv,
                  const int* order, const int* segs, const int* adapter, const long* counts, int S,
                  int Bn, long T, int shift, int columns, int whole, void* out, int R, int L,
                  hipStream_t st) {
    const Rows rows{order, (const int4*)segs, adapter, S, Bn, T};
    const int tiles = tiles_of(counts, S, T, shift);
    const long N = T * Bn;
#define GO(T, RCONT)                                                                             \
    outer<T, RCONT>(P, ps, plimit, NP, Q, part, W, wlimit, partv, N, rows, tiles, shift, columns,\
                    whole, out, R, L, st)
    if (type == LM_BF16) {
        if (rcont) GO(bf16_t, true);
        else GO(bf16_t, false);
    } else {
        if (rcont) GO(f16_t, true);
        else GO(f16_t, false);
    }
#undef GO
}

}  // extern "C"
