// The gated feed-forward product and its gradient:
//
//   [g | v] = x W^T (W: the gate's F rows, then the values'),  h = act(g) v
//   dv = dh act(g), dg = dh v act'(g);  dx = [dg | dv] W;  dW = [dg | dv]^T x
//
// act(g) = g sigmoid(u), u = g (silu) or 2 c (g + k g^3), c = sqrt(2 / pi), k = 0.044715 (gelu's tanh form).
//
// Forward: the product runs in the tiles of ce_gemm.h, whose rows are 16 of the gate and
// the same 16 of the values in turn (PAIR): a lane's accumulators hold g and v of the same place, and
// the epilogue stores h alone.  4096 x 2560 x 6912 bf16 take 228 us (1.27 PFLOP/s; the card's power bounds it: the matrix units
// are busy 55 to 63 % of the cycles at 1.85 GHz).  For a gradient the epilogue stores act(g) and v act'(g) too, by which
// dh is multiplied: to compute them again would take a third of the gradient's operations, to keep them costs their bytes
// twice.  8192 tokens so take 521 us, 1.11 PFLOP/s: all tiles end, and store their 453 MB, at the same times.
// Up to 64 tokens whose rows a lane can load in 16-byte pieces run k_glu_few, bound by reading W once.
//
// Backward: k_glu_dz makes dz = [dg | dv] = [dh v act'(g) | dh act(g)] (bf16, or three planes of it for float32), then two
// products read it: dx with K over W's rows, dW with K over the tokens (8192 x 2560 x 6912: 494 and 467 us, 1.17 and 1.24
// PFLOP/s).  Tiles that would leave CUs idle in the last round are cut along K into float32 parts (deal), which k_glu_join
// adds up (13 and 11 us).  float32: 1024 x 768 x 2048, 43 us the forward, 48 dx, 43 dW: six bf16 products, 0.8 to 0.9 PFLOP/s;
// a CU has one tile then, and its first loads and its epilogue have nothing beside them.
//
// Operands that direct loads cannot take in place (float32, widths that 64 does not divide, unaligned
// rows) are packed first: rows padded with zeros, the gate's and the values' to whole 64s.
#include "ce_gemm.h"

namespace {

using namespace m2ce;

constexpr float LOG2E = 1.4426950408889634f;

// act(g) and, for SLOPE, its derivative.  (Past +-100, +-20 of gelu, the sigmoid is 0 or 1 and its slope 0: g is bounded
// where that multiplies it, so that no 0 inf comes of it.)
template <bool GELU, bool SLOPE> M2_DEV float act(float g, float& slope) {
    constexpr float C2 = 1.5957691216057308f, K = 0.044715f, LIM = GELU ? 20.f : 100.f;
    const float u = GELU ? C2 * g * fmaf(K * g, g, 1.f) : g;
    const float s = __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(u * -LOG2E));
    if constexpr (SLOPE) {
        const float b = __builtin_amdgcn_fmed3f(g, -LIM, LIM), bs = b * s;
        slope = fmaf(GELU ? bs * (C2 * fmaf(3.f * K * b, b, 1.f)) : bs, 1.f - s, s);
    }
    return g * s;
}

// four consecutive values of a row of dim elements
template <typename T> M2_DEV void store_quad(T* row, int m, int64_t dim, const f32x4& v) {
    if (m + 4 <= dim) {
        if constexpr (sizeof(T) == 2) {
            typedef uint32_t any __attribute__((ext_vector_type(2), aligned(2)));
            *reinterpret_cast<any*>(row + m) = any{pk_bf16(v[0], v[1]), pk_bf16(v[2], v[3])};
        } else {
            store16(row + m, __builtin_bit_cast(u32x4, v));
        }
    } else {
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (m + r < dim) row[m + r] = from_f32<T>(v[r]);
    }
}

// The factors of dh, v act'(g) and act(g), as the lanes of the forward's product hold them: an entry is four places of
// the hidden size of one token; entries of a wavefront's 64 lanes lie beside each other, so that they are written and read in
// whole lines (in rows instead: 28 registers of the large tile spilled, 588 us for 521).  float32 as they are; of bf16
// operands the upper 24 bits (cut off: off by 2^-15 at most, dz's own rounding is 2^-8), the upper 16 in one array, 8
// more in another.  With 16 bits dx and dW of 8192 x 2560 x 6912 were 2.9e-3 off instead of 2.3e-3, of which 1.7e-3 is
// their own rounding, and a training step took 1545 us instead of 1562.
template <typename T> struct Factors;
template <> struct Factors<float> {
    f32x4* p;
    static size_t bytes(int64_t entries) { return 32 * (size_t)entries; }
    __host__ __device__ Factors(const void* at, int64_t) : p(static_cast<f32x4*>(const_cast<void*>(at))) {}
    // (entry e + lane: e is the wavefront's)
    M2_DEV void put(int64_t e, uint32_t lane, const f32x4& by, const f32x4& at) const {
        f32x4* d = p + 2 * e;
        d[2 * lane] = by;
        d[2 * lane + 1] = at;
    }
    M2_DEV void get(int64_t e, f32x4& by, f32x4& at) const {
        by = p[2 * e];
        at = p[2 * e + 1];
    }
};
template <> struct Factors<bf16> {
    typedef uint32_t u2 __attribute__((ext_vector_type(2)));
    u32x4* hi;
    u2* lo;
    static size_t bytes(int64_t entries) { return 24 * (size_t)entries; }
    __host__ __device__ Factors(const void* at, int64_t entries)
        : hi(static_cast<u32x4*>(const_cast<void*>(at))), lo(reinterpret_cast<u2*>(hi + entries)) {}
    // the upper halves of two floats; the next bytes of four; a float of its half `k` of h and its byte `i` of l
    static M2_DEV uint32_t high(float a, float b) { return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302); }
    static M2_DEV uint32_t next(const f32x4& v) {
        return __builtin_amdgcn_perm(__float_as_uint(v[1]), __float_as_uint(v[0]), 0x0c0c0501) |
               __builtin_amdgcn_perm(__float_as_uint(v[3]), __float_as_uint(v[2]), 0x05010c0c);
    }
    static M2_DEV float both(uint32_t h, int k, uint32_t l, int i) {
        const uint32_t sel = 0x0000000c | (uint32_t)i << 8 | (uint32_t)(4 + 2 * k) << 16 | (uint32_t)(5 + 2 * k) << 24;
        return __uint_as_float(__builtin_amdgcn_perm(h, l, sel));
    }
    M2_DEV void put(int64_t e, uint32_t lane, const f32x4& by, const f32x4& at) const {
        (hi + e)[lane] = u32x4{high(by[0], by[1]), high(by[2], by[3]), high(at[0], at[1]), high(at[2], at[3])};
        (lo + e)[lane] = u2{next(by), next(at)};
    }
    M2_DEV void get(int64_t e, f32x4& by, f32x4& at) const {
        const u32x4 h = hi[e];
        const u2 l = lo[e];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            by[i] = both(h[i >> 1], i & 1, l[0], i);
            at[i] = both(h[2 + (i >> 1)], i & 1, l[1], i);
        }
    }
};
// the first entry of a wavefront's (wm, wn) columns j and pairs of fragments p of the tile at (m0, n0); tn: tiles along n
template <class S> M2_DEV int64_t entry(int m0, int n0, int tn, int wm, int wn, int j, int p) {
    const int64_t tile = (int64_t)(m0 / S::BM) * tn + n0 / S::BN;
    return (((tile * S::NW + wm * S::WN + wn) * S::FN + j) * (S::FM / 2) + p) * 64;
}
template <class S> int64_t entries(int64_t m, int64_t n) { return (int64_t)tiles(m, S::BM) * tiles(n, S::BN) * (S::BM * S::BN / 8); }

// ---------------------------------------------------------------------------
// forward
// ---------------------------------------------------------------------------
// m: pairs of the hidden size, n: token -> h, and for a gradient the factors
template <typename T, bool SAVE> struct EpiGlu {
    static constexpr bool SEG = false;
    T* h;
    Factors<T> z;
    int64_t hidden;
    int tn, gelu;

    template <class S>
    M2_DEV void run(f32x4 (&acc)[S::FM][S::FN], int m0, int n0, int wm, int wn, int lane, int count, int, int) const {
        if (gelu) with<S, true>(acc, m0, n0, wm, wn, lane, count);
        else with<S, false>(acc, m0, n0, wm, wn, lane, count);
    }
    template <class S, bool GELU>
    M2_DEV void with(f32x4 (&acc)[S::FM][S::FN], int m0, int n0, int wm, int wn, int lane, int count) const {
        static_assert(S::FM % 2 == 0, "");
        constexpr bool WIDE = S::FM % 4 == 0;
        const int f0 = m0 / 2 + wm * S::FM * 8;
#pragma unroll
        for (int j = 0; j < S::FN; ++j) {
            const int n = n0 + (wn * S::FN + j) * 16 + (lane & 15);
            if (n >= count) continue;
            T* to = h + (int64_t)n * hidden;
#pragma unroll
            for (int i = 0; i < S::FM; i += WIDE ? 4 : 2) {
                const int f = f0 + 8 * i;
                constexpr int E = WIDE ? 2 : 1;
                f32x4 o[E];
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    f32x4 by, at;
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float v = acc[i + 2 * e + 1][j][r];
                        float slope;
                        at[r] = act<GELU, SAVE>(acc[i + 2 * e][j][r], slope);
                        o[e][r] = at[r] * v;
                        if constexpr (SAVE) by[r] = slope * v;
                    }
                    if constexpr (SAVE) z.put(entry<S>(m0, n0, tn, wm, wn, j, i / 2 + e), lane, by, at);
                }
                if constexpr (WIDE) store_row(to, f, hidden, lane, o[0], o[1]);
                else store_quad(to, f + 4 * (lane >> 4), hidden, o[0]);
            }
        }
    }
};

// 8 consecutive k of a row as matrix operands: bf16, or a float32's three planes
template <typename T> struct Few;
template <> struct Few<bf16> {
    bf16x8 v;
    M2_DEV void load(const bf16* p) { v = *reinterpret_cast<const bf16x8*>(p); }
    M2_DEV void keep(bool in) {
        const bf16x8 zero = {};
        if (!in) v = zero;
    }
    static M2_DEV f32x4 mma(const Few& a, const Few& b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.v, b.v, c, 0, 0, 0);
    }
};
template <> struct Few<float> {
    u32x4 lo, hi;
    M2_DEV void load(const float* p) {
        lo = reinterpret_cast<const u32x4*>(p)[0];
        hi = reinterpret_cast<const u32x4*>(p)[1];
    }
    M2_DEV void keep(bool in) {
        const u32x4 zero = {};
        if (!in) lo = hi = zero;
    }
    M2_DEV void planes(bf16x8 (&p)[3]) const {
        float h[8], m[8], l[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) split3(__uint_as_float(i < 4 ? lo[i & 3] : hi[i & 3]), h[i], m[i], l[i]);
        auto pack = [](const float(&f)[8]) {
            return as_bf16x8(pk_bf16(f[0], f[1]), pk_bf16(f[2], f[3]), pk_bf16(f[4], f[5]), pk_bf16(f[6], f[7]));
        };
        p[0] = pack(h); p[1] = pack(m); p[2] = pack(l);
    }
    static M2_DEV f32x4 mma(const Few& a, const Few& b, f32x4 c) {
        bf16x8 x[3], y[3];
        a.planes(x);
        b.planes(y);
        constexpr int PI[6] = {0, 2, 1, 0, 1, 0}, PJ[6] = {2, 0, 1, 1, 0, 0};      // the small products first
#pragma unroll
        for (int t = 0; t < 6; ++t) c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x[PI[t]], y[PJ[t]], c, 0, 0, 0);
        return c;
    }
};

struct FewArgs {
    const void *x, *w;
    void *h, *z;
    int64_t ldx, ldw, entries;
    int n, dim, hidden, gelu;
};
// Up to 16 MT tokens: a workgroup takes 8 FT of the hidden size, its NW wavefronts split K and meet in LDS.  Bound by W's
// bytes: 1 token x 2560 x 6912 bf16 18.9 us, 16 tokens 23.8 (71 MB, 3.7 and 3.0 TB/s; 13.7 and 15.4 where a part of the weights
// is in the last-level cache), float32 33, 35 and 64 tokens 61 (142 MB, 4.3, 4.0 and 2.3 TB/s: every pair of fragments splits
// both of them in three anew).
// The 16 rows of a matrix operand are 8 of the gate and the 8 of the values, so that lanes
// l and l + 32 hold g and v of the same place; every weight is read once, x comes from the cache.
// U steps of 32 of K are in flight: a step's operands are loaded again, U steps on, right behind its products.
// The factors lie as the shape S's lanes would hold them, whose tiles are of 64 tokens.
template <typename T, class S, int MT, int FT, int NW, int U>
__global__ void __launch_bounds__(NW * 64) k_glu_few(FewArgs a) {
    __shared__ f32x4 red[NW][FT * MT][64];
    const int lane = threadIdx.x & 63, w = wave_id();
    const int f0 = blockIdx.x * 8 * FT, row = lane & 15, kq = (lane >> 4) * 8;
    const T *wr[FT], *xr[MT];
#pragma unroll
    for (int i = 0; i < FT; ++i)
        wr[i] = static_cast<const T*>(a.w) +
                ((int64_t)(row >> 3) * a.hidden + min(f0 + 8 * i + (row & 7), a.hidden - 1)) * a.ldw;
#pragma unroll
    for (int t = 0; t < MT; ++t) xr[t] = static_cast<const T*>(a.x) + (int64_t)min(16 * t + row, a.n - 1) * a.ldx;
    const int steps = (a.dim + 31) / 32, per = (steps + NW - 1) / NW;
    const int s0 = w * per, s1 = min(steps, s0 + per);
    f32x4 acc[FT][MT];
#pragma unroll
    for (int i = 0; i < FT; ++i)
#pragma unroll
        for (int t = 0; t < MT; ++t) acc[i][t] = zero4();
    Few<T> fw[U][FT], fx[U][MT];
    auto load = [&](int q, int s) {
        const int k = min(s * 32 + kq, a.dim - 8);         // (past the end of a row: its last piece, not used)
#pragma unroll
        for (int i = 0; i < FT; ++i) fw[q][i].load(wr[i] + k);
#pragma unroll
        for (int t = 0; t < MT; ++t) fx[q][t].load(xr[t] + k);
    };
#pragma unroll
    for (int q = 0; q < U; ++q)
        if (s0 + q < s1) load(q, s0 + q);
    for (int s = s0; s < s1; s += U) {
#pragma unroll
        for (int q = 0; q < U; ++q) {
            if (s + q >= s1) break;
            if ((s + q) * 32 + 32 > a.dim) {               // a last step that is not whole
                const bool in = (s + q) * 32 + kq < a.dim;
#pragma unroll
                for (int i = 0; i < FT; ++i) fw[q][i].keep(in);
#pragma unroll
                for (int t = 0; t < MT; ++t) fx[q][t].keep(in);
            }
#pragma unroll
            for (int i = 0; i < FT; ++i)
#pragma unroll
                for (int t = 0; t < MT; ++t) acc[i][t] = Few<T>::mma(fw[q][i], fx[q][t], acc[i][t]);
            if (s + q + U < s1) load(q, s + q + U);
        }
    }
#pragma unroll
    for (int i = 0; i < FT; ++i)
#pragma unroll
        for (int t = 0; t < MT; ++t) red[w][i * MT + t][lane] = acc[i][t];
    __syncthreads();
    for (int p = w; p < FT * MT; p += NW) {
        f32x4 v = red[0][p][lane];
#pragma unroll
        for (int u = 1; u < NW; ++u) v += red[u][p][lane];
        f32x4 o, by, at;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const float other = __shfl_xor(v[r], 32);
            float slope;
            at[r] = a.gelu ? act<true, true>(v[r], slope) : act<false, true>(v[r], slope);
            o[r] = at[r] * other;
            by[r] = slope * other;
        }
        const int n = 16 * (p % MT) + (lane & 15), f = f0 + 8 * (p / MT) + 4 * ((lane >> 4) & 1);
        if (lane >= 32 || n >= a.n) continue;
        store_quad(static_cast<T*>(a.h) + (int64_t)n * a.hidden, f, a.hidden, o);
        static_assert(S::BN == 64 && S::FM == 2, "");
        if (a.z && f < a.hidden) {
            const int m0 = f / (S::BM / 2) * S::BM, wm = f % (S::BM / 2) / 16, t = n / 16;
            const int64_t e = entry<S>(m0, 0, 1, wm, t / S::FN, t % S::FN, 0);
            Factors<T>(a.z, a.entries).put(e, (n & 15) + 16 * (f / 4 & 3), by, at);
        }
    }
}

// ---------------------------------------------------------------------------
// packing, dz
// ---------------------------------------------------------------------------
// rows of src as bf16 (planes) with rows of dp elements, zeros behind dim and in the rows that src lacks: row j
// is src's j, or with `half` the j-th of the first `valid` rows, and half + j the j-th of the other `valid`
struct PackArgs {
    const void* src;
    bf16* dst;
    int64_t rows, dim, ld, dp, plane, half, valid;
};
constexpr int64_t PACK_ROWS = 1 << 24;       // of a launch, a wavefront each (a launch counts its threads in 32 bits)
template <typename T> __global__ void __launch_bounds__(256) k_glu_pack(PackArgs a) {
    const int lane = threadIdx.x & 63;
    for (int64_t r = (int64_t)blockIdx.x * 4 + wave_id(); r < a.rows; r += PACK_ROWS) {
        const int second = a.half && r >= a.half;
        const int64_t j = second ? r - a.half : r;
        const bool in = j < a.valid;
        const T* src = static_cast<const T*>(a.src) + (in ? j + (second ? a.valid : 0) : 0) * a.ld;
        for (int64_t c = lane * 8; c < a.dp; c += 512) {
            float v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
            if (in) load8(src, c, a.dim, v);
            store8<sizeof(T) == 4>(a.dst + r * a.dp + c, a.plane, v);
        }
    }
}
template <typename T> void pack_rows(const PackArgs& a, hipStream_t s) {
    const int64_t rows = a.rows < PACK_ROWS ? a.rows : PACK_ROWS;
    hipLaunchKernelGGL(k_glu_pack<T>, dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, s, a);
}

struct DzArgs {
    const void *z, *dh;
    bf16* dz;                // [np][2 fp], zeros past n and past hidden
    int64_t n, np, hidden, fp, ldg, plane, entries;
    int tm, tn;              // of the forward's product
};
// dz from the factors as the forward's shape S left them: a wavefront for 16 tokens and 32 of the hidden size (16 where a
// wavefront of S has no more).  Bound by bytes: 8192 x 6912 bf16 142 us (679 MB, 4.8 TB/s).
template <typename T, class S> __global__ void __launch_bounds__(256) k_glu_dz(DzArgs a) {
    constexpr bool WIDE = S::FM % 4 == 0;
    constexpr int E = WIDE ? 2 : 1, PER = S::FM / 2 / E, WAVES = S::NW * S::FN * PER;
    const int lane = threadIdx.x & 63;
    int64_t q = (int64_t)blockIdx.x * 4 + wave_id();
    const int64_t tile = q / WAVES;
    if (tile >= (int64_t)a.tm * a.tn) return;
    const int in = (int)(q - tile * WAVES), p = in % PER * E, j = in / PER % S::FN, w = in / PER / S::FN;
    const int m0 = (int)(tile / a.tn) * S::BM, n0 = (int)(tile % a.tn) * S::BN, wm = w / S::WN, wn = w % S::WN;
    const int64_t n = n0 + (wn * S::FN + j) * 16 + (lane & 15);
    const int64_t f0 = m0 / 2 + wm * S::FM * 8 + p * 16;
    if (f0 >= a.fp) return;                  // (a row ends at a multiple of 64: of all lanes or of none)
    const Factors<T> z(a.z, a.entries);
    const bool on = n < a.n;
    f32x4 by[E], at[E], up[E];
    const T* dh = static_cast<const T*>(a.dh) + (on ? n : 0) * a.ldg;
    if constexpr (WIDE && sizeof(T) == 2) {
        // 8 consecutive values a lane, exchanged to the fragments' order
        uint32_t v[4];
        const int64_t f = f0 + pair_m(lane);
        if (f + 8 <= a.hidden) {
            const u32x4 r = load16(dh + f);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = r[i];
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint16_t* s = reinterpret_cast<const uint16_t*>(dh) + f + 2 * i;
                v[i] = (f + 2 * i < a.hidden ? s[0] : 0) | (uint32_t)(f + 2 * i + 1 < a.hidden ? s[1] : 0) << 16;
            }
        }
        pair_swap(v[0], v[2]);
        pair_swap(v[1], v[3]);
#pragma unroll
        for (int e = 0; e < 2; ++e) up[e] = f32x4{bf16_lo(v[2 * e]), bf16_hi(v[2 * e]), bf16_lo(v[2 * e + 1]), bf16_hi(v[2 * e + 1])};
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int64_t f = f0 + 16 * e + 4 * (lane >> 4) + r;
                up[e][r] = f < a.hidden ? to_f32(dh[f]) : 0.f;
            }
    }
#pragma unroll
    for (int e = 0; e < E; ++e) z.get(entry<S>(m0, n0, a.tn, wm, wn, j, p + e) + lane, by[e], at[e]);
    // (what the factors hold past the tokens and the hidden size is anything)
#pragma unroll
    for (int e = 0; e < E; ++e)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const bool in = on && f0 + 16 * e + 4 * (lane >> 4) + r < a.hidden;
            by[e][r] = in ? up[e][r] * by[e][r] : 0.f;
            at[e][r] = in ? up[e][r] * at[e][r] : 0.f;
        }
    if (n >= a.np) return;                   // (np is a multiple of 16: all lanes or none)
    auto put = [&](bf16* to, const f32x4 (&v)[E]) {
        constexpr int PLANES = sizeof(T) == 4 ? 3 : 1;
        float part[PLANES][E][4];
#pragma unroll
        for (int e = 0; e < E; ++e)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                if constexpr (PLANES == 3) split3(v[e][r], part[0][e][r], part[1][e][r], part[2][e][r]);
                else part[0][e][r] = v[e][r];
            }
#pragma unroll
        for (int k = 0; k < PLANES; ++k) {
            if constexpr (WIDE) store_pair(to + k * a.plane + pair_m(lane), part[k][0], part[k][1]);
            else store_quad(to + k * a.plane, 4 * (lane >> 4), 16, f32x4{part[k][0][0], part[k][0][1], part[k][0][2], part[k][0][3]});
        }
    };
    bf16* row = a.dz + n * 2 * a.fp + f0;
    put(row, by);
    put(row + a.fp, at);
}

// ---------------------------------------------------------------------------
// the gradients' products
// ---------------------------------------------------------------------------
// where the rows (n) of a product go: the n-th, or with `half` the first `valid` of either half
template <typename T> struct Out {
    T* p;
    int64_t dim;
    int half, valid;
    M2_DEV T* row(int n) const {
        const int second = half && n >= half, j = second ? n - half : n;
        return j < valid ? p + (int64_t)(second ? j + valid : j) * dim : nullptr;
    }
};
// m: columns, n: rows.  A whole tile is stored; the parts of one that deal() cut as the lanes hold them,
// [part][wavefront][i][j][lane] of 4 values.
template <typename T> struct EpiOut {
    static constexpr bool SEG = true;
    Out<T> out;
    float* part;
    int full;                // tiles that are whole

    template <class S>
    M2_DEV void run(f32x4 (&acc)[S::FM][S::FN], int m0, int n0, int wm, int wn, int lane, int, int seg, int) const {
        static_assert(S::FM % 2 == 0, "");
        if (seg >= full) {
            f32x4* d = reinterpret_cast<f32x4*>(part) +
                       ((int64_t)(seg - full) * S::NW + wm * S::WN + wn) * S::FM * S::FN * 64 + lane;
#pragma unroll
            for (int i = 0; i < S::FM; ++i)
#pragma unroll
                for (int j = 0; j < S::FN; ++j) d[(i * S::FN + j) * 64] = acc[i][j];
            return;
        }
        const int mw = m0 + wm * S::FM * 16, nw = n0 + wn * S::FN * 16;
#pragma unroll
        for (int j = 0; j < S::FN; ++j) {
            T* to = out.row(nw + 16 * j + (lane & 15));
            if (!to) continue;
#pragma unroll
            for (int i = 0; i < S::FM; i += 2) store_row(to, mw + 16 * i, out.dim, lane, acc[i][j], acc[i + 1][j]);
        }
    }
};
// the parts of the cut tiles, in their order: a wavefront for two fragments (32 columns) of 16 rows
struct JoinArgs {
    const float* part;
    int tm, tn, full, rest, s;
};
template <typename T, class S> __global__ void __launch_bounds__(256) k_glu_join(JoinArgs a, Out<T> out) {
    const int lane = threadIdx.x & 63;
    constexpr int PAIRS = S::FM / 2, PER = S::NW * PAIRS * S::FN;
    int q = blockIdx.x * 4 + wave_id();
    const int t = q / PER;
    q -= t * PER;
    if (t >= a.rest) return;
    const int j = q % S::FN, i = q / S::FN % PAIRS * 2, w = q / S::FN / PAIRS;
    // (the tile's place as in the product's kernel)
    const int tile = a.full + t;
    const int grp = tile / (8 * a.tn), gm = min(8, a.tm - grp * 8), in = tile - grp * 8 * a.tn;
    const int m0 = (grp * 8 + in % gm) * S::BM + (w / S::WN * S::FM + i) * 16;
    T* to = out.row(in / gm * S::BN + (w % S::WN * S::FN + j) * 16 + (lane & 15));
    constexpr int64_t TILE = (int64_t)S::NW * S::FM * S::FN * 64;
    const f32x4* p = reinterpret_cast<const f32x4*>(a.part) + t * TILE + (w * S::FM * S::FN + i * S::FN + j) * 64 + lane;
    f32x4 x = p[0], y = p[S::FN * 64];
#pragma unroll 8
    for (int k = 1; k < a.s; ++k) {
        p += a.rest * TILE;
        x += p[0];
        y += p[S::FN * 64];
    }
    if (to) store_row(to, m0, out.dim, lane, x, y);
}

// few tokens (k_ce_stream): one array of dx for each split of K, [splits][np][dp]
struct EpiSplit {
    static constexpr bool SEG = false;
    float* part;
    int64_t np, dp;

    template <class S>
    M2_DEV void run(f32x4 (&acc)[S::FM][S::FN], int m0, int n0, int wm, int wn, int lane, int count, int split,
                    int) const {
        const int mv = m0 + wm * S::FM * 16 + 4 * (lane >> 4);
#pragma unroll
        for (int j = 0; j < S::FN; ++j) {
            const int n = n0 + (wn * S::FN + j) * 16 + (lane & 15);
            if (n >= count) continue;
            float* d = part + ((int64_t)split * np + n) * dp;
#pragma unroll
            for (int i = 0; i < S::FM; ++i)
                if (mv + 16 * i < dp) *reinterpret_cast<f32x4*>(d + mv + 16 * i) = acc[i][j];
        }
    }
};
__global__ void __launch_bounds__(64) k_glu_sum(const float* part, bf16* dx, int64_t np, int64_t dp, int64_t dim,
                                                int splits) {
    const int64_t n = blockIdx.y, c = ((int64_t)blockIdx.x * 64 + threadIdx.x) * 4;
    if (c >= dim) return;
    f32x4 v = zero4();
    const float* p = part + n * dp + c;
#pragma unroll 8
    for (int s = 0; s < splits; ++s) v += *reinterpret_cast<const f32x4*>(p + s * np * dp);
    store_quad(dx + n * dim, (int)c, dim, v);
}

// ---------------------------------------------------------------------------
// plans
// ---------------------------------------------------------------------------
// Tiles of the forward's product (Z), of dx (X) and of dW (W): large, middle, small; dx of few tokens (X64, X16)
template <bool F32> struct Shapes {
    typedef Shape<256, 256, 2, 4, 2, 64, false, false, 1, true> ZL;
    typedef Shape<256, 128, 2, 4, 2, 64, false, false, 1, true> ZM;
    typedef Shape<128, 64, 4, 1, 3, 64, false, false, 1, true> ZS;
    typedef Shape<256, 256, 2, 4, 2, 64, true, false, 1> XL;
    typedef Shape<256, 128, 2, 4, 2, 64, true, false, 1> XM;
    typedef XM XS;
    typedef Shape<256, 64, 4, 1, 3, 64, true, false, 1> X64;
    typedef Shape<256, 16, 4, 1, 3, 64, true, false, 1> X16;
    typedef Shape<256, 256, 2, 4, 2, 64, true, true, 1> WL;
    typedef Shape<256, 128, 2, 4, 2, 64, true, true, 1> WM;
    typedef WM WS;
};
template <> struct Shapes<true> {
    typedef Shape<256, 128, 4, 2, 2, 32, false, false, 6, true> ZL;
    typedef Shape<128, 128, 2, 4, 3, 32, false, false, 6, true> ZM;
    typedef Shape<128, 64, 4, 2, 4, 32, false, false, 6, true> ZS;
    typedef Shape<256, 128, 4, 2, 2, 32, true, false, 6> XL;
    typedef Shape<128, 128, 2, 4, 3, 32, true, false, 6> XM;
    typedef Shape<128, 64, 4, 2, 4, 32, true, false, 6> XS;
    typedef Shape<256, 128, 4, 2, 2, 32, true, true, 6> WL;
    typedef Shape<128, 128, 2, 4, 3, 32, true, true, 6> WM;
    typedef Shape<128, 64, 4, 2, 4, 32, true, true, 6> WS;
};

// The time of a step of K, in 5 ns, of all rounds of tiles over the CUs
template <class S> int64_t rounds(int64_t m, int64_t n) {
    const int64_t ncu = m2::cu_count();
    return S::STEP * (((int64_t)tiles(m, S::BM) * tiles(n, S::BN) + ncu - 1) / ncu);
}
// What both entry points share: how the operands are read
struct Common {
    int64_t n, np, dim, hidden, dp, fp;
    bool f32, pack_x, pack_w;
    int shape;               // of the forward's product: 0 large, 1 middle, 2 small
    int tm, tn;              // its tiles
    int64_t entries;         // of the factors
    size_t z, x, w;          // bytes of the factors, and of x and weight where they are packed
};
template <class F> auto with_shape(bool f32, int shape, F&& f) {
    typedef Shapes<false> B;
    typedef Shapes<true> P;
    if (f32) return shape == 0 ? f(P::ZL()) : shape == 1 ? f(P::ZM()) : f(P::ZS());
    return shape == 0 ? f(B::ZL()) : shape == 1 ? f(B::ZM()) : f(B::ZS());
}
template <bool F32> int shape_of(int64_t m, int64_t n) {
    typedef Shapes<F32> P;
    const int64_t l = rounds<typename P::ZL>(m, n), md = rounds<typename P::ZM>(m, n), sm = rounds<typename P::ZS>(m, n);
    return n <= 64 || (sm < md && sm < l) ? 2 : md < l ? 1 : 0;
}
// save: with what a gradient reads, whose K runs along the rows of both operands too, and not along dim only
Common common(int64_t n, int64_t dim, int64_t hidden, int64_t ldx, int64_t ldw, const void* x, const void* w, int dtype,
              bool save) {
    Common c{};
    c.n = n; c.dim = dim; c.hidden = hidden;
    c.np = (n + 63) / 64 * 64;
    c.dp = (dim + 63) / 64 * 64;
    c.fp = (hidden + 63) / 64 * 64;
    c.f32 = dtype == M2_F32;
    const int64_t m = 2 * ((hidden + 15) / 16 * 16);
    c.shape = c.f32 ? shape_of<true>(m, n) : shape_of<false>(m, n);
    with_shape(c.f32, c.shape, [&](auto shape) {
        typedef decltype(shape) S;
        c.tm = tiles(m, S::BM);
        c.tn = tiles(n, S::BN);
        c.entries = entries<S>(m, n);
    });
    // in place: bf16 rows of whole 128-byte pieces, whose offsets within a tile fit 32 bits
    auto direct = [&](const void* p, int64_t ld, int64_t apart) {
        return !c.f32 && dim % 64 == 0 && ld % 8 == 0 && al16(p) && ld <= (1 << 22) && ld * (apart + 256) < (1ll << 31);
    };
    c.pack_x = !direct(x, ldx, 0);
    c.pack_w = !direct(w, ldw, hidden) || (save && hidden % 64);
    const size_t planes = c.f32 ? 3 : 1;
    c.z = save ? align256(c.f32 ? Factors<float>::bytes(c.entries) : Factors<bf16>::bytes(c.entries)) : 0;
    c.x = align256(2 * planes * (size_t)c.np * c.dp);
    c.w = align256(2 * planes * (size_t)2 * c.fp * c.dp);
    if (c.w == c.x) c.w += 256;              // (so that the size of `saved` tells what lies in it)
    return c;
}
// What the forward leaves for the gradient: the factors, then x and weight if it packed them.  The gradient goes by the size, for
// x and weight may lie elsewhere by then, with other strides and another alignment.
struct Kept {
    bool x, w, known;
};
Kept kept(const Common& c, size_t bytes) {
    if (bytes == c.z) return {false, false, true};
    if (bytes == c.z + c.x) return {true, false, true};
    if (bytes == c.z + c.w) return {false, true, true};
    return {true, true, bytes == c.z + c.x + c.w};
}

// An operand in place, or (to) packed there; pack: it is not there yet
template <typename T> Operand operand_x(bf16* to, const Common& c, const void* x, int64_t ldx, bool pack, hipStream_t s) {
    if (!to) return Operand{static_cast<const bf16*>(x), ldx, 0, (int)c.n, (int)c.dim};
    const PackArgs a{x, to, c.np, c.dim, ldx, c.dp, c.np * c.dp, 0, c.n};
    if (pack) pack_rows<T>(a, s);
    return Operand{to, c.dp, c.np * c.dp, (int)c.np, (int)c.dp};
}
template <typename T> Operand operand_w(bf16* to, const Common& c, const void* w, int64_t ldw, bool pack, hipStream_t s) {
    if (!to) return Operand{static_cast<const bf16*>(w), ldw, 0, (int)c.hidden, (int)c.dim, (int)c.hidden};
    const PackArgs a{w, to, 2 * c.fp, c.dim, ldw, c.dp, 2 * c.fp * c.dp, c.fp, c.hidden};
    if (pack) pack_rows<T>(a, s);
    return Operand{to, c.dp, 2 * c.fp * c.dp, (int)c.fp, (int)c.dp, (int)c.fp};
}

int check_sizes(const char* who, int64_t n, int64_t dim, int64_t hidden, int64_t ldx, int64_t ldw, int dtype,
                int activation) {
    M2_REQUIRE(n >= 0 && n < (1 << 30) && dim > 0 && dim <= (1 << 20) && hidden > 0 && hidden < (1 << 28), M2_ERR_INVALID,
               "%s: bad sizes (n %lld, dim %lld, hidden %lld)", who, (long long)n, (long long)dim, (long long)hidden);
    M2_REQUIRE(ldx >= dim && ldw >= dim, M2_ERR_INVALID, "%s: row strides", who);
    M2_REQUIRE(dtype == M2_F32 || dtype == M2_BF16, M2_ERR_UNSUPPORTED, "%s: dtype %d", who, dtype);
    M2_REQUIRE(activation == M2_SILU || activation == M2_GELU, M2_ERR_UNSUPPORTED, "%s: activation %d", who, activation);
    // (offsets between the halves of a tile's rows, and between 256 rows of dz; counts of tiles)
    M2_REQUIRE(hidden <= (1 << 21) && (hidden + 64) * ((dim + 63) / 64 * 64) < (1ll << 30) &&
                   (int64_t)tiles(2 * hidden, 128) * tiles(n, 16) < (1ll << 30),
               M2_ERR_UNSUPPORTED, "%s: too large", who);
    return M2_OK;
}

// 16-byte pieces along K that a lane loads by itself
template <class A> bool few(const A& a) {
    const int64_t es = a.dtype == M2_F32 ? 4 : 2;
    return a.n <= 64 && a.dim % 8 == 0 && a.ldx * es % 16 == 0 && a.ldw * es % 16 == 0 && al16(a.x) && al16(a.weight);
}
template <class A> Common common_of(const A& a, bool save) {
    return common(a.n, a.dim, a.hidden, a.ldx, a.ldw, a.x, a.weight, a.dtype, save);
}

template <typename T> void run_few(const m2_gated_linear_args& a, hipStream_t s) {
    typedef typename Shapes<sizeof(T) == 4>::ZS S;
    const FewArgs k{a.x, a.weight, a.out, a.saved, a.ldx, a.ldw, entries<S>(2 * ((a.hidden + 15) / 16 * 16), a.n),
                    (int)a.n, (int)a.dim, (int)a.hidden, a.activation == M2_GELU};
    auto go = [&](auto mt) {
        constexpr int MT = decltype(mt)::value;
        auto with = [&](auto ft, auto nw, auto u) {
            constexpr int FT = decltype(ft)::value, NW = decltype(nw)::value, U = decltype(u)::value;
            hipLaunchKernelGGL((k_glu_few<T, S, MT, FT, NW, U>), dim3((unsigned)((a.hidden + 8 * FT - 1) / (8 * FT))), dim3(NW * 64), 0, s, k);
        };
        typedef std::integral_constant<int, 1> one;
        typedef std::integral_constant<int, 2> two;
        typedef std::integral_constant<int, 4> four;
        typedef std::integral_constant<int, 8> eight;
        // More of the hidden size for each workgroup reads x less often, as long as there are workgroups for most
        // CUs: 16 tokens x 2560 x 6912 by 8, 16, 32, of weights that no cache holds: 29, 25, 24 us, 2048 x 1024: 6.6, 8.0, 11.6;
        // float32 45, 38, 35 and 12.6, 15.8, 24.
        const int64_t wgs = (a.hidden + 7) / 8;
        if (wgs < 2 * 192) with(one(), eight(), four());
        else if (wgs < 4 * 192) with(two(), eight(), two());
        else if constexpr (sizeof(T) == 4 && MT < 4) with(four(), eight(), two());
        else with(four(), four(), two());
    };
    if (a.n <= 16) go(std::integral_constant<int, 1>());
    else if (a.n <= 32) go(std::integral_constant<int, 2>());
    else go(std::integral_constant<int, 4>());
}

template <bool F32, bool SAVE> int run_fwd(const m2_gated_linear_args& a, const Common& c, hipStream_t s) {
    typedef typename std::conditional<F32, float, bf16>::type T;
    typedef Shapes<F32> P;
    char* ws = static_cast<char*>(SAVE ? a.saved : a.workspace);
    bf16* xp = c.pack_x ? reinterpret_cast<bf16*>(ws + c.z) : nullptr;
    bf16* wp = c.pack_w ? reinterpret_cast<bf16*>(ws + c.z + (xp ? c.x : 0)) : nullptr;
    Gemm g{};
    g.n = (int)c.n; g.splits = 1;
    g.nk = (int)(c.dp / 64);
    g.b = operand_x<T>(xp, c, a.x, a.ldx, true, s);
    g.a = operand_w<T>(wp, c, a.weight, a.ldw, true, s);
    const EpiGlu<T, SAVE> e{static_cast<T*>(a.out), Factors<T>(ws, c.entries), c.hidden, c.tn, a.activation == M2_GELU};
    g.tm = c.tm;
    g.tn = c.tn;
    if (c.shape == 2) launch<typename P::ZS>(g, e, s);
    else if (c.shape == 1) launch<typename P::ZM>(g, e, s);
    else launch<typename P::ZL>(g, e, s);
    return m2::check_launch("gated_linear");
}

struct BwdPlan {
    Common c;
    Kept kept;               // what lies in saved; what does not and cannot be read in place is packed into the workspace
    bool pack_x, pack_w;
    size_t xp, wp, dz, part, total;
    int x;                   // dx: 0 the large tiles, 1 the middle, 2 the small, 64 / 16 k_ce_stream's
    int w;                   // dW: the same
    int splits;
};
template <class S> Deal deal_of(int64_t m, int64_t n, int64_t k) {
    return deal(tiles(m, S::BM) * tiles(n, S::BN), (int)(k / 64), m2::cu_count(), S::STEP, S::SEG);
}
template <bool F32> BwdPlan plan_bwd(const m2_gated_linear_grad_args& a) {
    typedef Shapes<F32> P;
    BwdPlan p{};
    p.c = common_of(a, true);
    const Common& c = p.c;
    p.kept = kept(c, a.saved_bytes);
    p.pack_x = a.grad_weight && c.pack_x && !p.kept.x;
    p.pack_w = a.grad_x && c.pack_w && !p.kept.w;
    size_t at = 0;
    auto take = [&](size_t b) { const size_t r = at; at += align256(b); return r; };
    p.xp = take(p.pack_x ? c.x : 0);
    p.wp = take(p.pack_w ? c.w : 0);
    p.dz = take(2 * (size_t)(F32 ? 3 : 1) * c.np * 2 * c.fp);
    // (the two products run one after the other and share the parts' buffer)
    size_t need = 0;
    auto parts = [&](const Deal& d, size_t tile) {
        const size_t b = d.s > 1 ? 4 * tile * d.rest * d.s : 0;
        if (b > need) need = b;
    };
    auto choose = [&](auto large, auto middle, auto small, int64_t m, int64_t n, int64_t k) {
        typedef decltype(large) A;
        typedef decltype(middle) B;
        typedef decltype(small) S;
        const Deal da = deal_of<A>(m, n, k), db = deal_of<B>(m, n, k), ds = deal_of<S>(m, n, k);
        if (da.cost <= db.cost && da.cost <= ds.cost) { parts(da, (size_t)A::BM * A::BN); return 0; }
        if (db.cost <= ds.cost) { parts(db, (size_t)B::BM * B::BN); return 1; }
        parts(ds, (size_t)S::BM * S::BN);
        return 2;
    };
    if (a.grad_x) {
        if (!F32 && c.n <= 64) {
            // as many parts of K as fill the CUs; a part costs a float32 array of dx, written and read once
            p.x = c.n <= 16 ? 16 : 64;
            const int ncu = m2::cu_count(), steps = (int)(2 * c.fp / 64), t = tiles(c.dim, 256);
            double best = 1e300;
            p.splits = 1;
            for (int s = 1; s <= 64 && s * 4 <= steps; ++s) {
                const double cost = (double)((t * s + ncu - 1) / ncu) * ((double)steps / s + 12.0) + 0.02 * s * t;
                if (cost < best) { best = cost; p.splits = s; }
            }
            need = 4 * (size_t)p.splits * c.np * c.dp;
        } else {
            p.x = choose(typename P::XL(), typename P::XM(), typename P::XS(), c.dim, c.n, 2 * c.fp);
        }
    }
    if (a.grad_weight) p.w = choose(typename P::WL(), typename P::WM(), typename P::WS(), c.dim, 2 * c.fp, c.np);
    p.part = take(need);
    p.total = at;
    return p;
}

// wavefronts of k_glu_dz
template <class S> int64_t dz_waves(const Common& c) {
    return (int64_t)c.tm * c.tn * (S::BM * S::BN / 2 / 16 / (S::FM % 4 ? 16 : 32));
}

template <bool F32> int run_bwd(const m2_gated_linear_grad_args& a, const BwdPlan& p, hipStream_t s) {
    typedef typename std::conditional<F32, float, bf16>::type T;
    typedef Shapes<F32> P;
    char* ws = static_cast<char*>(a.workspace);
    const Common& c = p.c;
    auto at = [](const void* base, size_t off) { return reinterpret_cast<bf16*>(static_cast<char*>(const_cast<void*>(base)) + off); };
    bf16* xp = p.kept.x ? at(a.saved, c.z) : p.pack_x ? at(ws, p.xp) : nullptr;
    bf16* wp = p.kept.w ? at(a.saved, c.z + (p.kept.x ? c.x : 0)) : p.pack_w ? at(ws, p.wp) : nullptr;
    bf16* dz = reinterpret_cast<bf16*>(ws + p.dz);
    float* part = reinterpret_cast<float*>(ws + p.part);
    const int64_t plane = c.np * 2 * c.fp;
    const DzArgs d{a.saved, a.grad_out, dz, c.n, c.np, c.hidden, c.fp, a.ldg, plane, c.entries, c.tm, c.tn};
    auto make = [&](auto shape) {
        typedef decltype(shape) S;
        hipLaunchKernelGGL((k_glu_dz<T, S>), dim3((unsigned)((dz_waves<S>(c) + 3) / 4)), dim3(256), 0, s, d);
    };
    if (c.shape == 2) make(typename P::ZS());
    else if (c.shape == 1) make(typename P::ZM());
    else make(typename P::ZL());
    auto product = [&](auto shape, Gemm g, int64_t m, int64_t n, int64_t k, const Out<T>& out) {
        typedef decltype(shape) S;
        g.tm = tiles(m, S::BM);
        g.tn = tiles(n, S::BN);
        g.nk = g.seg_nk = (int)(k / 64);
        g.splits = m2::cu_count();
        const Deal dl = deal_of<S>(m, n, k);
        const EpiOut<T> e{out, part, dl.s > 1 ? dl.full : g.tm * g.tn};
        launch<S>(g, e, s);
        if (dl.s > 1) {
            const JoinArgs j{part, g.tm, g.tn, dl.full, dl.rest, dl.s};
            const int64_t waves = (int64_t)dl.rest * (S::NW * S::FM / 2 * S::FN);
            hipLaunchKernelGGL((k_glu_join<T, S>), dim3((unsigned)((waves + 3) / 4)), dim3(256), 0, s, j, out);
        }
    };
    if (a.grad_x) {
        Gemm g{};
        g.n = (int)c.n;
        g.a = operand_w<T>(wp, c, a.weight, a.ldw, p.pack_w, s);
        g.a.lim = g.a.klim;                  // read by columns
        g.a.klim = (int)(2 * c.fp);
        g.b = Operand{dz, 2 * c.fp, plane, (int)c.np, (int)(2 * c.fp)};
        const Out<T> out{static_cast<T*>(a.grad_x), c.dim, 0, (int)c.n};
        if (p.x > 2) {
            if constexpr (!F32) {
                g.tm = tiles(c.dim, 256);
                g.tn = 1;
                g.nk = (int)(2 * c.fp / 64);
                g.splits = p.splits;
                const EpiSplit e{part, c.np, c.dp};
                if (p.x == 16) launch<typename P::X16>(g, e, s);
                else launch<typename P::X64>(g, e, s);
                hipLaunchKernelGGL(k_glu_sum, dim3((unsigned)((c.dim + 255) / 256), (unsigned)c.n), dim3(64), 0, s, part,
                                   static_cast<bf16*>(a.grad_x), c.np, c.dp, c.dim, p.splits);
            }
        } else if (p.x == 0) {
            product(typename P::XL(), g, c.dim, c.n, 2 * c.fp, out);
        } else if (p.x == 1) {
            product(typename P::XM(), g, c.dim, c.n, 2 * c.fp, out);
        } else if constexpr (F32) {
            product(typename P::XS(), g, c.dim, c.n, 2 * c.fp, out);
        }
    }
    if (a.grad_weight) {
        Gemm g{};
        g.n = (int)(2 * c.fp);
        g.a = operand_x<T>(xp, c, a.x, a.ldx, p.pack_x, s);
        g.a.klim = g.a.lim;                  // read by columns; zero rows of dz stand against the repeated last row
        g.a.lim = (int)c.dp;
        g.b = Operand{dz, 2 * c.fp, plane, (int)(2 * c.fp), (int)c.np};
        const Out<T> out{static_cast<T*>(a.grad_weight), c.dim, (int)c.fp, (int)c.hidden};
        if (p.w == 0) product(typename P::WL(), g, c.dim, 2 * c.fp, c.np, out);
        else if (p.w == 1) product(typename P::WM(), g, c.dim, 2 * c.fp, c.np, out);
        else if constexpr (F32) product(typename P::WS(), g, c.dim, 2 * c.fp, c.np, out);
    }
    return m2::check_launch("gated_linear_grad");
}

}  // namespace

namespace m2 {

static size_t packed_bytes(const Common& c) { return (c.pack_x ? c.x : 0) + (c.pack_w ? c.w : 0); }

size_t gated_linear_saved(const m2_gated_linear_args& a) {
    if (check_sizes("gated_linear", a.n, a.dim, a.hidden, a.ldx, a.ldw, a.dtype, a.activation)) return 0;
    const Common c = common_of(a, true);
    // (few tokens are packed for the gradient alone)
    const size_t b = c.z + (few(a) ? 0 : packed_bytes(c));
    return b ? b : 256;
}

size_t gated_linear_workspace(const m2_gated_linear_args& a) {
    if (check_sizes("gated_linear", a.n, a.dim, a.hidden, a.ldx, a.ldw, a.dtype, a.activation)) return 0;
    const size_t b = a.saved || few(a) ? 0 : packed_bytes(common_of(a, false));
    return b ? b : 256;
}

int launch_gated_linear(const m2_gated_linear_args& a, hipStream_t s) {
    const char* who = "gated_linear";
    if (int rc = check_sizes(who, a.n, a.dim, a.hidden, a.ldx, a.ldw, a.dtype, a.activation)) return rc;
    M2_REQUIRE(a.n == 0 || (a.x && a.weight && a.out), M2_ERR_INVALID, "%s: x, weight and out are required", who);
    M2_REQUIRE(al16(a.saved) && al16(a.workspace), M2_ERR_WORKSPACE, "%s: saved and workspace of 16-byte alignment needed", who);
    M2_REQUIRE(!a.saved || a.saved_bytes >= gated_linear_saved(a), M2_ERR_WORKSPACE,
               "%s: saved of %zu bytes needed, %zu given", who, gated_linear_saved(a), a.saved_bytes);
    if (a.n == 0) return M2_OK;
    if (few(a)) {
        if (a.dtype == M2_F32) run_few<float>(a, s);
        else run_few<bf16>(a, s);
        return check_launch(who);
    }
    const Common c = common_of(a, a.saved != nullptr);
    if (a.saved) return c.f32 ? run_fwd<true, true>(a, c, s) : run_fwd<false, true>(a, c, s);
    const size_t need = packed_bytes(c);
    M2_REQUIRE(need == 0 || (a.workspace && a.workspace_bytes >= need), M2_ERR_WORKSPACE,
               "%s: workspace of %zu bytes needed, %zu given", who, need, a.workspace_bytes);
    return c.f32 ? run_fwd<true, false>(a, c, s) : run_fwd<false, false>(a, c, s);
}

static BwdPlan plan(const m2_gated_linear_grad_args& a) {
    return a.dtype == M2_F32 ? plan_bwd<true>(a) : plan_bwd<false>(a);
}

size_t gated_linear_grad_workspace(const m2_gated_linear_grad_args& a) {
    if (check_sizes("gated_linear_grad", a.n, a.dim, a.hidden, a.ldx, a.ldw, a.dtype, a.activation)) return 0;
    const size_t b = plan(a).total;
    return b ? b : 256;
}

int launch_gated_linear_grad(const m2_gated_linear_grad_args& a, hipStream_t s) {
    const char* who = "gated_linear_grad";
    if (int rc = check_sizes(who, a.n, a.dim, a.hidden, a.ldx, a.ldw, a.dtype, a.activation)) return rc;
    M2_REQUIRE(a.n > 0, M2_ERR_INVALID, "%s: no tokens", who);
    M2_REQUIRE(a.ldg >= a.hidden, M2_ERR_INVALID, "%s: row strides", who);
    M2_REQUIRE(a.x && a.weight && a.saved && a.grad_out && (a.grad_x || a.grad_weight), M2_ERR_INVALID,
               "%s: x, weight, saved, grad_out and an output are required", who);
    M2_REQUIRE(al16(a.saved) && al16(a.workspace), M2_ERR_WORKSPACE, "%s: saved and workspace of 16-byte alignment needed", who);
    const BwdPlan p = plan(a);
    int64_t waves = 0;
    with_shape(p.c.f32, p.c.shape, [&](auto shape) { waves = dz_waves<decltype(shape)>(p.c); });
    M2_REQUIRE(waves < (1 << 26) - 4, M2_ERR_UNSUPPORTED, "%s: too many tokens (a launch counts its threads in 32 bits)", who);
    M2_REQUIRE(p.kept.known, M2_ERR_WORKSPACE, "%s: saved of %zu bytes is no forward's of these sizes", who, a.saved_bytes);
    M2_REQUIRE(a.workspace && a.workspace_bytes >= p.total, M2_ERR_WORKSPACE,
               "%s: workspace of %zu bytes needed, %zu given", who, p.total, a.workspace_bytes);
    return a.dtype == M2_F32 ? run_bwd<true>(a, p, s) : run_bwd<false>(a, p, s);
}

}  // namespace m2
