// Tiled bf16 matrix product D[m, n] = sum_k A[m, k] B[n, k] of the vocabulary's loss
// (linear_ce.hip) and of the gated feed-forward product (gated_linear.hip), with the epilogue as a template
// parameter: the logits, or the two products, of a tile exist in its accumulators only.
//
// A tile is BM x BN, K in steps of BK (64 or 32) through a ring of ST LDS slots filled by
// direct global -> LDS loads; WM x WN wavefronts, 16x16x32 MFMAs.  Each operand
// is stored in global memory either with K contiguous ("row": A[m][k]) or with K strided
// ("col": A[k][m]):
//   row tile in LDS: [R][BK], rows whose 16-byte pieces are XOR-swizzled by the row
//     (swz); fragments by ds_read_b128, without bank conflicts;
//   col tile in LDS: [BK][R], rows of 2 R bytes whose 32-byte pieces (the 16
//     columns of one fragment) are XOR-swizzled by f(k) = k & 3 | (k >> 3 & 1) << 2 (as far
//     as R has pieces);
//     fragments by ds_read_b64_tr_b16, whose sixteen lanes read 4 k rows: the 8 rows that
//     32 lanes touch lie on different banks.
// The swizzle is applied to the global address of each lane, since a direct
// load writes LDS linearly.
//
// float32 operands come as three bf16 planes (v = p0 + p1 + p2 exactly but for
// the last bits); the products p_i q_j with i + j <= 2 are added up, the small ones
// first; what is left out is 2^-24 of the product.
#pragma once

#include "m2_internal.h"

namespace m2ce {

// ---------------------------------------------------------------------------
// rows in and out
// ---------------------------------------------------------------------------
// 8 consecutive elements of a row, zero past its end
template <typename T> M2_DEV void load8(const T* row, int64_t c, int64_t dim, float (&v)[8]) {
    if (c + 8 <= dim) {
        if constexpr (sizeof(T) == 2) {
            const u32x4 r = load16(row + c);
#pragma unroll
            for (int i = 0; i < 4; ++i) { v[2 * i] = bf16_lo(r[i]); v[2 * i + 1] = bf16_hi(r[i]); }
        } else {
            const u32x4 a = load16(row + c), b = load16(row + c + 4);
#pragma unroll
            for (int i = 0; i < 4; ++i) { v[i] = __uint_as_float(a[i]); v[4 + i] = __uint_as_float(b[i]); }
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = c + i < dim ? to_f32(row[c + i]) : 0.f;
    }
}
// v = h + m + l, each bf16 (an infinity or NaN stays in h alone)
M2_DEV void split3(float v, float& h, float& m, float& l) {
    h = (float)(bf16)v;
    const float r = v - h;
    const bool fin = fabsf(h) < __builtin_inff();
    m = fin ? (float)(bf16)r : 0.f;
    l = fin ? r - m : 0.f;
}
template <bool PLANES> M2_DEV void store8(bf16* p, int64_t plane, const float (&v)[8]) {
    if constexpr (!PLANES) {
        const u32x4 r = {pk_bf16(v[0], v[1]), pk_bf16(v[2], v[3]), pk_bf16(v[4], v[5]), pk_bf16(v[6], v[7])};
        *reinterpret_cast<u32x4*>(p) = r;
    } else {
        float h[8], m[8], l[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) split3(v[i], h[i], m[i], l[i]);
        store8<false>(p, 0, h);
        store8<false>(p + plane, 0, m);
        store8<false>(p + 2 * plane, 0, l);
    }
}

// Two fragments of 16 m beside each other, x and y: lane rows (16 lanes) 0 and 2 exchange
// theirs of y for rows 1's and 3's of x, after which a lane holds 8 consecutive m from
// pair_m on: (p, q)
M2_DEV void pair_swap(uint32_t& p, uint32_t& q) {
    const auto r = __builtin_amdgcn_permlane16_swap(p, q, false, false);
    p = r[0];
    q = r[1];
}
M2_DEV int pair_m(int lane) { return 16 * ((lane >> 4) & 1) + 8 * (lane >> 5); }
M2_DEV void store_pair(bf16* d, const float (&x)[4], const float (&y)[4]) {
    uint32_t a0 = pk_bf16(x[0], x[1]), a1 = pk_bf16(x[2], x[3]);
    uint32_t b0 = pk_bf16(y[0], y[1]), b1 = pk_bf16(y[2], y[3]);
    pair_swap(a0, b0);
    pair_swap(a1, b1);
    *reinterpret_cast<u32x4*>(d) = u32x4{a0, a1, b0, b1};
}
// the 32 values of m from m0 on (two fragments) of one n into a row of dim elements
template <typename T>
M2_DEV void store_row(T* row, int m0, int64_t dim, int lane, const f32x4& x, const f32x4& y) {
    if constexpr (sizeof(T) == 2) {
        // (the exchange is among the lanes of this n: all of them are here)
        uint32_t p[4] = {pk_bf16(x[0], x[1]), pk_bf16(x[2], x[3]), pk_bf16(y[0], y[1]), pk_bf16(y[2], y[3])};
        pair_swap(p[0], p[2]);
        pair_swap(p[1], p[3]);
        const int m = m0 + pair_m(lane);
        if (m + 8 <= dim) {
            store16(row + m, u32x4{p[0], p[1], p[2], p[3]});
        } else {
#pragma unroll
            for (int r = 0; r < 8; ++r)
                if (m + r < dim) reinterpret_cast<uint16_t*>(row)[m + r] = (uint16_t)(p[r >> 1] >> (16 * (r & 1)));
        }
    } else {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int m = m0 + 16 * e + 4 * (lane >> 4);
            const f32x4& v = e ? y : x;
            if (m + 4 <= dim) {
                store16(row + m, __builtin_bit_cast(u32x4, v));
            } else {
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (m + r < dim) row[m + r] = v[r];
            }
        }
    }
}

struct Operand {
    const bf16* p;
    int64_t ld;          // elements between rows (row: of m; col: of k)
    int64_t plane;       // elements between the planes of a float32 operand
    int lim;             // valid m (row: rows past it read the last one; col: columns, a multiple of 8)
    int klim;            // valid k (row: pieces past it read zeros; col: rows past it read the last one)
    int pair;            // of a paired row operand: rows between the two halves
};

struct Gemm {
    Operand a, b;
    const int* count;    // tokens that take part (device), or NULL: n
    int n;
    int nk;              // K steps of 64, 0: from count
    int tm, tn;
    int tok_n;           // n is the token: tiles past the kept ones are left out
    int splits;          // k_ce_stream: K in so many parts
    int seg_nk;          // persistent kernels with EPI::SEG: the K steps that deal() goes by
};

// Persistent kernels with EPI::SEG: as many whole tiles as fill the workgroups, and the rest of the tiles
// cut in s parts of K each, so that few workgroups are idle in the end.  Parts of the same
// K lie beside each other (they share panels).  Segment numbers: the tile of a whole
// one; full + part * rest + (tile - full).
struct Deal {
    int full, rest, s;
    int64_t cost;            // 5 ns
};
// step: the time of one, seg: of writing and reading a segment by the whole chip, in 5 ns
// (whole numbers: the host sizes the workspace by the same)
__host__ __device__ inline Deal deal(int tiles, int nk, int nwg, int step, int seg) {
    Deal d;
    d.full = tiles / nwg * nwg;
    d.rest = tiles - d.full;
    d.s = 1;
    d.cost = INT64_MAX;
    for (int s = 1; s <= 64 && (s == 1 || (s * 4 <= nk && d.rest * s <= 2 * nwg)); ++s) {
        const int64_t cost = (int64_t)step * ((d.rest * s + nwg - 1) / nwg) * ((nk + s - 1) / s) + (int64_t)seg * d.rest * s;
        if (cost < d.cost) { d.cost = cost; d.s = s; }
    }
    d.cost += (int64_t)(d.full / nwg) * nk * step + (int64_t)seg * d.full;
    return d;
}

__device__ const uint32_t ZEROS[4] = {0, 0, 0, 0};      // what stands past a row's end

// ---------------------------------------------------------------------------
// global -> LDS: R rows (columns) of BK of K
// ---------------------------------------------------------------------------
// 16-byte piece p of row r of a row tile lies at slot p ^ swz(r) of the row: 16 rows of one
// piece fill all banks, and so do the quarters of 16 lanes that a ds_read_b128 takes
// together (4 rows of two pieces each)
template <int BK> M2_DEV int swz(int r) {
    if constexpr (BK == 64) return r & 7;
    const int b = (r >> 2) & 3;
    return ((b ^ (b >> 1)) & 1) << 1 | b >> 1;
}

// PAIR (row operands): the tile's rows are 16 of one half of the matrix and the same 16 of the other
// half, in turn, so that a wavefront's accumulators hold both of each pair; m0 counts the rows
// of both, lim those of a half.
template <int R, bool TR, int NW, int BK, bool PAIR = false> struct Loader {
    static_assert(!(TR && PAIR), "");
    static constexpr int BYTES = R * BK * 2;
    static constexpr int INSTR = BYTES / 1024;                   // 1 KB each
    static constexpr int J = INSTR >= NW ? INSTR / NW : 1;       // per wavefront
    static constexpr int PP = BK / 8;                            // pieces of a row
    static constexpr int PR = R / 8;                             // pieces of a k row
    uint32_t off[J];         // byte offset from the tile's base
    int m0;

    // m0: first row (column) of the tile
    M2_DEV void init(const Operand& o, int m0_, int w, int lane) {
        m0 = PAIR ? m0_ / 2 : m0_;
#pragma unroll
        for (int j = 0; j < J; ++j) {
            const int in = (w * J + j) % INSTR;
            if constexpr (PAIR) {
                const int row = in * (64 / PP) + lane / PP;
                const int c = (lane & (PP - 1)) ^ swz<BK>(row);
                const int f = min(m0 + (row >> 5) * 16 + (row & 15), o.lim - 1) - m0;
                off[j] = (uint32_t)((int64_t)(f + ((row >> 4) & 1) * o.pair) * o.ld * 2 + c * 16);
            } else if constexpr (!TR) {
                const int row = in * (64 / PP) + lane / PP;
                const int c = (lane & (PP - 1)) ^ swz<BK>(row);
                off[j] = (uint32_t)((int64_t)(min(m0 + row, o.lim - 1) - m0) * o.ld * 2 + c * 16);
            } else {
                const int q = in * 64 + lane;
                const int k = q / PR, c = q % PR;
                const int f = ((k & 3) | (((k >> 3) & 1) << 2)) & (R / 16 - 1);
                int m = ((((c >> 1) ^ f) << 1) | (c & 1)) * 8;
                m = min(m0 + m, o.lim - 8) - m0;
                off[j] = (uint32_t)((int64_t)k * o.ld * 2 + m * 2);
            }
        }
    }
    // K step kt of plane pl: where it begins
    M2_DEV const bf16* base(const Operand& o, int kt, int pl) const {
        if constexpr (!TR) return o.p + pl * o.plane + (int64_t)m0 * o.ld + (int64_t)kt * BK;
        else return o.p + pl * o.plane + (int64_t)min(kt * BK, o.klim - 1) * o.ld + m0;
    }
    // load j of a step into the tile at LDS address `lds`; no branches: a row operand holds
    // whole steps, a col operand's rows past the end are its last one
    M2_DEV void piece(const Operand& o, const bf16* base, int kt, int j, uint32_t lds, int w, int lane) const {
        const int in = (w * J + j) % INSTR;
        if constexpr (!TR) {
            dma16s(base, off[j], lds + in * 1024);
        } else {
            const int k = (in * 64 + lane) / PR;
            const int last = o.klim - 1 - min(kt * BK, o.klim - 1);
            dma16s(base, off[j] - (uint32_t)max(k - last, 0) * (uint32_t)(o.ld * 2), lds + in * 1024);
        }
    }
    // a whole step; a row operand's pieces past klim read zeros
    M2_DEV void issue(const Operand& o, int kt, int pl, uint32_t lds, int w, int lane) const {
        const bf16* b = base(o, kt, pl);
        if (TR || kt * BK + BK <= o.klim) {
#pragma unroll
            for (int j = 0; j < J; ++j) piece(o, b, kt, j, lds, w, lane);
        } else {
#pragma unroll
            for (int j = 0; j < J; ++j) {
                const int in = (w * J + j) % INSTR;
                const int c = (lane & (PP - 1)) ^ swz<BK>(in * (64 / PP) + lane / PP);
                dma16(kt * BK + c * 8 < o.klim ? reinterpret_cast<const char*>(b) + off[j]
                                               : reinterpret_cast<const char*>(ZEROS), lds + in * 1024);
            }
        }
    }
};

// ---------------------------------------------------------------------------
// LDS -> fragments: F fragments of 16 rows from row r0 of the tile, 32 of K from 32 kk on
// ---------------------------------------------------------------------------
template <int R, bool TR, int F, int BK> struct Reader {
    int x;
    M2_DEV void init(int r0, int lane) {
        if constexpr (!TR) {
            x = (r0 + (lane & 15)) * BK * 2;
        } else {
            const int g = lane >> 4, r = (lane & 15) >> 2;
            const int f = (r | ((g & 1) << 2)) & (R / 16 - 1);
            x = (8 * g + r) * (2 * R) + (lane & 3) * 8 + (((r0 >> 4) ^ f) << 5);
        }
    }
    M2_DEV bf16x8 one(const char* s, int kk, int lane, int i) const {
        if constexpr (!TR) {
            const int sl = (((lane >> 4) + 4 * kk) ^ swz<BK>(lane & 15)) << 4;
            return *reinterpret_cast<const bf16x8*>(s + x + sl + i * 32 * BK);
        } else {
            const char* p = s + (x ^ (i << 5)) + kk * 32 * 2 * R;
            const bf16x4 lo = ds_read_tr(p), hi = ds_read_tr(p + 4 * 2 * R);
            return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        }
    }
    M2_DEV void read(const char* s, int kk, int lane, bf16x8 (&o)[F]) const {
#pragma unroll
        for (int i = 0; i < F; ++i) o[i] = one(s, kk, lane, i);
    }
};

template <int BM_, int BN_, int WM_, int WN_, int ST_, int BK_, bool ATR_, bool BTR_, int TERMS_, bool PAIR_ = false>
struct Shape {
    static constexpr int BK = BK_, BM = BM_, BN = BN_, WM = WM_, WN = WN_, ST = ST_, TERMS = TERMS_;
    static constexpr bool ATR = ATR_, BTR = BTR_;
    static constexpr int NW = WM * WN, NT = NW * 64;
    static constexpr int FM = BM / WM / 16, FN = BN / WN / 16;
    typedef Loader<BM, ATR, NW, BK, PAIR_> LA;
    typedef Loader<BN, BTR, NW, BK> LB;
    static constexpr int SLOT = LA::BYTES + LB::BYTES;
    static constexpr int LDS = SLOT * ST;
    static constexpr int LOADS = LA::J + LB::J;
    // what deal() and the choices of shapes go by: 1.4 us a step of 256 x 256 (as measured), 0.85 us of 256 x 128,
    // 0.5 us of 128 x 64; six products 4.5 us of 256 x 128, 2.4 us of 128 x 128, 1.5 us of 128 x 64; a segment of
    // 256 KB 0.11 us
    static constexpr int STEP = TERMS == 1 ? (BN == 256 ? 280 : BN == 64 ? 100 : 170)
                                : BN == 128 ? (BM == 128 ? 480 : 900) : BN == 64 ? 300 : 100;
    static constexpr int SEG = BM * BN * 22 / 65536 + 1;
};

// bf16, few tokens (or tiles): the operand of the vocabulary streams from HBM through a deep
// ring, two workgroups a CU where two rings of the shape fit its LDS (the logits' and dw's do,
// dx's tiles of 256 columns do not).  16 tokens over 50288 x 2560: 257 MB in 51 us, 5.0 TB/s (38
// where a part of the weights is in the last-level cache).
template <class S, class EPI>
__global__ void __launch_bounds__(S::NT, 2 * S::LDS <= 160 * 1024 ? 2 : 1) k_ce_stream(Gemm g, EPI epi) {
    __shared__ __align__(1024) char smem[S::LDS];
    const int lane = threadIdx.x & 63, w = wave_id();
    const int wm = w / S::WN, wn = w % S::WN;
    // tiles of one XCD: 8 tiles of m beside each other, then the next n (shared panels in its L2)
    int id = xcd_remap(blockIdx.x, gridDim.x);
    const int per = g.tm * g.tn;
    const int split = id / per;
    id -= split * per;
    const int grp = id / (8 * g.tn), gm = min(8, g.tm - grp * 8), in = id - grp * 8 * g.tn;
    const int tm = grp * 8 + in % gm, tn = in / gm;
    const int m0 = tm * S::BM, n0 = tn * S::BN;

    const int count = g.count ? *g.count : g.n;
    if (g.tok_n && n0 >= ((count + 63) & ~63)) return;
    const int nk = g.nk ? g.nk : (count + 63) >> 6;
    const int k0 = (int)((int64_t)nk * split / g.splits), k1 = (int)((int64_t)nk * (split + 1) / g.splits);
    const int total = k1 - k0;

    typename S::LA la;
    typename S::LB lb;
    la.init(g.a, m0, w, lane);
    lb.init(g.b, n0, w, lane);
    const uint32_t lds0 = lds_addr(smem);
    int ikt = k0, islot = 0;
    auto issue = [&]() {
        const uint32_t l = lds0 + islot * S::SLOT;
        la.issue(g.a, ikt, 0, l, w, lane);
        lb.issue(g.b, ikt, 0, l + S::LA::BYTES, w, lane);
        ++ikt;
        if (++islot == S::ST) islot = 0;
    };

    Reader<S::BM, S::ATR, S::FM, S::BK> ra;
    Reader<S::BN, S::BTR, S::FN, S::BK> rb;
    ra.init(wm * S::FM * 16, lane);
    rb.init(wn * S::FN * 16, lane);

    f32x4 acc[S::FM][S::FN];
#pragma unroll
    for (int i = 0; i < S::FM; ++i)
#pragma unroll
        for (int j = 0; j < S::FN; ++j) acc[i][j] = zero4();

#pragma unroll
    for (int s = 0; s < S::ST - 1; ++s)
        if (s < total) issue();
    int slot = 0;
    for (int it = 0; it < total; ++it) {
        // step `it` has landed; everybody is done with the slot that is filled next
        if (it + S::ST - 1 <= total) wait_vmem<(S::ST - 2) * S::LOADS>();
        else wait_vmem<0>();
        lds_barrier();
        if (it + S::ST - 1 < total) issue();
        const char* sa = smem + slot * S::SLOT;
        const char* sb = sa + S::LA::BYTES;
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
            bf16x8 fa[S::FM], fb[S::FN];
            ra.read(sa, kk, lane, fa);
            rb.read(sb, kk, lane, fb);
#pragma unroll
            for (int i = 0; i < S::FM; ++i)
#pragma unroll
                for (int j = 0; j < S::FN; ++j)
                    acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fa[i], fb[j], acc[i][j], 0, 0, 0);
        }
        if (++slot == S::ST) slot = 0;
    }
    epi.template run<S>(acc, m0, n0, wm, wn, lane, count, split, tm);
}

struct Work {                 // of a workgroup: its item i, a tile and its K steps of 64
    int i, tile, k0, k1, seg;
};
// The tiles and segments of a workgroup of the persistent kernels: whole tiles one workgroup
// after the other, each XCD a contiguous range, which its share of the workgroups gives.
template <class S, class EPI> struct Schedule {
    int tm_all, tn_all, nk, full, rest, s, f0, rounds, r0, r1, lw, items;

    M2_DEV void init(const Gemm& g, int count) {
        tm_all = g.tm;
        tn_all = g.tok_n ? min(g.tn, (((count + 63) & ~63) + S::BN - 1) / S::BN) : g.tn;
        nk = g.nk ? g.nk : (count + 63) >> 6;
        const int tiles = g.tm * tn_all;
        const int xcd = blockIdx.x & 7, local = blockIdx.x >> 3, nwg = gridDim.x;
        lw = (nwg - xcd + 7) >> 3;
        const int before = xcd * (nwg >> 3) + min(xcd, nwg & 7);
        full = 0; rest = tiles; s = 1;
        if constexpr (EPI::SEG) {
            const Deal d = deal(tiles, g.seg_nk, nwg, S::STEP, S::SEG);
            full = d.full; rest = d.rest; s = d.s;
        }
        f0 = full / nwg * before + local;
        rounds = full / nwg;
        const int64_t cut = (int64_t)rest * s;
        r0 = (int)(cut * before / nwg) + local;
        r1 = (int)(cut * (before + lw) / nwg);
        items = rounds + (r1 > r0 ? (r1 - r0 + lw - 1) / lw : 0);
    }
    M2_DEV Work work(int i) const {
        if (EPI::SEG && i < rounds) return Work{i, f0 + i * lw, 0, nk, f0 + i * lw};
        const int id = r0 + (i - rounds) * lw;
        const int part = EPI::SEG ? id / rest : 0;
        Work x{i, full + id - part * rest, 0, nk, full + id};
        if constexpr (EPI::SEG) {
            x.k0 = (int)((int64_t)nk * part / s);
            x.k1 = (int)((int64_t)nk * (part + 1) / s);
        }
        return x;
    }
    // the first item from i on that has steps (a short piece's parts may not), or items
    M2_DEV int with_steps(int i) const {
        if constexpr (EPI::SEG)
            for (; i < items; ++i) {
                const Work x = work(i);
                if (x.k0 < x.k1) break;
            }
        return i;
    }
    // 8 tiles of m beside each other, then the next n
    M2_DEV void place(int tile, int& tm, int& m0, int& n0) const {
        const int grp = tile / (8 * tn_all), gm = min(8, tm_all - grp * 8), in = tile - grp * 8 * tn_all;
        tm = grp * 8 + in % gm;
        m0 = tm * S::BM;
        n0 = in / gm * S::BN;
    }
};
template <class LD> struct Cursor {      // the step of an operand that is loaded next
    LD ld;
    Work at;
    int k;
};

// bf16, many tokens.  K in steps of 64, A through a ring of three slots, B of two (all
// 160 KB for 256 x 256); the fragments of a half step (32 of K) are read while the half step
// before multiplies, so the matrix units wait for neither LDS nor the other
// wavefronts but once a step:
//   half 0 of step i: multiply F0, read F1 (half 1 of step i), load A of step i + 2
//   wait until step i + 1 has landed; barrier: everybody has read step i
//   half 1 of step i: multiply F1, read F0 (half 0 of step i + 1), load B of step i + 2
// so that both halves carry as many loads (all of them in one half leave too few cycles for
// the 64 bytes a cycle that a CU takes in).  The loads run on into the next tile, whose first
// steps arrive during the epilogue.
// 8192 x 50288 x 2560 with EpiLse: 1.55 ms, 1.36 PFLOP/s (a library product of these sizes 1.75 ms).
// The matrix units are busy in 70 % of the cycles, at the 1.82 GHz that the card's power leaves
// them (with 59 % busy it ran at 1.9 GHz): what is left to gain in cycles the clock
// takes back.  Measured and dropped: steps of 32 through a ring of four (a barrier twice
// as often, half cache lines: 12 % slower), one contiguous round of tiles over all XCDs
// (5 % slower: less of a panel stays in an XCD's L2).
template <class S, class EPI>
__global__ void __launch_bounds__(S::NT, S::NT / 256) k_ce_tile(Gemm g, EPI epi) {
    static_assert(S::BK == 64 && S::TERMS == 1, "");
    constexpr int B_AT = 3 * S::LA::BYTES;
    __shared__ __align__(1024) char smem[B_AT + 2 * S::LB::BYTES];
    const int lane = threadIdx.x & 63, w = wave_id();
    const int wm = w / S::WN, wn = w % S::WN;
    const int count = g.count ? *g.count : g.n;
    Schedule<S, EPI> sc;
    sc.init(g, count);
    const int first = sc.nk > 0 ? sc.with_steps(0) : 0;
    if (first >= sc.items) return;
    Cursor<typename S::LA> ca;
    Cursor<typename S::LB> cb;
    auto start = [&](auto& c, const Operand& o, bool is_a, int item) {
        int tm, m0, n0;
        c.at = sc.work(item);
        sc.place(c.at.tile, tm, m0, n0);
        c.ld.init(o, is_a ? m0 : n0, w, lane);
        c.k = c.at.k0;
    };
    // past the last step the last tile's last step is loaded again (nobody reads it)
    auto next = [&](auto& c, const Operand& o, bool is_a) {
        if (++c.k < c.at.k1) return;
        const int i = sc.with_steps(c.at.i + 1);
        if (i < sc.items) start(c, o, is_a, i);
        else c.k = c.at.k1 - 1;
    };
    const uint32_t lds0 = lds_addr(smem);

    Reader<S::BM, S::ATR, S::FM, 64> ra;
    Reader<S::BN, S::BTR, S::FN, 64> rb;
    ra.init(wm * S::FM * 16, lane);
    rb.init(wn * S::FN * 16, lane);
    f32x4 acc[S::FM][S::FN];
    bf16x8 a0[S::FM], b0[S::FN], a1[S::FM], b1[S::FN];
    int sa = 0, sb = 0;           // byte offsets of the slots of the current step
    auto after = [](int slot) { return slot == 2 * S::LA::BYTES ? 0 : slot + S::LA::BYTES; };
    if (sc.nk > 0) {
        start(ca, g.a, true, first);
        start(cb, g.b, false, first);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            ca.ld.issue(g.a, ca.k, 0, lds0 + i * S::LA::BYTES, w, lane);
            cb.ld.issue(g.b, cb.k, 0, lds0 + B_AT + i * S::LB::BYTES, w, lane);
            next(ca, g.a, true);
            next(cb, g.b, false);
        }
        wait_vmem<S::LOADS>();
        lds_barrier();
        ra.read(smem, 0, lane, a0);
        rb.read(smem + B_AT, 0, lane, b0);
    }
    constexpr int RD = S::FM + S::FN;
    for (int item = first; item < sc.items; item = sc.with_steps(item + 1)) {
        const Work wk = sc.work(item);
        int tm, m0, n0;
        sc.place(wk.tile, tm, m0, n0);
#pragma unroll
        for (int i = 0; i < S::FM; ++i)
#pragma unroll
            for (int j = 0; j < S::FN; ++j) acc[i][j] = zero4();
        const int steps = wk.k1 - wk.k0;
        for (int st = 0; st < steps; ++st) {
            {
                const char* pa = smem + sa;
                const char* pb = smem + B_AT + sb;
                const uint32_t l = lds0 + after(after(sa));
                const bf16* from = ca.ld.base(g.a, ca.k, 0);
#pragma unroll
                for (int i = 0; i < S::FM; ++i) {
#pragma unroll
                    for (int q = i * RD / S::FM; q < (i + 1) * RD / S::FM; ++q) {
                        if (q < S::FN) b1[q] = rb.one(pb, 1, lane, q);
                        else a1[q - S::FN] = ra.one(pa, 1, lane, q - S::FN);
                    }
#pragma unroll
                    for (int q = i * S::LA::J / S::FM; q < (i + 1) * S::LA::J / S::FM; ++q)
                        ca.ld.piece(g.a, from, ca.k, q, l, w, lane);
#pragma unroll
                    for (int j = 0; j < S::FN; ++j)
                        acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a0[i], b0[j], acc[i][j], 0, 0, 0);
                    __builtin_amdgcn_sched_barrier(0);
                }
                next(ca, g.a, true);
            }
            // (behind an epilogue they have: its stores need not have)
            if (st > 0 || item == first) wait_vmem<S::LA::J>();
            lds_barrier();
            __builtin_amdgcn_sched_barrier(0);
            {
                const uint32_t l = lds0 + B_AT + sb;
                sa = after(sa);
                sb ^= S::LB::BYTES;
                const char* pa = smem + sa;
                const char* pb = smem + B_AT + sb;
                const bf16* from = cb.ld.base(g.b, cb.k, 0);
#pragma unroll
                for (int i = 0; i < S::FM; ++i) {
#pragma unroll
                    for (int q = i * RD / S::FM; q < (i + 1) * RD / S::FM; ++q) {
                        if (q < S::FN) b0[q] = rb.one(pb, 0, lane, q);
                        else a0[q - S::FN] = ra.one(pa, 0, lane, q - S::FN);
                    }
#pragma unroll
                    for (int q = i * S::LB::J / S::FM; q < (i + 1) * S::LB::J / S::FM; ++q)
                        cb.ld.piece(g.b, from, cb.k, q, l, w, lane);
#pragma unroll
                    for (int j = 0; j < S::FN; ++j)
                        acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a1[i], b1[j], acc[i][j], 0, 0, 0);
                    __builtin_amdgcn_sched_barrier(0);
                }
                next(cb, g.b, false);
            }
        }
        // what is loaded so far (step 0 and 1 of the next tile) is there before any store
        wait_vmem<0>();
        epi.template run<S>(acc, m0, n0, wm, wn, lane, count, wk.seg, tm);
    }
    wait_vmem<0>();           // no load may land after the workgroup has ended
}

// float32 operands, any number of tokens: persistent workgroups, steps of 32 of K through ST
// slots that hold the three planes of both operands: each plane is loaded once for the
// products it takes part in (loading the pair of planes of one product after the
// other moves twice as much and takes six times as many steps, whose latency is
// what bounds a few tiles).  B's fragments of a step and those of one row of A's stay in
// registers; the row after it is read while this one multiplies.  The last row of a step
// multiplies behind the step's barrier, while the next step's first fragments are read
// and the slot is filled again.  1024 x 50288 x 768, a quarter of the tokens left out: dw in
// 305 us, 1.17 PFLOP/s of the six products (pair by pair 428 us).
template <class S, class EPI>
__global__ void __launch_bounds__(S::NT, S::NT / 256) k_ce_planes(Gemm g, EPI epi) {
    static_assert(S::BK == 32 && S::TERMS == 6 && S::FM % 2 == 0, "");
    constexpr int PA = S::LA::BYTES, PB = S::LB::BYTES, SLOT = 3 * (PA + PB), LOADS = 3 * S::LOADS;
    __shared__ __align__(1024) char smem[SLOT * S::ST];
    const int lane = threadIdx.x & 63, w = wave_id();
    const int wm = w / S::WN, wn = w % S::WN;
    const int count = g.count ? *g.count : g.n;
    Schedule<S, EPI> sc;
    sc.init(g, count);
    const int first = sc.nk > 0 ? sc.with_steps(0) : 0;
    if (first >= sc.items) return;
    Cursor<typename S::LA> c;
    typename S::LB lb;
    auto start = [&](int item) {
        int tm, m0, n0;
        c.at = sc.work(item);
        sc.place(c.at.tile, tm, m0, n0);
        c.ld.init(g.a, m0, w, lane);
        lb.init(g.b, n0, w, lane);
        c.k = 2 * c.at.k0;
    };
    // past the last step the last tile's last step is loaded again (nobody reads it)
    auto next = [&]() {
        if (++c.k < 2 * c.at.k1) return;
        const int i = sc.with_steps(c.at.i + 1);
        if (i < sc.items) start(i);
        else c.k = 2 * c.at.k1 - 1;
    };
    // load q of a step's LOADS
    auto load = [&](int q, uint32_t l) {
        constexpr int J = S::LA::J, K = S::LB::J;
        if (q < 3 * J) c.ld.piece(g.a, c.ld.base(g.a, c.k, q / J), c.k, q % J, l + q / J * PA, w, lane);
        else lb.piece(g.b, lb.base(g.b, c.k, (q - 3 * J) / K), c.k, (q - 3 * J) % K, l + 3 * PA + (q - 3 * J) / K * PB, w, lane);
    };
    const uint32_t lds0 = lds_addr(smem);
    Reader<S::BM, S::ATR, S::FM, 32> ra;
    Reader<S::BN, S::BTR, S::FN, 32> rb;
    ra.init(wm * S::FM * 16, lane);
    rb.init(wn * S::FN * 16, lane);
    f32x4 acc[S::FM][S::FN];
    bf16x8 a[2][3], b0[3][S::FN], b1[3][S::FN];
    int slot = 0;                 // byte offset of the current step's
    if (sc.nk > 0) {
        start(first);
#pragma unroll
        for (int i = 0; i < S::ST; ++i) {
#pragma unroll
            for (int q = 0; q < LOADS; ++q) load(q, lds0 + i * SLOT);
            next();
        }
        wait_vmem<(S::ST - 1) * LOADS>();
        lds_barrier();
#pragma unroll
        for (int p = 0; p < 3; ++p) {
            rb.read(smem + 3 * PA + p * PB, 0, lane, b0[p]);
            a[0][p] = ra.one(smem + p * PA, 0, lane, 0);
        }
    }
    // the small products first
    constexpr int PI[6] = {0, 2, 1, 0, 1, 0}, PJ[6] = {2, 0, 1, 1, 0, 0};
    auto step = [&](const bf16x8(&b)[3][S::FN], bf16x8(&nb)[3][S::FN]) {
        const char* s0 = smem + slot;
        const uint32_t l = lds0 + slot;
        slot = slot == (S::ST - 1) * SLOT ? 0 : slot + SLOT;
        const char* s1 = smem + slot;
#pragma unroll
        for (int i = 0; i < S::FM; ++i) {
            const bool last = i == S::FM - 1;
            if (!last) {
#pragma unroll
                for (int p = 0; p < 3; ++p) a[(i + 1) & 1][p] = ra.one(s0 + p * PA, 0, lane, i + 1);
            } else {
                wait_vmem<(S::ST - 2) * LOADS>();
                lds_barrier();
                __builtin_amdgcn_sched_barrier(0);
            }
#pragma unroll
            for (int t = 0; t < 6; ++t) {
                if (last) {
                    constexpr int RD = 3 * S::FN + 3;
#pragma unroll
                    for (int q = t * RD / 6; q < (t + 1) * RD / 6; ++q) {
                        if (q < 3 * S::FN) nb[q / S::FN][q % S::FN] = rb.one(s1 + 3 * PA + q / S::FN * PB, 0, lane, q % S::FN);
                        else a[0][q - 3 * S::FN] = ra.one(s1 + (q - 3 * S::FN) * PA, 0, lane, 0);
                    }
#pragma unroll
                    for (int q = t * LOADS / 6; q < (t + 1) * LOADS / 6; ++q) load(q, l);
                }
#pragma unroll
                for (int j = 0; j < S::FN; ++j)
                    acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[i & 1][PI[t]], b[PJ[t]][j], acc[i][j], 0, 0, 0);
                if (last) __builtin_amdgcn_sched_barrier(0);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        next();
    };
    for (int item = first; item < sc.items; item = sc.with_steps(item + 1)) {
        const Work wk = sc.work(item);
        int tm, m0, n0;
        sc.place(wk.tile, tm, m0, n0);
#pragma unroll
        for (int i = 0; i < S::FM; ++i)
#pragma unroll
            for (int j = 0; j < S::FN; ++j) acc[i][j] = zero4();
        for (int k = wk.k0; k < wk.k1; ++k) {
            step(b0, b1);
            step(b1, b0);
        }
        epi.template run<S>(acc, m0, n0, wm, wn, lane, count, wk.seg, tm);
    }
    wait_vmem<0>();           // no load may land after the workgroup has ended
}

// ---------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------
inline size_t align256(size_t v) { return (v + 255) & ~size_t(255); }
inline bool al16(const void* p) { return ((uintptr_t)p & 15) == 0; }

template <class S, class EPI> void launch(const Gemm& g, const EPI& e, hipStream_t s) {
    const int64_t tiles = (int64_t)g.tm * g.tn;
    if constexpr (S::TERMS == 1 && S::BN < 128) {
        hipLaunchKernelGGL((k_ce_stream<S, EPI>), dim3((unsigned)(tiles * g.splits)), dim3(S::NT), 0, s, g, e);
    } else {
        const int64_t ncu = m2::cu_count();
        const unsigned nwg = (unsigned)(EPI::SEG ? g.splits : tiles < ncu ? tiles : ncu);
        if constexpr (S::TERMS == 1) hipLaunchKernelGGL((k_ce_tile<S, EPI>), dim3(nwg), dim3(S::NT), 0, s, g, e);
        else hipLaunchKernelGGL((k_ce_planes<S, EPI>), dim3(nwg), dim3(S::NT), 0, s, g, e);
    }
}
inline int tiles(int64_t n, int t) { return (int)((n + t - 1) / t); }

}  // namespace m2ce
