// Tiled bf16 matrix product D[m, n] = sum_k A[m, k] B[n, k] of the vocabulary's loss
// (linear_ce.hip), with the epilogue as a template parameter: the logits of a tile
// exist in its accumulators only.
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
// the last bits) and K runs six times: the products p_i q_j with i + j <= 2, the small
// ones first; what is left out is 2^-24 of the product.
#pragma once

#include "m2_internal.h"

namespace m2ce {

struct Operand {
    const bf16* p;
    int64_t ld;          // elements between rows (row: of m; col: of k)
    int64_t plane;       // elements between the planes of a float32 operand
    int lim;             // valid m (row: rows past it read the last one; col: columns, a multiple of 8)
    int klim;            // valid k (row: pieces past it read zeros; col: rows past it read the last one)
};

struct Gemm {
    Operand a, b;
    const int* count;    // tokens that take part (device), or NULL: n
    int n;
    int nk;              // K steps of 64 (per plane product), 0: from count
    int tm, tn;
    int tok_n;           // n is the token: tiles past the kept ones are left out
    int splits;          // k_ce_stream: K in so many parts
    int seg_nk;          // k_ce_tile with EPI::SEG: the K steps that deal() goes by
};

// k_ce_tile with EPI::SEG: as many whole tiles as fill the workgroups, and the rest of the tiles
// cut in s parts of K each, so that few workgroups are idle in the end.  Parts of the same
// K lie beside each other (they share panels).  Segment numbers: the tile of a whole
// one; full + part * rest + (tile - full).
struct Deal {
    int full, rest, s;
    int64_t cost;            // 5 ns
};
// bn: the tile's n, 256 or 128
__host__ __device__ inline Deal deal(int tiles, int nk, int nwg, int bn) {
    // a step takes about 1.4 us (0.85 us), writing and reading a segment of 256 KB the chip
    // 0.11 us (whole numbers: the host sizes the workspace by the same)
    const int step = bn == 256 ? 280 : 170, seg = bn == 256 ? 22 : 11;
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

template <int R, bool TR, int NW, int BK> struct Loader {
    static constexpr int BYTES = R * BK * 2;
    static constexpr int INSTR = BYTES / 1024;                   // 1 KB each
    static constexpr int J = INSTR >= NW ? INSTR / NW : 1;       // per wavefront
    static constexpr int PP = BK / 8;                            // pieces of a row
    static constexpr int PR = R / 8;                             // pieces of a k row
    uint32_t off[J];         // byte offset from the tile's base
    int m0;

    // m0: first row (column) of the tile
    M2_DEV void init(const Operand& o, int m0_, int w, int lane) {
        m0 = m0_;
#pragma unroll
        for (int j = 0; j < J; ++j) {
            const int in = (w * J + j) % INSTR;
            if constexpr (!TR) {
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

template <int BM_, int BN_, int WM_, int WN_, int ST_, int BK_, bool ATR_, bool BTR_, int TERMS_> struct Shape {
    static constexpr int BK = BK_, BM = BM_, BN = BN_, WM = WM_, WN = WN_, ST = ST_, TERMS = TERMS_;
    static constexpr bool ATR = ATR_, BTR = BTR_;
    static constexpr int NW = WM * WN, NT = NW * 64;
    static constexpr int FM = BM / WM / 16, FN = BN / WN / 16;
    typedef Loader<BM, ATR, NW, BK> LA;
    typedef Loader<BN, BTR, NW, BK> LB;
    static constexpr int SLOT = LA::BYTES + LB::BYTES;
    static constexpr int LDS = SLOT * ST;
    static constexpr int LOADS = LA::J + LB::J;
};

// The order of the products of the planes: (0,2) (2,0) (1,1) (0,1) (1,0) (0,0)
template <int TERMS> M2_DEV int plane_a(int t) { return TERMS == 1 ? 0 : t == 1 ? 2 : (t == 2 || t == 4) ? 1 : 0; }
template <int TERMS> M2_DEV int plane_b(int t) { return TERMS == 1 ? 0 : t == 0 ? 2 : (t == 2 || t == 3) ? 1 : 0; }

// Few tokens: the operand of the vocabulary streams from HBM through a deep ring
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
    const int total = (k1 - k0) * S::TERMS;

    typename S::LA la;
    typename S::LB lb;
    la.init(g.a, m0, w, lane);
    lb.init(g.b, n0, w, lane);
    const uint32_t lds0 = lds_addr(smem);
    int ikt = k0, iterm = 0, islot = 0;
    auto issue = [&]() {
        const uint32_t l = lds0 + islot * S::SLOT;
        la.issue(g.a, ikt, plane_a<S::TERMS>(iterm), l, w, lane);
        lb.issue(g.b, ikt, plane_b<S::TERMS>(iterm), l + S::LA::BYTES, w, lane);
        if (++ikt == k1) { ikt = k0; ++iterm; }
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
    epi.template run<S>(acc, smem, m0, n0, wm, wn, lane, count, split, tm);
}

// Many tokens: persistent workgroups (whole tiles, or with EPI::SEG segments of them), each XCD with a contiguous range of the tiles
// (neighbours share panels in its L2).  K in steps of 64, A through a ring of three slots, B of
// two (all 160 KB for 256 x 256); the fragments of a half step (32 of K) are read while the half
// step before multiplies, so the matrix units wait for neither LDS nor the
// other wavefronts but once a step:
//   half 0 of step i: multiply F0, read F1 (half 1 of step i), load A of step i + 2
//   wait until step i + 1 has landed; barrier: everybody has read step i
//   half 1 of step i: multiply F1, read F0 (half 0 of step i + 1), load B of step i + 2
// so that both halves carry as many loads (all of them in one half leave too few cycles for
// the 64 bytes a cycle that a CU takes in).  The loads run on into the next tile, whose first
// steps arrive during the epilogue.
struct Work {                 // of a workgroup: its item i, a tile and its K steps
    int i, tile, k0, k1, seg;
};
template <class LD> struct Cursor {      // the step of an operand that is loaded next
    LD ld;
    Work at;
    int k, term;
};

template <class S, class EPI>
__global__ void __launch_bounds__(S::NT, S::NT / 256) k_ce_tile(Gemm g, EPI epi) {
    static_assert(S::BK == 64, "");
    constexpr int B_AT = 3 * S::LA::BYTES;
    __shared__ __align__(1024) char smem[B_AT + 2 * S::LB::BYTES];
    const int lane = threadIdx.x & 63, w = wave_id();
    const int wm = w / S::WN, wn = w % S::WN;
    const int count = g.count ? *g.count : g.n;
    const int tn_all = g.tok_n ? min(g.tn, (((count + 63) & ~63) + S::BN - 1) / S::BN) : g.tn;
    const int tiles = g.tm * tn_all;
    const int nk = g.nk ? g.nk : (count + 63) >> 6;
    // this workgroup's place: those of an XCD beside each other
    const int xcd = blockIdx.x & 7, local = blockIdx.x >> 3;
    const int nwg = gridDim.x, lw = (nwg - xcd + 7) >> 3;
    const int before = xcd * (nwg >> 3) + min(xcd, nwg & 7);
    // whole tiles one workgroup after the other; each XCD a contiguous range, which its
    // share of the workgroups gives
    Deal dl{0, tiles, 1, 0};
    if constexpr (EPI::SEG) dl = deal(tiles, g.seg_nk, nwg, S::BN);
    const int f0 = dl.full / nwg * before + local, rounds = dl.full / nwg;
    const int64_t cut = (int64_t)dl.rest * dl.s;
    const int r0 = (int)(cut * before / nwg) + local, r1 = (int)(cut * (before + lw) / nwg);
    auto work = [&](int i) {
        if (EPI::SEG && i < rounds) return Work{i, f0 + i * lw, 0, nk, f0 + i * lw};
        const int id = r0 + (i - rounds) * lw;
        Work x{i, 0, 0, 0, dl.full + id};
        if (id >= r1) return x;
        const int part = EPI::SEG ? id / dl.rest : 0;
        x.tile = dl.full + id - part * dl.rest;
        x.k0 = EPI::SEG ? (int)((int64_t)nk * part / dl.s) : 0;
        x.k1 = EPI::SEG ? (int)((int64_t)nk * (part + 1) / dl.s) : nk;
        return x;
    };
    const int items = rounds + (r1 > r0 ? (r1 - r0 + lw - 1) / lw : 0);
    if (items == 0) return;
    auto place = [&](int id, int& tm, int& m0, int& n0) {
        // 8 tiles of m beside each other, then the next n
        const int grp = id / (8 * tn_all), gm = min(8, g.tm - grp * 8), in = id - grp * 8 * tn_all;
        tm = grp * 8 + in % gm;
        m0 = tm * S::BM;
        n0 = in / gm * S::BN;
    };
    Cursor<typename S::LA> ca;
    Cursor<typename S::LB> cb;
    auto start = [&](auto& c, const Operand& o, bool is_a, const Work& x) {
        int tm, m0, n0;
        place(x.tile, tm, m0, n0);
        c.ld.init(o, is_a ? m0 : n0, w, lane);
        c.at = x;
        c.k = x.k0;
        c.term = 0;
    };
    // past the last step the last tile's last step is loaded again (nobody reads it)
    auto next = [&](auto& c, const Operand& o, bool is_a) {
        if (++c.k < c.at.k1) return;
        c.k = c.at.k0;
        if (++c.term < S::TERMS) return;
        for (int i = c.at.i + 1; i < items; ++i) {
            const Work x = work(i);
            if (x.k0 < x.k1) return start(c, o, is_a, x);
        }
        c.k = c.at.k1 - 1;
        c.term = S::TERMS - 1;
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
    int first = 0;                // the first item that has steps (a short piece's parts may not)
    while (first < items && nk > 0 && work(first).k0 >= work(first).k1) ++first;
    if (first == items) return;
    if (nk > 0) {
        start(ca, g.a, true, work(first));
        start(cb, g.b, false, work(first));
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            ca.ld.issue(g.a, ca.k, plane_a<S::TERMS>(ca.term), lds0 + i * S::LA::BYTES, w, lane);
            cb.ld.issue(g.b, cb.k, plane_b<S::TERMS>(cb.term), lds0 + B_AT + i * S::LB::BYTES, w, lane);
            next(ca, g.a, true);
            next(cb, g.b, false);
        }
        wait_vmem<S::LOADS>();
        lds_barrier();
        ra.read(smem, 0, lane, a0);
        rb.read(smem + B_AT, 0, lane, b0);
    }
    constexpr int RD = S::FM + S::FN;
    for (int item = first; item < items; ++item) {
        const Work wk = work(item);
        if (EPI::SEG && wk.k0 >= wk.k1) continue;
        int tm, m0, n0;
        place(wk.tile, tm, m0, n0);
#pragma unroll
        for (int i = 0; i < S::FM; ++i)
#pragma unroll
            for (int j = 0; j < S::FN; ++j) acc[i][j] = zero4();
        const int steps = S::TERMS * (wk.k1 - wk.k0);
        for (int st = 0; st < steps; ++st) {
            {
                const char* pa = smem + sa;
                const char* pb = smem + B_AT + sb;
                const uint32_t l = lds0 + after(after(sa));
                const bf16* from = ca.ld.base(g.a, ca.k, plane_a<S::TERMS>(ca.term));
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
                const bf16* from = cb.ld.base(g.b, cb.k, plane_b<S::TERMS>(cb.term));
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
        epi.template run<S>(acc, nullptr, m0, n0, wm, wn, lane, count, wk.seg, tm);
    }
    wait_vmem<0>();           // no load may land after the workgroup has ended
}

}  // namespace m2ce
