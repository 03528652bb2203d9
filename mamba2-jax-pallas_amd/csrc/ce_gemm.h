// Tiled bf16 matrix product D[m, n] = sum_k A[m, k] B[n, k] of the vocabulary's loss
// (linear_ce.hip), with the epilogue as a template parameter: the logits of a tile
// exist in its accumulators only.
//
// A tile is BM x BN, K in steps of 64 through a ring of ST LDS slots filled by
// direct global -> LDS loads; WM x WN wavefronts, 16x16x32 MFMAs.  Each operand
// is stored in global memory either with K contiguous ("row": A[m][k]) or with K strided
// ("col": A[k][m]):
//   row tile in LDS: [R][64], 128-byte rows whose 16-byte pieces are XOR-swizzled by
//     the row (piece ^ (row & 7)); fragments by ds_read_b128, eight consecutive
//     lanes on eight different pieces: no bank conflicts;
//   col tile in LDS: [64][R], rows of 2 R bytes whose 32-byte pieces (the 16
//     columns of one fragment) are XOR-swizzled by f(k) = k & 3 | (k >> 3 & 1) << 2;
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
    const void* zeros;   // 16 zero bytes
    const int* count;    // kept tokens (device)
    int nk;              // K steps of 64 (per plane product), 0: from count
    int tm, tn, splits;
    int tok_n;           // n is the token: tiles past the kept ones end at once
};

// ---------------------------------------------------------------------------
// global -> LDS
// ---------------------------------------------------------------------------
template <int R, bool TR, int NW> struct Loader {
    static constexpr int INSTR = R / 8;                          // 1 KB each
    static constexpr int J = INSTR >= NW ? INSTR / NW : 1;       // per wavefront
    static constexpr int BYTES = R * 128;
    uint32_t off[J];         // byte offset from the tile's base
    int m0;

    // m0: first row (column) of the tile
    M2_DEV void init(const Operand& o, int m0_, int w, int lane) {
        m0 = m0_;
#pragma unroll
        for (int j = 0; j < J; ++j) {
            const int in = (w * J + j) % INSTR;
            if constexpr (!TR) {
                int r = in * 8 + (lane >> 3);
                const int c = (lane & 7) ^ (lane >> 3);
                r = min(m0 + r, o.lim - 1) - m0;     // may be negative: tile past the end
                off[j] = (uint32_t)((int64_t)r * o.ld * 2 + c * 16);
            } else {
                constexpr int PR = R / 8;            // 16-byte pieces of a k row
                const int q = in * 64 + lane;
                const int k = q / PR, c = q % PR;
                const int f = (k & 3) | (((k >> 3) & 1) << 2);
                int m = ((((c >> 1) ^ f) << 1) | (c & 1)) * 8;
                m = min(m0 + m, o.lim - 8) - m0;
                off[j] = (uint32_t)((int64_t)k * o.ld * 2 + m * 2);
            }
        }
    }
    // the tile of K step kt, plane pl, into LDS at `lds`
    M2_DEV void issue(const Operand& o, const void* zeros, int kt, int pl, uint32_t lds, int w, int lane) const {
        if constexpr (!TR) {
            const bf16* base = o.p + pl * o.plane + (int64_t)m0 * o.ld + (int64_t)kt * 64;
            if (kt * 64 + 64 <= o.klim) {
#pragma unroll
                for (int j = 0; j < J; ++j)
                    dma16s(base, off[j], lds + ((w * J + j) % INSTR) * 1024);
            } else {
                const int c = (lane & 7) ^ (lane >> 3);
                const bool ok = kt * 64 + c * 8 < o.klim;
#pragma unroll
                for (int j = 0; j < J; ++j)
                    dma16(ok ? reinterpret_cast<const char*>(base) + off[j] : zeros,
                          lds + ((w * J + j) % INSTR) * 1024);
            }
        } else {
            const bf16* base = o.p + pl * o.plane + (int64_t)kt * 64 * o.ld + m0;
            if (kt * 64 + 64 <= o.klim) {
#pragma unroll
                for (int j = 0; j < J; ++j)
                    dma16s(base, off[j], lds + ((w * J + j) % INSTR) * 1024);
            } else {
                constexpr int PR = R / 8;
#pragma unroll
                for (int j = 0; j < J; ++j) {
                    const int k = (((w * J + j) % INSTR) * 64 + lane) / PR;
                    const int64_t over = max(kt * 64 + k - (o.klim - 1), 0);
                    dma16(reinterpret_cast<const char*>(base) + off[j] - over * o.ld * 2,
                          lds + ((w * J + j) % INSTR) * 1024);
                }
            }
        }
    }
};

// ---------------------------------------------------------------------------
// LDS -> fragments: F fragments of 16 rows from row r0 of the tile, K half kk
// ---------------------------------------------------------------------------
template <int R, bool TR, int F> struct Reader {
    int x;
    M2_DEV void init(int r0, int lane) {
        if constexpr (!TR) {
            x = (r0 + (lane & 15)) * 128;
        } else {
            const int g = lane >> 4, r = (lane & 15) >> 2;
            const int f = r | ((g & 1) << 2);
            x = (8 * g + r) * (2 * R) + (lane & 3) * 8 + (((r0 >> 4) ^ f) << 5);
        }
    }
    M2_DEV void read(const char* s, int kk, int lane, bf16x8 (&o)[F]) const {
        if constexpr (!TR) {
            const int sl = ((((lane >> 4) + 4 * kk) ^ (lane & 7)) << 4);
            const char* p = s + x + sl;
#pragma unroll
            for (int i = 0; i < F; ++i) o[i] = *reinterpret_cast<const bf16x8*>(p + i * 2048);
        } else {
#pragma unroll
            for (int i = 0; i < F; ++i) {
                const char* p = s + (x ^ (i << 5)) + kk * 32 * 2 * R;
                const bf16x4 lo = ds_read_tr(p), hi = ds_read_tr(p + 4 * 2 * R);
                o[i] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
            }
        }
    }
};

template <int BM_, int BN_, int WM_, int WN_, int ST_, bool ATR_, bool BTR_, int TERMS_> struct Shape {
    static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, ST = ST_, TERMS = TERMS_;
    static constexpr bool ATR = ATR_, BTR = BTR_;
    static constexpr int NW = WM * WN, NT = NW * 64;
    static constexpr int FM = BM / WM / 16, FN = BN / WN / 16;
    typedef Loader<BM, ATR, NW> LA;
    typedef Loader<BN, BTR, NW> LB;
    static constexpr int SLOT = LA::BYTES + LB::BYTES;
    static constexpr int LDS = SLOT * ST;
    static constexpr int LOADS = LA::J + LB::J;
};

template <class S, class EPI>
__global__ void __launch_bounds__(S::NT, S::NT >= 512 || 2 * S::LDS <= 160 * 1024 ? 2 : 1) k_ce_gemm(Gemm g, EPI epi) {
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

    const int count = *g.count;
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
        // products in the order (0,2) (2,0) (1,1) (0,1) (1,0) (0,0)
        const int pa = S::TERMS == 1 ? 0 : iterm == 1 ? 2 : (iterm == 2 || iterm == 4) ? 1 : 0;
        const int pb = S::TERMS == 1 ? 0 : iterm == 0 ? 2 : (iterm == 2 || iterm == 3) ? 1 : 0;
        const uint32_t l = lds0 + islot * S::SLOT;
        la.issue(g.a, g.zeros, ikt, pa, l, w, lane);
        lb.issue(g.b, g.zeros, ikt, pb, l + S::LA::BYTES, w, lane);
        if (++ikt == k1) { ikt = k0; ++iterm; }
        if (++islot == S::ST) islot = 0;
    };

    Reader<S::BM, S::ATR, S::FM> ra;
    Reader<S::BN, S::BTR, S::FN> rb;
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
    lds_barrier();
    epi.template run<S>(acc, smem, m0, n0, wm, wn, lane, count, split, tm);
}

}  // namespace m2ce
