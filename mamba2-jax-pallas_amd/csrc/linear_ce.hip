// linear_cross_entropy and its gradient: softmax cross entropy of a linear head
// over a large vocabulary in pieces, without the logits ever being stored.
//
//   z[n, v] = x[n] . w[v];  loss[n] = log sum_v exp(z[n, v]) - z[n, t[n]]
//   G[n, v] = g[n] (exp(z[n, v] - lse[n]) - [v == t[n]]);  dx = G w;  dw = G^T x
//
// Forward: the product runs in tiles (ce_gemm.h); each leaves, per token and 128 logits, the
// maximum m of the logits but the target's and the sum s of their exponentials
// below it (8 bytes), and the target's logit z_t where it holds it.  A second kernel
// joins them: loss = log(1 + s exp(m - z_t)), which keeps its accuracy down to
// losses far below the step of the logits.
// Backward: a piece of the vocabulary at a time, the same product again gives G in its
// epilogue (rounded to bf16 once, as the results are; what that takes from the target's is
// given back in float32, lost_of; float32 operands keep three bf16 planes of it), then dw of the
// piece and the piece's part of dx, which float32 partial sums collect over pieces.  At
// the target G is g expm1(-loss), not a difference of near-equal numbers.
//
// Tokens that are left out (ignore_index) are dropped at the start: the kept rows of x
// are packed (zero-padded to whole K steps), so they cost nothing afterwards
// and what stands in a row left out (a NaN, say) touches nothing.  The number of
// kept tokens stays on the device, where the tiles are dealt out by it.  Only
// the scoring of up to 64 bf16 tokens reads x in place: every token is a column of its
// own there, and the join passes over those left out.
//
// Bound by the matrix units for more than a few hundred tokens (2 n V D operations
// forward, 6 n V D backward with the logits computed again), by reading the
// weights for few.  bf16, 50288 x 2560: 16 tokens scored in 56 us (4.6 TB/s of weights), 4096
// in 0.80 to 0.83 ms (1.3 PFLOP/s), loss and gradients of 8192 in 6.8 ms (1.24 PFLOP/s with the
// logits computed twice).  Keeping the logits would save a quarter of the
// latter and hold 1.6 GB instead of 512 MB of G.
#include "ce_gemm.h"

namespace {

using namespace m2ce;

constexpr float LOG2E = 1.4426950408889634f;

struct Tokens {              // of the kept tokens: in the workspace, or saved for the gradient
    int* idx;                // [np] row of x of each
    int* inv;                // [n] kept index of each row, -1: left out
    int* tgt;                // [np] target, -1: outside the vocabulary
    float* lse;              // [np]
    float* em1;              // [np] expm1(-loss): G at the target
    int* count;              // [2] their number; workgroups of k_ce_join that are done
    float* zt;               // [np] the target's logit (forward)
    float* lost;             // [np] what bf16 takes from G at the target (backward, EpiG)
    int* first;              // [vocab] the first kept token with this target, or NONE
    unsigned long long* runs;    // [vocab][run_words] which 64s of kept tokens have this target
    int run_words;
};
constexpr int NONE = 0x7fffffff;

M2_DEV int64_t load_target(const void* targets, int t64, int64_t i) {
    return t64 ? reinterpret_cast<const int64_t*>(targets)[i] : (int64_t) reinterpret_cast<const int32_t*>(targets)[i];
}

// ---------------------------------------------------------------------------
// which rows are kept, in order
// ---------------------------------------------------------------------------
__global__ void __launch_bounds__(1024) k_ce_compact(const void* targets, int64_t n, int64_t ignore, int t64,
                                                     Tokens tk) {
    __shared__ int wsum[16];
    const int t = threadIdx.x, lane = t & 63, w = wave_id();
    int base = 0;
    constexpr int E = 8;
    for (int64_t i0 = 0; i0 < n; i0 += 1024 * E) {
        bool keep[E];
        int mine = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int64_t i = i0 + (int64_t)t * E + e;
            keep[e] = false;
            if (i < n) {
                keep[e] = load_target(targets, t64, i) != ignore;
            }
            mine += keep[e];
        }
        int s = mine;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int u = __shfl_up(s, o);
            if (lane >= o) s += u;
        }
        if (lane == 63) wsum[w] = s;
        __syncthreads();
        int at = base + s - mine, all = 0;
#pragma unroll
        for (int q = 0; q < 16; ++q) {
            at += q < w ? wsum[q] : 0;
            all += wsum[q];
        }
        base += all;
        __syncthreads();
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int64_t i = i0 + (int64_t)t * E + e;
            if (i >= n) break;
            tk.inv[i] = keep[e] ? at : -1;
            if (keep[e]) tk.idx[at++] = (int)i;
        }
    }
    if (t < 2) tk.count[t] = t == 0 ? base : 0;
}

struct PackArgs {
    const void* src;
    bf16* dst;
    int64_t rows, dim, ld, dp, plane;
    // of the tokens
    const void* targets;
    const float* lse;        // given to a gradient that finds nothing saved
    const float* loss;
    int64_t vocab, n, ignore;
    int t64;
    int row_blocks;          // further workgroups clear tk.first and tk.runs
};
constexpr int64_t PACK_FINDS = 1024;     // up to so many tokens the packing finds the kept ones itself
constexpr int CLEAR = 2048;              // rows of the vocabulary that one workgroup clears them for

// Rows of src as bf16 (planes) with rows of dp elements, zeros behind dim: the weights
// where they cannot be read in place, or the kept rows of x (TOK), with zero rows up to
// the next whole K step.  Up to PACK_FINDS tokens a wavefront for each row counts
// the kept ones before it, and 64 more write the zero rows; beyond, k_ce_compact has found them.
template <typename T, bool TOK>
__global__ void __launch_bounds__(256) k_ce_pack(PackArgs a, Tokens tk) {
    int64_t r = (int64_t)blockIdx.x * 4 + wave_id();
    const int lane = threadIdx.x & 63;
    int64_t from = r;
    if constexpr (TOK) {
        if ((int)blockIdx.x >= a.row_blocks) {
            const int64_t v0 = (int64_t)(blockIdx.x - a.row_blocks) * CLEAR;
            const int64_t v1 = min(v0 + CLEAR, a.vocab);
            for (int64_t v = v0 + threadIdx.x; v < v1; v += 256) tk.first[v] = NONE;
            for (int64_t i = v0 * tk.run_words + threadIdx.x; i < v1 * tk.run_words; i += 256) tk.runs[i] = 0;
            return;
        }
        if (a.n <= PACK_FINDS) {
            if (r >= a.n + 64) return;
            int before = 0;
            const int64_t end = min(r, a.n);
#pragma unroll 4
            for (int64_t i = 0; i < end; i += 64)
                before += __popcll(__ballot(i + lane < end && load_target(a.targets, a.t64, i + lane) != a.ignore));
            if (r >= a.n) {                   // before: all of them
                if (r == a.n && lane < 2) tk.count[lane] = lane == 0 ? before : 0;
                r += before - a.n;
                if (r >= ((before + 63) & ~63)) return;
                from = -1;
            } else {
                const bool keep = load_target(a.targets, a.t64, r) != a.ignore;
                if (lane == 0) {
                    tk.inv[r] = keep ? before : -1;
                    if (keep) tk.idx[before] = (int)r;
                }
                if (!keep) return;
                r = before;
            }
        } else {
            const int count = *tk.count;
            if (r >= ((count + 63) & ~63)) return;
            from = r < count ? tk.idx[r] : -1;
        }
        if (lane == 0) {
            int tg = -1;
            if (from >= 0) {
                const int64_t v = load_target(a.targets, a.t64, from);
                tg = v >= 0 && v < a.vocab ? (int)v : -1;
                if (a.loss) {
                    tk.lse[r] = a.lse[from];
                    tk.em1[r] = expm1f(-a.loss[from]);
                }
            }
            tk.tgt[r] = tg;
            if (tk.zt) tk.zt[r] = __builtin_nanf("");
        }
    } else {
        if (r >= a.rows) return;
    }
    const T* src = static_cast<const T*>(a.src) + (from < 0 ? 0 : from) * a.ld;
    bf16* dst = a.dst + r * a.dp;
    for (int64_t c = lane * 8; c < a.dp; c += 512) {
        float v[8];
        if (from >= 0) {
            load8(src, c, a.dim, v);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = 0.f;
        }
        store8<sizeof(T) == 4>(dst + c, a.plane, v);
    }
}

// ---------------------------------------------------------------------------
// epilogues.  A lane holds, of each 16x16 block, one n (lane & 15) and 4 consecutive
// m (4 (lane >> 4) ..).
// ---------------------------------------------------------------------------
// a running maximum and the sum of exp(z - maximum)
struct LogSum {
    float mx = -__builtin_inff(), s = 0.f;
    M2_DEV void add(float2 u) {
        const float m = fmaxf(mx, u.x), b = m == -__builtin_inff() ? 0.f : m;
        s = s * __builtin_amdgcn_exp2f((mx - b) * LOG2E) + u.y * __builtin_amdgcn_exp2f((u.x - b) * LOG2E);
        mx = m;
    }
    // (loss, lse): exp(loss) = 1 + the others' sum over exp(z_t).  lse from the larger of maximum
    // and z_t on: z_t + loss would keep z_t's roundings where it lies far below the others.  A
    // target's logit of -inf has loss inf and the others' lse; a logit of +inf, the target's or
    // not (s is NaN then), no softmax: an overflow is not a perfect prediction.
    M2_DEV float2 with_target(float zt) const {
        if (zt == __builtin_inff()) return make_float2(__builtin_nanf(""), __builtin_nanf(""));
        const float d = mx - zt, e = __builtin_amdgcn_exp2f(-fabsf(d) * LOG2E);
        if (d <= 0.f) {
            const float l = log1pf(s * e);
            return make_float2(l, zt + l);
        }
        const float l = logf(s + e);
        return make_float2(d + l, mx + l);
    }
};
// m: vocabulary, n: token -> per token (max, sum of exp(z - max)) without the target: of a tile
// (k_ce_stream), or of the BM / WM rows of the vocabulary that a row of wavefronts holds
// (the others, whose LDS is full)
struct EpiLse {
    static constexpr bool SEG = false;
    const int* tgt;          // of the kept tokens, or NULL: the caller's targets
    const void* targets;
    int64_t ignore;
    float* zt;
    float2* part;            // [parts][np]
    int64_t np;
    int vocab, t64;

    M2_DEV int target(int n) const {
        if (tgt) return tgt[n];
        const int64_t v = load_target(targets, t64, n);
        return v >= 0 && v < vocab && v != ignore ? (int)v : -1;
    }

    template <class S>
    M2_DEV void run(f32x4 (&acc)[S::FM][S::FN], int m0, int n0, int wm, int wn, int lane, int count, int, int tm) const {
        // (LDS of their own: the operands' ring may still be read by other wavefronts)
        constexpr bool JOIN = S::BN < 128 && S::TERMS == 1;
        __shared__ float2 sums[JOIN ? S::WM * S::BN : 1];
        const int v0 = m0 + wm * S::FM * 16 + 4 * (lane >> 4);
        const float ninf = -__builtin_inff();
        if (m0 + S::BM > vocab) {
#pragma unroll
            for (int i = 0; i < S::FM; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (v0 + 16 * i + r >= vocab)
#pragma unroll
                        for (int j = 0; j < S::FN; ++j) acc[i][j][r] = ninf;
        }
#pragma unroll
        for (int j = 0; j < S::FN; ++j) {
            const int n = n0 + (wn * S::FN + j) * 16 + (lane & 15);
            // the target's place among this lane's values, if it is there (few wavefronts
            // have one: the others pay for one comparison)
            const int d = n < count ? target(n) - v0 : -1;
            if (__ballot(d >= 0 && d < 16 * S::FM && (d & 12) == 0)) {
#pragma unroll
                for (int i = 0; i < S::FM; ++i)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (d == 16 * i + r) {
                            zt[n] = acc[i][j][r];
                            acc[i][j][r] = ninf;
                        }
            }
            float mx = ninf;
#pragma unroll
            for (int i = 0; i < S::FM; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r) mx = fmaxf(mx, acc[i][j][r]);
            mx = fmaxf(mx, __shfl_xor(mx, 16));
            mx = fmaxf(mx, __shfl_xor(mx, 32));
            const float b = mx == ninf ? 0.f : mx * -LOG2E;
            float s = 0.f;
#pragma unroll
            for (int i = 0; i < S::FM; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r) s += __builtin_amdgcn_exp2f(fmaf(acc[i][j][r], LOG2E, b));
            s += __shfl_xor(s, 16);
            s += __shfl_xor(s, 32);
            if constexpr (JOIN) {
                if (lane < 16) sums[wm * S::BN + n - n0] = make_float2(mx, s);
            } else {
                if (lane < 16 && n < count) part[((int64_t)tm * S::WM + wm) * np + n] = make_float2(mx, s);
            }
        }
        if constexpr (JOIN) {
            __syncthreads();
            const int t = threadIdx.x;
            if (t < S::BN && n0 + t < count) {
                LogSum o = {};
#pragma unroll
                for (int q = 0; q < S::WM; ++q) o.add(sums[q * S::BN + t]);
                part[(int64_t)tm * np + n0 + t] = make_float2(o.mx, o.s);
            }
        }
    }
};

// The upstream gradient of the kept tokens' losses.
struct Up {
    const float* g;
    int64_t stride;          // 0: one value
    int mean;
    // of a token, in G; of all, where they have one value: dx and dw are multiplied by it behind
    // their products and G is softmax - onehot alone, whose bf16 is nearly exact at a
    // target of small probability.
    M2_DEV float of(const Tokens& tk, int n, int count) const {
        return stride ? g[tk.idx[n] * stride] * (mean ? 1.f / (float)count : 1.f) : 1.f;
    }
    M2_DEV float all(int count) const {
        if (stride || count == 0) return 1.f;
        // (a scalar load: a vector load would wait for the loads of the next tile)
        return *(const __attribute__((address_space(4))) float*)(uintptr_t)g * (mean ? 1.f / (float)count : 1.f);
    }
};
// What bf16 takes from G at the target, where most of a row's weight is, is up to 2^-8 of it
// and the same for every column.  dx and dw get it back in float32: dx is 1.66e-3 off, as one
// rounding alone, where it was 2.0 to 3.7e-3, dw of 300 tokens over 32003 x 1001 1.44e-3 (1.71)
M2_DEV float lost_of(const Tokens& tk, int n) { return tk.tgt[n] >= 0 ? tk.lost[n] : 0.f; }
M2_DEV float lost_at(float gt) {
    const float r = gt - (float)(bf16)gt;
    return fabsf(r) < __builtin_inff() ? r : 0.f;         // (an infinity or NaN is G itself)
}
M2_DEV f32x4 load4(const bf16* p) {          // 8-byte aligned
    typedef uint32_t u2 __attribute__((ext_vector_type(2)));
    const u2 v = *reinterpret_cast<const u2*>(p);
    return f32x4{bf16_lo(v[0]), bf16_hi(v[0]), bf16_lo(v[1]), bf16_hi(v[1])};
}

// m: vocabulary, n: token -> G, bf16 (three planes for float32 operands), zero past the
// vocabulary and past the kept tokens
struct EpiG {
    static constexpr bool SEG = false;
    Tokens tk;
    Up up;
    bf16* G;
    int64_t ldg, plane;
    int v_first, vocab;      // of the piece; of all

    template <class S>
    M2_DEV void run(f32x4 (&acc)[S::FM][S::FN], int m0, int n0, int wm, int wn, int lane, int count, int, int) const {
        static_assert(S::FM % 2 == 0, "");
        const int mw = m0 + wm * S::FM * 16, mv = mw + 4 * (lane >> 4);
        const int lim = (count + 63) & ~63;
        // of the tokens, before the first store (a load behind it would wait for it)
        int t[S::FN];
        float ls[S::FN], g[S::FN], gt[S::FN];
#pragma unroll
        for (int j = 0; j < S::FN; ++j) {
            const int n = n0 + (wn * S::FN + j) * 16 + (lane & 15);
            const bool on = n < count;
            t[j] = on ? tk.tgt[n] : 0;
            ls[j] = on ? tk.lse[n] * -LOG2E : 0.f;
            g[j] = on ? up.of(tk, n, count) : 0.f;
            gt[j] = on ? g[j] * tk.em1[n] : 0.f;
            if (t[j] < 0) g[j] = __builtin_nanf("");       // a target outside the vocabulary
            t[j] -= v_first;
        }
        // rows past the vocabulary: zeros, whatever x holds
        const bool edge = v_first + m0 + S::BM > vocab;
#pragma unroll
        for (int j = 0; j < S::FN; ++j) {
            const int n = n0 + (wn * S::FN + j) * 16 + (lane & 15);
            if (n >= lim) continue;
            const bool on = n < count;
            const int d = on ? t[j] - mv : -1;
            const bool mine = d >= 0 && d < 16 * S::FM && (d & 12) == 0, here = __ballot(mine);
            if (S::TERMS == 1 && mine)
                tk.lost[n] = lost_at(gt[j]);
            bf16* to = G + (int64_t)n * ldg + mw + pair_m(lane);
#pragma unroll
            for (int i = 0; i < S::FM; i += 2) {
                float o[2][4];
#pragma unroll
                for (int e = 0; e < 2; ++e)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float p = g[j] * __builtin_amdgcn_exp2f(fmaf(acc[i + e][j][r], LOG2E, ls[j]));
                        o[e][r] = on ? p : 0.f;
                    }
                if (here)
#pragma unroll
                    for (int e = 0; e < 2; ++e)
#pragma unroll
                        for (int r = 0; r < 4; ++r) o[e][r] = d == 16 * (i + e) + r ? gt[j] : o[e][r];
                if (edge)
#pragma unroll
                    for (int e = 0; e < 2; ++e)
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            if (v_first + mv + 16 * (i + e) + r >= vocab) o[e][r] = 0.f;
                if constexpr (S::TERMS == 1) {
                    store_pair(to + 16 * i, o[0], o[1]);
                } else {
                    float h[2][4], md[2][4], l[2][4];
#pragma unroll
                    for (int e = 0; e < 2; ++e)
#pragma unroll
                        for (int r = 0; r < 4; ++r) split3(o[e][r], h[e][r], md[e][r], l[e][r]);
                    store_pair(to + 16 * i, h[0], h[1]);
                    store_pair(to + 16 * i + plane, md[0], md[1]);
                    store_pair(to + 16 * i + 2 * plane, l[0], l[1]);
                }
            }
        }
    }
};

// m: dim, n: token -> float32 partial sums of dx, added to over the pieces of the vocabulary.
// Few tokens (k_ce_stream): one array per split of K.
struct EpiDxSplit {
    float* part;             // [splits][np][dp]
    int64_t np, dp;
    int add;

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
            for (int i = 0; i < S::FM; ++i) {
                const int m = mv + 16 * i;
                if (m >= dp) continue;
                f32x4 v = acc[i][j];
                if (add) v += *reinterpret_cast<const f32x4*>(d + m);
                *reinterpret_cast<f32x4*>(d + m) = v;
            }
        }
    }
};
// Many (k_ce_tile): a segment as the lanes hold it, [wavefront][i][j][lane] of 4 values.
struct EpiDxSeg {
    static constexpr bool SEG = true;
    float* part;             // [segments][BM * BN]
    int add;

    template <class S>
    M2_DEV void run(f32x4 (&acc)[S::FM][S::FN], int, int, int wm, int wn, int lane, int, int seg, int) const {
        f32x4* d = reinterpret_cast<f32x4*>(part) +
                   ((int64_t)seg * S::NW + wm * S::WN + wn) * S::FM * S::FN * 64 + lane;
        if (add) {
#pragma unroll
            for (int i = 0; i < S::FM; ++i)
#pragma unroll
                for (int j = 0; j < S::FN; ++j) acc[i][j] += d[(i * S::FN + j) * 64];
        }
#pragma unroll
        for (int i = 0; i < S::FM; ++i)
#pragma unroll
            for (int j = 0; j < S::FN; ++j) d[(i * S::FN + j) * 64] = acc[i][j];
    }
};

// m: dim, n: vocabulary -> rows of dw, with what G lost at the targets (bf16: back, k_ce_back)
template <typename T> struct EpiDw {
    static constexpr bool SEG = false;
    T* dw;
    int64_t dim, dp;
    const float* back;       // [np][dp], the rows of the first token of each target
    const int* first;        // of the piece
    Up up;
    int rows;                // of the piece

    template <class S>
    M2_DEV void run(f32x4 (&acc)[S::FM][S::FN], int m0, int n0, int wm, int wn, int lane, int count, int, int) const {
        const int mw = m0 + wm * S::FM * 16, nw = n0 + wn * S::FN * 16;
        const float all = up.all(count);
        if constexpr (sizeof(T) == 2) {
            int k[S::FN];
#pragma unroll
            for (int j = 0; j < S::FN; ++j) {
                const int n = nw + 16 * j + (lane & 15);
                k[j] = n < rows ? first[n] : NONE;
            }
#pragma unroll
            for (int j = 0; j < S::FN; ++j) {
                if (k[j] == NONE) continue;
                const int m = mw + 4 * (lane >> 4);
                const float* b = back + k[j] * dp + m;
#pragma unroll
                for (int i = 0; i < S::FM; ++i)
                    if (m + 16 * i < dp) acc[i][j] += *reinterpret_cast<const f32x4*>(b + 16 * i);
            }
        }
#pragma unroll
        for (int j = 0; j < S::FN; ++j) {
            const int n = nw + 16 * j + (lane & 15);
            if (n >= rows) continue;
#pragma unroll
            for (int i = 0; i < S::FM; i += 2)
                store_row(dw + (int64_t)n * dim, mw + 16 * i, dim, lane, all * acc[i][j], all * acc[i + 1][j]);
        }
    }
};

// ---------------------------------------------------------------------------
// what G lost at the targets, for dw
// ---------------------------------------------------------------------------
struct BackArgs {
    const bf16* x;           // packed, rows of dp
    float* back;             // out [np][dp]
    int64_t dp;
    int v_first, rows;       // of the piece
};
// Of each target of the piece: lost[n] x[n] summed over its tokens among 64, in their order, into the row
// of the first of them: a wavefront for a token and 512 columns.  (One product more for
// each token in dw's epilogue, as matrix instructions, costs the main loop its registers and
// leaves a frequent target to one wavefront.)  1230 kept of 2048 tokens x 768 over 50288: 7 us here, 7 in
// k_ce_back_join, of 484 with the gradient.
__global__ void __launch_bounds__(256) k_ce_back(BackArgs a, Tokens tk) {
    const int n = blockIdx.x * 4 + wave_id(), lane = threadIdx.x & 63;
    if (n >= *tk.count) return;
    const int t = tk.tgt[n] - a.v_first, n0 = n & ~63;
    if (t < 0 || t >= a.rows) return;
    // (past the kept tokens stands -1 up to the next multiple of 64)
    uint64_t same = __ballot(tk.tgt[n0 + lane] - a.v_first == t);
    const float lost = tk.lost[n0 + lane];
    if (n0 + __ffsll((unsigned long long)same) - 1 != n) return;
    if (blockIdx.y == 0 && lane == 0) {
        const int64_t v = a.v_first + t;
        atomicMin(tk.first + v, n);
        atomicOr(tk.runs + v * tk.run_words + (n >> 12), 1ull << ((n >> 6) & 63));
    }
    const int64_t c = (int64_t)blockIdx.y * 512 + lane * 8;
    float s[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    while (same) {
        constexpr int UN = 4;
        u32x4 v[UN];
        float l[UN];
        int k = 0;
#pragma unroll
        for (int u = 0; u < UN; ++u)
            if (same) {
                const int at = __ffsll((unsigned long long)same) - 1;
                same &= same - 1;
                l[u] = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(lost), at));
                v[u] = *reinterpret_cast<const u32x4*>(a.x + (n0 + at) * a.dp + min(c, a.dp - 8));
                k = u + 1;
            }
#pragma unroll
        for (int u = 0; u < UN; ++u)
            if (u < k)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    s[2 * i] = fmaf(l[u], bf16_lo(v[u][i]), s[2 * i]);
                    s[2 * i + 1] = fmaf(l[u], bf16_hi(v[u][i]), s[2 * i + 1]);
                }
    }
    if (c >= a.dp) return;
    f32x4* d = reinterpret_cast<f32x4*>(a.back + n * a.dp + c);
    d[0] = f32x4{s[0], s[1], s[2], s[3]};
    d[1] = f32x4{s[4], s[5], s[6], s[7]};
}
// More than 64 tokens: the first token of a target adds the rows of the later 64s, in their order.  (Found by
// going through all tokens' targets instead of the bits: 104 us for 8192 x 50288 x 2560, 34 so.)
__global__ void __launch_bounds__(256) k_ce_back_join(BackArgs a, Tokens tk) {
    const int n = blockIdx.x * 4 + wave_id(), lane = threadIdx.x & 63, count = *tk.count;
    if (n >= count) return;
    const int tgt = tk.tgt[n];
    if (tgt < a.v_first || tgt - a.v_first >= a.rows || tk.first[tgt] != n) return;
    const int64_t c = min((int64_t)blockIdx.y * 512 + lane * 8, a.dp - 8);      // (not stored twice)
    f32x4 x = zero4(), y = zero4();
    bool any = false;
    const unsigned long long* runs = tk.runs + (int64_t)tgt * tk.run_words;
    for (int word = n >> 12; word < tk.run_words; ++word) {
        uint64_t m = runs[word];
        if (word == n >> 12) m &= m - 1;             // n's own
        while (m) {
            constexpr int UN = 8;
            int run[UN], t[UN], k = 0;
#pragma unroll
            for (int u = 0; u < UN; ++u)
                if (m) {
                    run[u] = (word << 12) + ((__ffsll((unsigned long long)m) - 1) << 6);
                    m &= m - 1;
                    t[u] = tk.tgt[run[u] + lane];
                    k = u + 1;
                }
            f32x4 v[UN], w[UN];
#pragma unroll
            for (int u = 0; u < UN; ++u)
                if (u < k) {
                    const int i = run[u] + __ffsll((unsigned long long)__ballot(t[u] == tgt)) - 1;
                    const f32x4* p = reinterpret_cast<const f32x4*>(a.back + i * a.dp + c);
                    v[u] = p[0];
                    w[u] = p[1];
                }
#pragma unroll
            for (int u = 0; u < UN; ++u)
                if (u < k) {
                    x += v[u];
                    y += w[u];
                }
            any = true;
        }
    }
    if (!any) return;
    f32x4* d = reinterpret_cast<f32x4*>(a.back + (int64_t)n * a.dp + c);
    x += d[0];
    y += d[1];
    if ((int64_t)blockIdx.y * 512 + lane * 8 >= a.dp) return;
    d[0] = x;
    d[1] = y;
}

// ---------------------------------------------------------------------------
// joins
// ---------------------------------------------------------------------------
struct JoinArgs {
    const float2* part;
    int64_t np, n;
    float* loss;             // of every position, or NULL
    float* lse;              // the same
    float* total;            // or NULL
    double* sums;            // of each workgroup
    int parts, mean;
};

// 16 tokens per workgroup, 64 lanes each: lane q joins parts q, q + 64, ...  The losses are added
// up in float64, those of a workgroup first, then by the last one to be done the workgroups' in
// their order: which one is last changes nothing.
__global__ void __launch_bounds__(1024) k_ce_join(JoinArgs a, Tokens tk) {
    __shared__ float2 red[64][17];
    __shared__ bool last;
    __shared__ double wsum[16];
    const int t = threadIdx.x, tok = t & 15, q = t >> 4;
    const int64_t n = (int64_t)blockIdx.x * 16 + tok;
    const int k = n < a.n ? tk.inv[n] : -1;
    LogSum o;
    if (k >= 0) {
#pragma unroll 4
        for (int i = q; i < a.parts; i += 64) o.add(a.part[(int64_t)i * a.np + k]);
    }
    red[q][tok] = make_float2(o.mx, o.s);
    __syncthreads();
    if (q < 8) {
        o = LogSum();
#pragma unroll
        for (int i = q; i < 64; i += 8) o.add(red[i][tok]);
    }
    __syncthreads();
    if (q < 8) red[q][tok] = make_float2(o.mx, o.s);
    __syncthreads();
    if (t < 16) {
        float loss = 0.f, lse = 0.f;
        if (k >= 0) {
            o = LogSum();
#pragma unroll
            for (int i = 0; i < 8; ++i) o.add(red[i][tok]);
            const float zt = tk.zt[k];
            const float2 r = o.with_target(zt);
            loss = r.x;
            lse = r.y;
            tk.lse[k] = lse;
            tk.em1[k] = expm1f(-loss);
        }
        if (n < a.n) {
            if (a.loss) a.loss[n] = loss;
            if (a.lse) a.lse[n] = lse;
        }
        double s = loss;
#pragma unroll
        for (int e = 8; e >= 1; e >>= 1) s += __shfl_xor(s, e);
        if (t == 0) {
            last = false;
            if (a.total) {
                a.sums[blockIdx.x] = s;
                last = __hip_atomic_fetch_add(tk.count + 1, 1, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) ==
                       (int)gridDim.x - 1;
            }
        }
    }
    __syncthreads();
    if (!last) return;
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");
    double s = 0;
    for (int i = t; i < (int)gridDim.x; i += 1024) s += a.sums[i];
#pragma unroll
    for (int e = 32; e >= 1; e >>= 1) s += __shfl_xor(s, e);
    if ((t & 63) == 0) wsum[t >> 6] = s;
    __syncthreads();
    if (t == 0) {
        s = 0;
        for (int i = 0; i < 16; ++i) s += wsum[i];
        *a.total = (float)(s / (a.mean ? max(*tk.count, 1) : 1));
    }
}

// Up to 64 tokens, none of them dropped before the product: one workgroup, 16 to 64 lanes a
// token, which also adds the losses up
__global__ void __launch_bounds__(1024) k_ce_join_few(JoinArgs a, EpiLse e) {
    __shared__ float2 red[1024];
    const int w = a.n <= 16 ? 16 : a.n <= 32 ? 32 : 64;
    const int t = threadIdx.x, tok = t & (w - 1), q = t / w, lanes = 1024 / w;
    LogSum o;
    if (tok < a.n) {
#pragma unroll 4
        for (int i = q; i < a.parts; i += lanes) o.add(a.part[(int64_t)i * a.np + tok]);
    }
    red[t] = make_float2(o.mx, o.s);
    __syncthreads();
    // 4 lanes of the first wavefronts join the lanes' sums, the first of them the four
    if (q < 4) {
        o = LogSum();
        for (int i = q; i < lanes; i += 4) o.add(red[i * w + tok]);
    }
    __syncthreads();
    if (q < 4) red[t] = make_float2(o.mx, o.s);
    __syncthreads();
    if (t >= 64) return;
    float loss = 0.f, lse = 0.f;
    bool kept = false;
    if (t < a.n) {              // q == 0
        for (int i = 1; i < 4; ++i) o.add(red[i * w + tok]);
        kept = load_target(e.targets, e.t64, t) != e.ignore;
        if (kept) {
            const float zt = e.target(t) >= 0 ? e.zt[t] : __builtin_nanf("");
            const float2 r = o.with_target(zt);
            loss = r.x;
            lse = r.y;
        }
        if (a.loss) a.loss[t] = loss;
        if (a.lse) a.lse[t] = lse;
    }
    if (!a.total) return;
    double s = loss;
#pragma unroll
    for (int k = 32; k >= 1; k >>= 1) s += __shfl_xor(s, k);
    const int count = __popcll(__ballot(kept));
    if (t == 0) *a.total = (float)(s / (a.mean ? max(count, 1) : 1));
}

__global__ void k_ce_nothing(float* total) { *total = 0.f; }      // of no tokens

struct DxArgs {
    const float* part;
    bf16* dx;
    const bf16* w;           // the weights, rows of ldw
    int64_t n, np, dp, dim, ldw;
    int splits;
    Up up;
};

// dx of every row, 0 where it was left out: a wavefront per row and 512 columns
__global__ void __launch_bounds__(256) k_ce_dx(DxArgs a, Tokens tk) {
    const int64_t n = (int64_t)blockIdx.x * 4 + wave_id();
    if (n >= a.n) return;
    const int k = tk.inv[n];
    bf16* d = a.dx + n * a.dim;
    const int64_t c = (int64_t)blockIdx.y * 512 + (threadIdx.x & 63) * 8;
    if (c >= a.dim) return;
    f32x4 x = zero4(), y = zero4();
    if (k >= 0) {
        const float r = lost_of(tk, k);
        const bf16* w = a.w + max(tk.tgt[k], 0) * a.ldw + c;
        x = r * load4(w);
        y = r * load4(w + 4);
        const float* p = a.part + (int64_t)k * a.dp + c;
#pragma unroll 4
        for (int s = 0; s < a.splits; ++s, p += a.np * a.dp) {
            x += *reinterpret_cast<const f32x4*>(p);
            y += *reinterpret_cast<const f32x4*>(p + 4);
        }
        const float all = a.up.all(*tk.count);
        x *= all;
        y *= all;
    }
    const u32x4 o = {pk_bf16(x[0], x[1]), pk_bf16(x[2], x[3]), pk_bf16(y[0], y[1]), pk_bf16(y[2], y[3])};
    if (c + 8 <= a.dim) {
        store16(d + c, o);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (c + i < a.dim) reinterpret_cast<uint16_t*>(d)[c + i] = (uint16_t)(o[i >> 1] >> (16 * (i & 1)));
    }
}

// The same from the segments of k_ce_tile, in their order: a wavefront for two fragments (32
// columns) of 16 tokens; further workgroups zero the rows that were left out.
struct DxSegArgs {
    const float* part;
    void* dx;
    const bf16* w;           // the weights, rows of ldw
    int64_t n, dim, ldw;
    int tm, tn, seg_nk, nwg, nred;
    Up up;
};
template <typename T, class S> __global__ void __launch_bounds__(256) k_ce_dx_seg(DxSegArgs a, Tokens tk) {
    const int lane = threadIdx.x & 63;
    T* dx = static_cast<T*>(a.dx);
    if ((int)blockIdx.x >= a.nred) {
        for (int64_t r = (int64_t)(blockIdx.x - a.nred) * 4 + wave_id(); r < a.n; r += (int64_t)(gridDim.x - a.nred) * 4)
            if (tk.inv[r] < 0)
                for (int64_t c = lane; c < a.dim; c += 64) dx[r * a.dim + c] = from_f32<T>(0.f);
        return;
    }
    const int count = *tk.count;
    const int tn = min(a.tn, (((count + 63) & ~63) + S::BN - 1) / S::BN), tiles = a.tm * tn;
    constexpr int PAIRS = S::FM / 2, PER = S::NW * PAIRS * S::FN;
    int q = blockIdx.x * 4 + wave_id();
    const int tile = q / PER;
    q -= tile * PER;
    if (tile >= tiles) return;
    const int j = q % S::FN, i = q / S::FN % PAIRS * 2, w = q / S::FN / PAIRS;
    // (the tile's place as in k_ce_tile)
    const int grp = tile / (8 * tn), gm = min(8, a.tm - grp * 8), in = tile - grp * 8 * tn;
    const int m0 = (grp * 8 + in % gm) * S::BM + (w / S::WN * S::FM + i) * 16;
    const int n = in / gm * S::BN + (w % S::WN * S::FN + j) * 16 + (lane & 15);
    if (n - (lane & 15) >= count || m0 >= a.dim) return;
    f32x4 x = zero4(), y = zero4();
    if (sizeof(T) == 2 && n < count) {
        const float r = lost_of(tk, n);
        const int m = m0 + 4 * (lane >> 4);
        const bf16* w = a.w + max(tk.tgt[n], 0) * a.ldw + m;
        if (m < a.dim) x = r * load4(w);
        if (m + 16 < a.dim) y = r * load4(w + 16);
    }
    const Deal d = deal(tiles, a.seg_nk, a.nwg, S::STEP, S::SEG);
    constexpr int64_t SEG = (int64_t)S::NW * S::FM * S::FN * 64;
    const f32x4* p = reinterpret_cast<const f32x4*>(a.part) + tile * SEG + (w * S::FM * S::FN + i * S::FN + j) * 64 + lane;
    x += p[0];
    y += p[S::FN * 64];
    if (tile >= d.full) {
#pragma unroll 8
        for (int k = 1; k < d.s; ++k) {
            p += d.rest * SEG;
            x += p[0];
            y += p[S::FN * 64];
        }
    }
    const float all = a.up.all(count);
    if (n < count) store_row(dx + (int64_t)tk.idx[n] * a.dim, m0, a.dim, lane, all * x, all * y);
}

// ---------------------------------------------------------------------------
// plans
// ---------------------------------------------------------------------------
// Tiles of the logits (Z), of dx (X) and of dw (W); the number is a tile's n
template <bool F32> struct Shapes {
    typedef Shape<256, 256, 2, 4, 2, 64, false, false, 1> Z256;
    typedef Shape<128, 64, 4, 1, 3, 64, false, false, 1> Z64;
    typedef Shape<128, 16, 4, 1, 4, 64, false, false, 1> Z16;
    typedef Shape<256, 256, 2, 4, 2, 64, true, false, 1> X256;
    typedef Shape<256, 128, 2, 4, 2, 64, true, false, 1> X128;
    typedef Shape<256, 64, 4, 1, 3, 64, true, false, 1> X64;
    typedef Shape<256, 16, 4, 1, 3, 64, true, false, 1> X16;
    typedef Shape<256, 256, 2, 4, 2, 64, true, true, 1> W256;
    typedef Shape<128, 64, 4, 1, 3, 64, true, true, 1> W64;
};
template <> struct Shapes<true> {
    typedef Shape<256, 128, 4, 2, 2, 32, false, false, 6> Z128;
    typedef Shape<128, 64, 4, 2, 4, 32, false, false, 6> Z64;
    typedef Shape<128, 16, 4, 1, 4, 32, false, false, 6> Z16;
    typedef Shape<256, 128, 4, 2, 2, 32, true, false, 6> X128;
    typedef Shape<128, 64, 4, 2, 4, 32, true, false, 6> X64;
    typedef Shape<128, 16, 4, 1, 4, 32, true, false, 6> X16;
    typedef Shape<256, 128, 4, 2, 2, 32, true, true, 6> W128;
    typedef Shape<128, 64, 4, 2, 4, 32, true, true, 6> W64;
};

// Tokens of a tile of the logits.  bf16: the tiles of 256 x 256 run at three times the rate of
// those of 128 x 64, but where they leave more than half of the CUs without one, the
// small ones are faster.  float32: 256 x 128 and 128 x 64 alike, by rounds over the CUs.
bool fills(int64_t m, int64_t n) { return 2 * (int64_t)tiles(m, 256) * tiles(n, 256) > m2::cu_count(); }
bool large_planes(int64_t m, int64_t n) {
    typedef Shapes<true>::Z128 L;
    typedef Shapes<true>::Z64 S;
    const int64_t ncu = m2::cu_count();
    return L::STEP * (((int64_t)tiles(m, L::BM) * tiles(n, L::BN) + ncu - 1) / ncu) <=
           S::STEP * (((int64_t)tiles(m, S::BM) * tiles(n, S::BN) + ncu - 1) / ncu);
}
int z_tile(int64_t n, int64_t vocab, bool f32) {
    if (n <= 16) return 16;
    if (f32) return n > 64 && large_planes(vocab, n) ? 128 : 64;
    return n <= 64 || !fills(vocab, n) ? 64 : 256;
}
int z_rows(int z) { return z < 128 ? 128 : 256; }
// parts of a tile whose sums EpiLse leaves apart
int z_parts(int z, bool f32) { return f32 ? 4 : z < 256 ? 1 : 2; }

// What the two entry points share: sizes, the packed operands and the tokens' arrays.
struct Common {
    int64_t n, vocab, dim, np, dp;
    bool f32, pack_w;
    size_t idx, inv, tgt, lse, em1, count, first, runs, x, w, at;
    int run_words;
    int z;                   // tokens of a tile of the logits
};

// grad: with what only a gradient reads
Common common(int64_t n, int64_t vocab, int64_t dim, int64_t ldw, const void* w, int dtype, bool grad) {
    Common c{};
    c.n = n; c.vocab = vocab; c.dim = dim;
    c.np = (n + 63) / 64 * 64;
    c.dp = (dim + 63) / 64 * 64;
    c.f32 = dtype == M2_F32;
    c.z = z_tile(n, vocab, c.f32);
    // the weights are read in place where direct loads can: bf16 rows of whole 16-byte
    // pieces (and offsets within a tile that fit 32 bits), of whole K steps for k_ce_tile; else
    // a copy in the workspace
    c.pack_w = c.f32 || dim % (c.z < 256 ? 8 : 64) || ldw % 8 || !al16(w) || ldw > (1 << 22);
    auto take = [&](size_t b) { const size_t r = c.at; c.at += align256(b); return r; };
    c.idx = take(4 * (size_t)c.np);
    c.inv = take(4 * (size_t)c.np);
    c.tgt = take(4 * (size_t)c.np);
    c.lse = take(4 * (size_t)c.np);
    c.em1 = take(4 * (size_t)c.np);
    c.count = take(8);
    // (bf16's gradient: 4 bytes and a bit for each 64 tokens a row of the vocabulary)
    c.run_words = (int)((n + 4095) / 4096);
    c.first = c.f32 || !grad ? c.at : take(4 * (size_t)vocab);
    c.runs = c.f32 || !grad ? c.at : take(8 * (size_t)vocab * c.run_words);
    const size_t planes = c.f32 ? 3 : 1;
    c.x = take(2 * planes * (size_t)c.np * c.dp);
    c.w = c.pack_w ? take(2 * planes * (size_t)vocab * c.dp) : c.at;
    return c;
}

template <bool F32, class EPI> void launch_z(Gemm& g, int z, int64_t rows, int64_t n, const EPI& e, hipStream_t s) {
    typedef Shapes<F32> P;
    g.tm = tiles(rows, z_rows(z));
    g.tn = tiles(n, z);
    switch (z) {
        case 16: launch<typename P::Z16>(g, e, s); break;
        case 64: launch<typename P::Z64>(g, e, s); break;
        default:
            if constexpr (F32) launch<typename P::Z128>(g, e, s);
            else launch<typename P::Z256>(g, e, s);
    }
}

int check_sizes(const char* who, int64_t n, int64_t vocab, int64_t dim, int64_t ldx, int64_t ldw, int dtype,
                int tdtype) {
    M2_REQUIRE(n >= 0 && n < (1 << 30) && vocab > 0 && vocab < (1 << 30) && dim > 0 && dim <= (1 << 20),
               M2_ERR_INVALID, "%s: bad sizes (n %lld, vocab %lld, dim %lld)", who, (long long)n,
               (long long)vocab, (long long)dim);
    M2_REQUIRE(ldx >= dim && ldw >= dim, M2_ERR_INVALID, "%s: row strides", who);
    M2_REQUIRE(dtype == M2_F32 || dtype == M2_BF16, M2_ERR_UNSUPPORTED, "%s: dtype %d", who, dtype);
    M2_REQUIRE(tdtype == M2_I32 || tdtype == M2_I64, M2_ERR_UNSUPPORTED, "%s: target dtype %d", who, tdtype);
    M2_REQUIRE((int64_t)tiles(vocab, 128) * tiles(n, 16) < (1ll << 28) || n > 64, M2_ERR_UNSUPPORTED,
               "%s: too large", who);
    M2_REQUIRE((int64_t)tiles(vocab, 256) * tiles(n, 256) < (1ll << 30), M2_ERR_UNSUPPORTED, "%s: too large", who);
    // (a launch counts its threads in 32 bits: a wavefront for each token, and a workgroup for CLEAR rows of the vocabulary)
    M2_REQUIRE((n + 67) / 4 + tiles(vocab, CLEAR) < (1 << 24), M2_ERR_UNSUPPORTED, "%s: too many rows", who);
    return M2_OK;
}
// the same of weight's rows, where they are packed
int check_packed(const char* who, const Common& c) {
    M2_REQUIRE(!c.pack_w || (c.vocab + 3) / 4 < (1 << 24), M2_ERR_UNSUPPORTED, "%s: too many rows to pack", who);
    return M2_OK;
}

struct FwdPlan {
    Common c;
    bool direct;             // x read in place, nothing packed: few tokens
    size_t zt, part, sums, total;
};
FwdPlan fwd_plan(const m2_linear_cross_entropy_args& a) {
    FwdPlan p{};
    p.c = common(a.n, a.vocab, a.dim, a.ldw, a.weight, a.dtype, a.saved != nullptr);
    // (the kernel's offsets within a tile are of 32 bits: rows that lie further apart, the last
    // positions of long prompts, are packed, with 64-bit addresses)
    p.direct = a.n <= 64 && !a.saved && !p.c.pack_w && a.ldx % 8 == 0 && al16(a.x) &&
               a.ldx <= (1ll << 30) / (a.n > 1 ? a.n - 1 : 1);
    size_t at = p.direct || a.saved ? 0 : p.c.at;
    auto take = [&](size_t b) { const size_t r = at; at += align256(b); return r; };
    p.zt = take(4 * (size_t)p.c.np);
    p.part = take(8 * (size_t)z_parts(p.c.z, p.c.f32) * tiles(a.vocab, z_rows(p.c.z)) * p.c.np);
    p.sums = take(8 * (size_t)tiles(a.n, 16));
    p.total = at ? at : 256;
    return p;
}

// G's workspace: 512 MB of it, or one tile of the vocabulary (256 rows) for all tokens where that
// is more (from a million bf16 tokens, 350000 of float32, on).  More
// pieces cost launches and passes over the partial dx (8192 x 50288 x 2560: with 192 MB 6.92 ms
// against 6.66, with 1 GB 6.67).
constexpr int64_t G_BYTES = 512ll << 20;
struct BwdPlan {
    Common c;
    int64_t piece;
    int pieces;
    int x, splits;           // dx: tokens of a tile; parts of K (few tokens) or workgroups (many)
    size_t G, dx, lost, back, total;
};
BwdPlan bwd_plan(const m2_linear_cross_entropy_grad_args& a) {
    BwdPlan p{};
    p.c = common(a.n, a.vocab, a.dim, a.ldw, a.weight, a.dtype, true);
    size_t at = a.saved ? 0 : p.c.at;
    auto take = [&](size_t b) { const size_t r = at; at += align256(b); return r; };
    const int planes = p.c.f32 ? 3 : 1;
    const int64_t all = (a.vocab + 255) / 256 * 256;
    int64_t most = G_BYTES / (2 * planes * (p.c.np ? p.c.np : 64)) / 256 * 256;
    if (most < 256) most = 256;
    p.pieces = (int)((all + most - 1) / most);
    p.piece = ((all / 256 + p.pieces - 1) / p.pieces) * 256;
    p.pieces = (int)((all + p.piece - 1) / p.piece);
    p.lost = take(4 * (size_t)p.c.np);
    p.back = p.c.f32 || !a.grad_weight ? 0 : take(4 * (size_t)p.c.np * p.c.dp);
    p.G = take(2 * planes * (size_t)(p.c.np ? p.c.np : 64) * p.piece);
    // dx: K is the piece.  Many tokens: dealt out with the tiles (k_ce_tile), whose number
    // depends on the tokens that are kept.  Few: split so that the tiles fill the CUs; a
    // split costs a float32 array of dx, written and read once per piece
    const int ncu = m2::cu_count();
    const int steps = (int)((a.vocab < p.piece ? a.vocab + 63 : p.piece) / 64);
    const int tm = tiles(a.dim, 256);
    // with the shape S: what its plan costs, and the most segments over the numbers of kept tokens
    auto cost = [&](auto shape) {
        typedef decltype(shape) S;
        return deal(tiles(a.dim, S::BM) * tiles(a.n ? a.n : 1, S::BN), steps, ncu, S::STEP, S::SEG).cost;
    };
    int64_t all_segs = 0;
    auto take_segs = [&](auto shape) {
        typedef decltype(shape) S;
        int64_t segs = 0;
        for (int k = 1; k <= tiles(a.n ? a.n : 1, S::BN); ++k) {
            const Deal d = deal(tiles(a.dim, S::BM) * k, steps, ncu, S::STEP, S::SEG);
            all_segs = d.full + (int64_t)d.rest * d.s;
            if (all_segs > segs) segs = all_segs;
        }
        p.x = S::BN;
        p.splits = ncu;
        return 4 * (size_t)S::BM * S::BN * segs;
    };
    if (p.c.f32) {
        typedef Shapes<true> P;
        const size_t b = a.n <= 16 ? take_segs(P::X16())
                         : a.n > 64 && cost(P::X128()) <= cost(P::X64()) ? take_segs(P::X128()) : take_segs(P::X64());
        p.dx = a.grad_x ? take(b) : 0;
        p.total = at;
        return p;
    }
    if (a.n > 64) {
        typedef Shapes<false> P;
        const size_t b = cost(P::X256()) <= cost(P::X128()) ? take_segs(P::X256()) : take_segs(P::X128());
        if (2 * all_segs > ncu) {
            p.dx = a.grad_x ? take(b) : 0;
            p.total = at;
            return p;
        }
    }
    p.x = a.n <= 16 ? 16 : 64;                // few: the smaller tiles, as for the logits
    const int64_t t = (int64_t)tm * tiles(a.n ? a.n : 1, p.x);
    double best = 1e300;
    p.splits = 1;
    for (int s = 1; s <= 64 && s * 4 <= steps; ++s) {
        const double rounds = (double)((t * s + ncu - 1) / ncu);
        const double cost = rounds * ((double)steps / s + 12.0) + 0.02 * s * t;
        if (cost < best) { best = cost; p.splits = s; }
    }
    p.dx = a.grad_x ? take(4 * (size_t)p.splits * p.c.np * p.c.dp) : 0;
    p.total = at;
    return p;
}

Tokens tokens(char* ws, const Common& c) {
    Tokens t{};
    t.idx = reinterpret_cast<int*>(ws + c.idx);
    t.inv = reinterpret_cast<int*>(ws + c.inv);
    t.tgt = reinterpret_cast<int*>(ws + c.tgt);
    t.lse = reinterpret_cast<float*>(ws + c.lse);
    t.em1 = reinterpret_cast<float*>(ws + c.em1);
    t.count = reinterpret_cast<int*>(ws + c.count);
    t.first = reinterpret_cast<int*>(ws + c.first);
    t.runs = reinterpret_cast<unsigned long long*>(ws + c.runs);
    t.run_words = c.run_words;
    return t;
}

template <typename T>
void pack(char* ws, const Common& c, const void* x, int64_t ldx, const void* w, int64_t ldw, PackArgs a,
          const Tokens& tk, int64_t ignore, bool grad, hipStream_t s) {
    a.n = c.n; a.ignore = ignore;
    const bool finds = c.n <= PACK_FINDS;
    if (!finds) hipLaunchKernelGGL(k_ce_compact, dim3(1), dim3(1024), 0, s, a.targets, c.n, ignore, a.t64, tk);
    a.dim = c.dim; a.dp = c.dp;
    a.src = x; a.ld = ldx; a.dst = reinterpret_cast<bf16*>(ws + c.x); a.rows = c.np; a.plane = c.np * c.dp;
    a.row_blocks = (int)((finds ? c.n + 67 : c.np) / 4);
    const int clear = grad && !c.f32 ? tiles(c.vocab, CLEAR) : 0;
    hipLaunchKernelGGL((k_ce_pack<T, true>), dim3((unsigned)(a.row_blocks + clear)), dim3(256), 0, s, a, tk);
    if (c.pack_w) {
        a.src = w; a.ld = ldw; a.dst = reinterpret_cast<bf16*>(ws + c.w); a.rows = c.vocab;
        a.plane = c.vocab * c.dp;
        hipLaunchKernelGGL((k_ce_pack<T, false>), dim3((unsigned)((c.vocab + 3) / 4)), dim3(256), 0, s, a, tk);
    }
}

Operand operand_w(char* ws, const Common& c, const void* w, int64_t ldw) {
    if (c.pack_w) return Operand{reinterpret_cast<bf16*>(ws + c.w), c.dp, c.vocab * c.dp, 0, 0};
    return Operand{static_cast<const bf16*>(w), ldw, 0, 0, 0};
}

template <bool F32> int run_fwd(const m2_linear_cross_entropy_args& a, const FwdPlan& p, hipStream_t s) {
    typedef typename std::conditional<F32, float, bf16>::type T;
    char* ws = static_cast<char*>(a.workspace);
    char* cm = a.saved ? static_cast<char*>(a.saved) : ws;
    const Common& c = p.c;
    const int t64 = a.target_dtype == M2_I64;
    float* zt = reinterpret_cast<float*>(ws + p.zt);
    EpiLse e{nullptr, a.targets, a.ignore_index, zt, reinterpret_cast<float2*>(ws + p.part), c.np, (int)c.vocab, t64};
    Gemm g{};
    g.tok_n = 1; g.splits = 1;
    g.nk = (int)(c.dp / 64);
    JoinArgs j{e.part, c.np, c.n, a.loss, a.lse, a.total, reinterpret_cast<double*>(ws + p.sums), 0, a.mean};
    if (p.direct) {
        g.n = (int)c.n;
        g.a = Operand{static_cast<const bf16*>(a.weight), a.ldw, 0, (int)c.vocab, (int)c.dim};
        g.b = Operand{static_cast<const bf16*>(a.x), a.ldx, 0, (int)c.n, (int)c.dim};
        launch_z<F32>(g, c.z, c.vocab, c.n, e, s);
        j.parts = g.tm;
        hipLaunchKernelGGL(k_ce_join_few, dim3(1), dim3(1024), 0, s, j, e);
        return m2::check_launch("linear_cross_entropy");
    }
    Tokens tk = tokens(cm, c);
    tk.zt = zt;
    PackArgs pa{};
    pa.targets = a.targets; pa.vocab = a.vocab; pa.t64 = t64;
    pack<T>(cm, c, a.x, a.ldx, a.weight, a.ldw, pa, tk, a.ignore_index, a.saved != nullptr, s);
    g.count = tk.count;
    g.a = operand_w(cm, c, a.weight, a.ldw);
    g.a.lim = (int)c.vocab;
    g.a.klim = (int)(c.pack_w ? c.dp : c.dim);
    g.b = Operand{reinterpret_cast<bf16*>(cm + c.x), c.dp, c.np * c.dp, (int)c.np, (int)c.dp};
    e.tgt = tk.tgt;
    launch_z<F32>(g, c.z, c.vocab, c.n, e, s);
    j.parts = g.tm * z_parts(c.z, F32);
    hipLaunchKernelGGL(k_ce_join, dim3((unsigned)tiles(c.n, 16)), dim3(1024), 0, s, j, tk);
    return m2::check_launch("linear_cross_entropy");
}

template <bool F32> int run_bwd(const m2_linear_cross_entropy_grad_args& a, const BwdPlan& p, hipStream_t s) {
    typedef typename std::conditional<F32, float, bf16>::type T;
    typedef Shapes<F32> P;
    char* ws = static_cast<char*>(a.workspace);
    char* cm = a.saved ? static_cast<char*>(a.saved) : ws;
    const Common& c = p.c;
    Tokens tk = tokens(cm, c);
    tk.lost = reinterpret_cast<float*>(ws + p.lost);
    PackArgs pa{};
    pa.targets = a.targets; pa.vocab = a.vocab; pa.t64 = a.target_dtype == M2_I64;
    pa.lse = a.lse; pa.loss = a.loss;
    if (!a.saved) pack<T>(cm, c, a.x, a.ldx, a.weight, a.ldw, pa, tk, a.ignore_index, true, s);
    const Operand w = operand_w(cm, c, a.weight, a.ldw);
    bf16* G = reinterpret_cast<bf16*>(ws + p.G);
    const int64_t gplane = c.np * p.piece;
    Gemm g0{};
    g0.count = tk.count; g0.splits = 1;
    float* dxp = reinterpret_cast<float*>(ws + p.dx);
    const int wlim = (int)(c.pack_w ? c.dp : c.dim);
    const Up up{a.grad_loss, a.grad_loss_stride, a.mean};
    DxSegArgs dxs{};
    dxs.up = up;
    for (int q = 0; q < p.pieces; ++q) {
        const int64_t v0 = q * p.piece;
        const int64_t rows = c.vocab - v0 < p.piece ? c.vocab - v0 : p.piece;
        // G of the piece
        Gemm g = g0;
        g.nk = (int)(c.dp / 64); g.tok_n = 1;
        g.a = w;
        g.a.p += v0 * w.ld;
        g.a.lim = (int)rows;
        g.a.klim = wlim;
        g.b = Operand{reinterpret_cast<bf16*>(cm + c.x), c.dp, c.np * c.dp, (int)c.np, (int)c.dp};
        const EpiG eg{tk, up, G, p.piece, gplane, (int)v0, (int)c.vocab};
        launch_z<F32>(g, c.z, (rows + 63) / 64 * 64, c.n, eg, s);
        if (a.grad_x) {
            Gemm d = g0;
            d.nk = (int)((rows + 63) / 64); d.tok_n = 1;
            d.splits = p.splits;
            d.a = w;
            d.a.p += v0 * w.ld;
            d.a.lim = wlim;
            d.a.klim = (int)rows;
            d.b = Operand{G, p.piece, gplane, (int)c.np, (int)p.piece};
            d.tn = tiles(c.n, p.x);
            if (q == 0) dxs.seg_nk = d.nk;
            d.seg_nk = dxs.seg_nk;
            const EpiDxSeg seg{dxp, q > 0};
            auto go = [&](auto shape, const auto& e) {
                typedef decltype(shape) S;
                d.tm = tiles(c.dim, S::BM);
                launch<S>(d, e, s);
            };
            if constexpr (F32) {
                if (p.x == 128) go(typename P::X128(), seg);
                else if (p.x == 64) go(typename P::X64(), seg);
                else go(typename P::X16(), seg);
            } else if (p.x >= 128) {
                if (p.x == 256) go(typename P::X256(), seg);
                else go(typename P::X128(), seg);
            } else {
                if (d.splits > d.nk) d.splits = d.nk;             // a short last piece
                const EpiDxSplit e{dxp, c.np, c.dp, q > 0};
                if (p.x == 16) go(typename P::X16(), e);
                else go(typename P::X64(), e);
            }
            dxs.tm = d.tm; dxs.tn = d.tn; dxs.nwg = p.splits;
        }
        if (a.grad_weight) {
            const BackArgs back{reinterpret_cast<const bf16*>(cm + c.x), reinterpret_cast<float*>(ws + p.back), c.dp,
                                (int)v0, (int)rows};
            if constexpr (!F32) {
                const dim3 grid((unsigned)(c.np / 4), (unsigned)((c.dp + 511) / 512));
                hipLaunchKernelGGL(k_ce_back, grid, dim3(256), 0, s, back, tk);
                if (c.n > 64) hipLaunchKernelGGL(k_ce_back_join, grid, dim3(256), 0, s, back, tk);
            }
            Gemm d = g0;
            d.nk = 0;
            d.a = Operand{reinterpret_cast<bf16*>(cm + c.x), c.dp, c.np * c.dp, (int)c.dp, (int)c.np};
            // rows of G past a tile of 16 tokens are not there: its last row stands for them,
            // against zero rows of x
            d.b = Operand{G, p.piece, gplane, (int)p.piece, c.z == 16 ? 16 : (int)c.np};
            auto go = [&](auto shape) {
                typedef decltype(shape) S;
                d.tm = tiles(c.dim, S::BM); d.tn = tiles(rows, S::BN);
                T* dw = static_cast<T*>(a.grad_weight) + v0 * c.dim;
                launch<S>(d, EpiDw<T>{dw, c.dim, c.dp, back.back, tk.first + v0, up, (int)rows}, s);
            };
            if constexpr (F32) {
                if (large_planes(c.dim, rows)) go(typename P::W128());
                else go(typename P::W64());
            } else {
                if (fills(c.dim, rows)) go(typename P::W256());
                else go(typename P::W64());
            }
        }
    }
    if (!a.grad_x) return m2::check_launch("linear_cross_entropy_grad");
    auto reduce = [&](auto shape) {
        typedef decltype(shape) S;
        dxs.part = dxp; dxs.dx = a.grad_x; dxs.n = c.n; dxs.dim = c.dim;
        dxs.w = w.p; dxs.ldw = w.ld;
        dxs.nred = (dxs.tm * dxs.tn * (S::NW * S::FM / 2 * S::FN) + 3) / 4;
        hipLaunchKernelGGL((k_ce_dx_seg<T, S>), dim3((unsigned)(dxs.nred + tiles(c.n, 64))), dim3(256), 0, s, dxs, tk);
    };
    if constexpr (F32) {
        if (p.x == 128) reduce(typename P::X128());
        else if (p.x == 64) reduce(typename P::X64());
        else reduce(typename P::X16());
    } else if (p.x >= 128) {
        if (p.x == 256) reduce(typename P::X256());
        else reduce(typename P::X128());
    } else {
        const DxArgs d{dxp, static_cast<bf16*>(a.grad_x), w.p, c.n, c.np, c.dp, c.dim, w.ld, p.splits, up};
        hipLaunchKernelGGL(k_ce_dx, dim3((unsigned)((c.n + 3) / 4), (unsigned)((c.dim + 511) / 512)), dim3(256), 0, s, d,
                           tk);
    }
    return m2::check_launch("linear_cross_entropy_grad");
}

}  // namespace

namespace m2 {

size_t linear_ce_saved(const m2_linear_cross_entropy_args& a) {
    if (check_sizes("linear_cross_entropy", a.n, a.vocab, a.dim, a.ldx, a.ldw, a.dtype, a.target_dtype)) return 0;
    const Common c = common(a.n, a.vocab, a.dim, a.ldw, a.weight, a.dtype, true);
    return check_packed("linear_cross_entropy", c) ? 0 : c.at;
}

size_t linear_ce_workspace(const m2_linear_cross_entropy_args& a) {
    if (check_sizes("linear_cross_entropy", a.n, a.vocab, a.dim, a.ldx, a.ldw, a.dtype, a.target_dtype)) return 0;
    const FwdPlan p = fwd_plan(a);
    return check_packed("linear_cross_entropy", p.c) ? 0 : p.total;
}

int launch_linear_ce(const m2_linear_cross_entropy_args& a, hipStream_t s) {
    const char* who = "linear_cross_entropy";
    if (int rc = check_sizes(who, a.n, a.vocab, a.dim, a.ldx, a.ldw, a.dtype, a.target_dtype)) return rc;
    M2_REQUIRE(a.weight && (a.n == 0 || (a.x && a.targets)) && (a.loss || a.total), M2_ERR_INVALID,
               "%s: x, weight, targets and loss or total are required", who);
    const FwdPlan p = fwd_plan(a);
    if (int rc = check_packed(who, p.c)) return rc;
    M2_REQUIRE(a.workspace && a.workspace_bytes >= p.total, M2_ERR_WORKSPACE,
               "%s: workspace of %zu bytes needed, %zu given", who, p.total, a.workspace_bytes);
    M2_REQUIRE(!a.saved || a.saved_bytes >= p.c.at, M2_ERR_WORKSPACE, "%s: saved of %zu bytes needed, %zu given",
               who, p.c.at, a.saved_bytes);
    if (a.n == 0) {
        if (a.total) hipLaunchKernelGGL(k_ce_nothing, dim3(1), dim3(1), 0, s, a.total);
        return check_launch(who);
    }
    return a.dtype == M2_F32 ? run_fwd<true>(a, p, s) : run_fwd<false>(a, p, s);
}

size_t linear_ce_grad_workspace(const m2_linear_cross_entropy_grad_args& a) {
    if (check_sizes("linear_cross_entropy_grad", a.n, a.vocab, a.dim, a.ldx, a.ldw, a.dtype, a.target_dtype))
        return 0;
    const BwdPlan p = bwd_plan(a);
    return check_packed("linear_cross_entropy_grad", p.c) ? 0 : p.total;
}

int launch_linear_ce_grad(const m2_linear_cross_entropy_grad_args& a, hipStream_t s) {
    const char* who = "linear_cross_entropy_grad";
    if (int rc = check_sizes(who, a.n, a.vocab, a.dim, a.ldx, a.ldw, a.dtype, a.target_dtype)) return rc;
    M2_REQUIRE(a.n > 0, M2_ERR_INVALID, "%s: no tokens", who);
    M2_REQUIRE(a.weight && a.grad_loss && (a.grad_x || a.grad_weight), M2_ERR_INVALID,
               "%s: weight, grad_loss and an output are required", who);
    M2_REQUIRE(a.saved || (a.x && a.targets && a.loss && a.lse), M2_ERR_INVALID,
               "%s: saved, or x, targets, loss and lse are required", who);
    M2_REQUIRE(a.grad_loss_stride >= 0, M2_ERR_INVALID, "%s: grad_loss stride", who);
    const BwdPlan p = bwd_plan(a);
    if (int rc = check_packed(who, p.c)) return rc;
    M2_REQUIRE(!a.saved || a.saved_bytes >= p.c.at, M2_ERR_WORKSPACE, "%s: saved of %zu bytes needed, %zu given",
               who, p.c.at, a.saved_bytes);
    M2_REQUIRE(a.workspace && a.workspace_bytes >= p.total, M2_ERR_WORKSPACE,
               "%s: workspace of %zu bytes needed, %zu given", who, p.total, a.workspace_bytes);
    return a.dtype == M2_F32 ? run_bwd<true>(a, p, s) : run_bwd<false>(a, p, s);
}

}  // namespace m2
