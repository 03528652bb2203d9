// The gated linear recurrence over time and its gradient: independent per channel,
//
//   q = sigmoid(r), s = sigmoid(i), log a = A q (A <= 0), beta = sqrt(1 - a^2)
//   h[t] = a h[t-1] + beta s x[t]
//   l[t] = g[t] + m[t+1], m[t] = a l[t]        (l: the gradient of h[t], m: what of it goes on)
//   dx = l beta s;  di = dx x (1 - s);  dL = l (a h[t-1] - a^2 / beta s x);  dr = dL A q (1 - q)
//   dA = sum dL q;  dh0 = m[0]
//
// A workgroup owns the channels of a slab of one batch row and walks its whole length in
// tiles, forward or backward; the state is carried from tile to tile in registers, so every
// input is read once and nothing passes between workgroups.  Inside a tile each thread runs TS
// consecutive steps of V channels; a run of steps is an affine map h -> P h + H, and the maps of the
// threads of a wavefront (by lane shifts) and then of the wavefronts (by LDS, one barrier a tile)
// are joined to the state that each thread's run begins with.  The forward leaves the state
// that enters every span of 64 steps (float32, 1/64 of a stream); the backward goes through
// the tiles from the last to the first, computes the states of a tile again from there and both joins at
// once (a run's map backward, m -> P m + M, has the same P).
//
// Everything is float32 but what is loaded and stored.  alpha = 1 - a is kept in place of a: near
// 1, where memories are long, a itself has too few bits (beta^2 = alpha (2 - alpha) loses none,
// and h - alpha h + b rounds by the step's own size only).
//
// Where seq_idx changes the state is cleared: P = -1 marks a run that holds such a step, so that what
// came before (a NaN, say) is selected away and not multiplied by zero.  Negative seq_idx is
// padding: a = 1, nothing added, 0 stored; so are the steps past the end of the row.
#include "m2_internal.h"

namespace {

constexpr float LOG2E = 1.4426950408889634f;
constexpr int SPAN = M2_RECURRENCE_SPAN;

// V consecutive channels of a row, as loaded; rows need be aligned as their elements only
template <typename T, int V> struct Raw;
template <> struct Raw<bf16, 4> {
    typedef uint32_t any __attribute__((ext_vector_type(2), aligned(2)));
    any v;
    M2_DEV void load(const bf16* p) { v = *reinterpret_cast<const any*>(p); }
    M2_DEV float get(int i) const { return i & 1 ? bf16_hi(v[i >> 1]) : bf16_lo(v[i >> 1]); }
    static M2_DEV void store(bf16* p, const float (&f)[4]) {
        *reinterpret_cast<any*>(p) = any{pk_bf16(f[0], f[1]), pk_bf16(f[2], f[3])};
    }
};
template <> struct Raw<float, 4> {
    typedef uint32_t any __attribute__((ext_vector_type(4), aligned(4)));
    any v;
    M2_DEV void load(const float* p) { v = *reinterpret_cast<const any*>(p); }
    M2_DEV float get(int i) const { return __uint_as_float(v[i]); }
    static M2_DEV void store(float* p, const float (&f)[4]) {
        *reinterpret_cast<any*>(p) = any{__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]),
                                         __float_as_uint(f[3])};
    }
};
template <typename T> struct Raw<T, 1> {
    T v;
    M2_DEV void load(const T* p) { v = *p; }
    M2_DEV float get(int) const { return to_f32(v); }
    static M2_DEV void store(T* p, const float (&f)[1]) { *p = from_f32<T>(f[0]); }
};
// the values from `skip` on
template <typename T, int V> M2_DEV void put(T* p, const float (&f)[V], int skip) {
    if (skip == 0) {
        Raw<T, V>::store(p, f);
    } else {
#pragma unroll
        for (int v = 1; v < V; ++v)
            if (v >= skip) p[v] = from_f32<T>(f[v]);
    }
}

M2_DEV float sigmoid(float v) { return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(v * -LOG2E)); }
// 1 - sigmoid(v), which keeps its bits where the sigmoid is near 1
M2_DEV float co_sigmoid(float v, float s) { return v > 0.f ? s * __builtin_amdgcn_exp2f(v * -LOG2E) : 1.f - s; }
// 1 - exp(L): the series to L^7 / 7! (its rest is below 2^-25 of it) where 1 - exp would cancel
M2_DEV float decay(float L) {
    float p = fmaf(L, 1.f / 7, 1.f);
    p = fmaf(L * p, 1.f / 6, 1.f);
    p = fmaf(L * p, 1.f / 5, 1.f);
    p = fmaf(L * p, 1.f / 4, 1.f);
    p = fmaf(L * p, 1.f / 3, 1.f);
    p = fmaf(L * p, 1.f / 2, 1.f);
    return L < -0.35f ? 1.f - __builtin_amdgcn_exp2f(L * LOG2E) : -L * p;
}
// a p + b.  (The product's operand is bounded: an infinite p stays what it is and is not inf - inf.)
M2_DEV float step(float alpha, float p, float b) {
    constexpr float MAX = 3.402823466e38f;
    return fmaf(-alpha, __builtin_amdgcn_fmed3f(p, -MAX, MAX), p + b);
}
// 1 / sqrt(1 - a^2), 0 where a is 1 (below 1e-37 the hardware's root has no argument left)
M2_DEV float inv_beta(float alpha, float& y) {
    y = alpha * (2.f - alpha);
    return fabsf(y) <= 1e-37f ? 0.f : __builtin_amdgcn_rsqf(y);
}

// an affine map v -> P v + H; P = -1: the state is cleared in it, v -> H
template <bool SEQ> struct Map {
    float P, H;
    M2_DEV float of(float v) const { return SEQ && P < 0.f ? H : fmaf(P, v, H); }
    // this one behind `first`
    M2_DEV Map after(const Map& first) const {
        Map m;
        m.H = of(first.H);
        m.P = P * first.P;
        if constexpr (SEQ) m.P = P < 0.f || first.P < 0.f ? -1.f : m.P;
        return m;
    }
};

struct RecArgs {
    const void *x, *r, *i;
    const float *A, *h0;
    const int32_t* seq;
    int64_t xb, xt, rb, rt, ib, it;      // strides of batch and time
    float* ck;                           // [batch][spans][dim]
    int64_t L, spans;
    int dim, slabs;
    // forward
    void* out;
    float* last;
    // backward
    const void* g;
    int64_t gb, gt;
    const float* glast;
    void *dx, *dr, *di;
    float* dA;                           // [batch][dim]
    float* dh0;
};

// Which channels and steps of a tile a thread has
template <int V, int LC, int TS, int W> struct Place {
    static constexpr int G = 64 / LC, TILE = G * W * TS, C = V * LC;
    int b, c, col, tg, w, step;          // col: place in the slab
    int skip;                            // the lane's first channels that another one stores
    M2_DEV Place(const RecArgs& a) {
        const int lane = threadIdx.x & 63;
        const int id = xcd_remap(blockIdx.x, gridDim.x);
        b = id / a.slabs;
        w = wave_id();
        col = (lane % LC) * V;
        tg = lane / LC;
        // (a lane that reaches past the last channel has the last V, and those past it V that others store)
        const int from = (id - b * a.slabs) * C + col;
        c = min(from, a.dim - V);
        skip = from - c;
        step = (w * G + tg) * TS;
    }
};

// The steps of a tile that a thread has: bit j of live: inside the row and no padding; of clear: the
// state is cleared before it
template <int TS, bool SEQ> struct Steps {
    int sq[SEQ ? TS + 1 : 1];
    uint32_t live, clear;
    M2_DEV void load(const int32_t* row, int64_t t, int64_t L) {
        if constexpr (SEQ) {
#pragma unroll
            for (int j = 0; j <= TS; ++j) {
                const int64_t at = t + j - 1;
                sq[j] = row[at < 0 ? 0 : at < L ? at : L - 1];
            }
        }
    }
    M2_DEV void set(int64_t t, int64_t L) {
        live = clear = 0;
#pragma unroll
        for (int j = 0; j < TS; ++j) {
            const bool in = t + j < L;
            if constexpr (SEQ) {
                live |= (uint32_t)(in && sq[j + 1] >= 0) << j;
                clear |= (uint32_t)(in && sq[j + 1] >= 0 && sq[j + 1] != sq[j]) << j;
            } else {
                live |= (uint32_t)in << j;
            }
        }
    }
    M2_DEV bool is_live(int j) const { return live >> j & 1; }
    M2_DEV bool clears(int j) const { return SEQ && (clear >> j & 1); }
};

// the maps of the lanes of each channel, joined in the order of their steps: inclusive
template <int LC, bool SEQ> M2_DEV Map<SEQ> scan_up(Map<SEQ> m, int lane) {
#pragma unroll
    for (int o = LC; o < 64; o <<= 1) {
        const Map<SEQ> e{__shfl_up(m.P, o), __shfl_up(m.H, o)};
        if (lane >= o) m = m.after(e);
    }
    return m;
}
template <int LC, bool SEQ> M2_DEV Map<SEQ> scan_down(Map<SEQ> m, int lane) {
#pragma unroll
    for (int o = LC; o < 64; o <<= 1) {
        const Map<SEQ> e{__shfl_down(m.P, o), __shfl_down(m.H, o)};
        if (lane + o < 64) m = m.after(e);
    }
    return m;
}

template <typename T, int V, int LC, int TS, int W, bool SEQ>
__global__ void __launch_bounds__(W * 64) k_rec_forward(RecArgs a) {
    typedef Place<V, LC, TS, W> P;
    __shared__ float2 tot[2][W][P::C];
    const P at(a);
    const int lane = threadIdx.x & 63;
    const T* x = static_cast<const T*>(a.x) + at.b * a.xb + at.c;
    const T* r = static_cast<const T*>(a.r) + at.b * a.rb + at.c;
    const T* i = static_cast<const T*>(a.i) + at.b * a.ib + at.c;
    T* out = static_cast<T*>(a.out) + at.b * a.L * a.dim + at.c;
    const int32_t* seq = SEQ ? a.seq + at.b * a.L : nullptr;
    float A[V], h[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        A[v] = a.A[at.c + v];
        h[v] = a.h0 ? a.h0[(int64_t)at.b * a.dim + at.c + v] : 0.f;
    }
    Raw<T, V> nx[TS], nr[TS], ni[TS];
    Steps<TS, SEQ> ns, cs;
    auto load = [&](int64_t t0) {
        const int64_t t = t0 + at.step;
#pragma unroll
        for (int j = 0; j < TS; ++j) {
            const int64_t u = min(t + j, a.L - 1);
            nx[j].load(x + u * a.xt);
            nr[j].load(r + u * a.rt);
            ni[j].load(i + u * a.it);
        }
        ns.load(seq, t, a.L);
    };
    load(0);
    int buf = 0;
    for (int64_t t0 = 0; t0 < a.L; t0 += P::TILE, buf ^= 1) {
        const int64_t t = t0 + at.step;
        Raw<T, V> cx[TS], cr[TS], ci[TS];
#pragma unroll
        for (int j = 0; j < TS; ++j) { cx[j] = nx[j]; cr[j] = nr[j]; ci[j] = ni[j]; }
        cs = ns;
        if (t0 + P::TILE < a.L) load(t0 + P::TILE);
        cs.set(t, a.L);
        const bool masked = SEQ || t0 + P::TILE > a.L;
        // the gates, and the map of this thread's steps
        float al[TS][V], add[TS][V];
        Map<SEQ> m[V];
#pragma unroll
        for (int v = 0; v < V; ++v) {
            float S = 0.f, H = 0.f;
#pragma unroll
            for (int j = 0; j < TS; ++j) {
                float q = sigmoid(cr[j].get(v)), s = sigmoid(ci[j].get(v)), xv = cx[j].get(v);
                if (masked && !cs.is_live(j)) q = s = xv = 0.f;
                const float L = A[v] * q;
                al[j][v] = decay(L);
                float y;
                const float ib = inv_beta(al[j][v], y);
                add[j][v] = y * ib * s * xv;
                S += L;
                const float e = cs.clears(j) ? 0.f : H;
                H = step(al[j][v], e, add[j][v]);
            }
            m[v].P = SEQ && cs.clear ? -1.f : __builtin_amdgcn_exp2f(S * LOG2E);
            m[v].H = H;
        }
        Map<SEQ> ex[V];
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const Map<SEQ> in = scan_up<LC, SEQ>(m[v], lane);
            ex[v] = Map<SEQ>{__shfl_up(in.P, LC), __shfl_up(in.H, LC)};
            if (at.tg == 0) ex[v] = Map<SEQ>{1.f, 0.f};
            if (at.tg == P::G - 1) tot[buf][at.w][at.col + v] = make_float2(in.P, in.H);
        }
        lds_barrier();
        float e[V];
#pragma unroll
        for (int u = 0; u < W; ++u) {
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const float2 p = tot[buf][u][at.col + v];
                if (u == at.w) e[v] = h[v];
                h[v] = Map<SEQ>{p.x, p.y}.of(h[v]);
            }
        }
#pragma unroll
        for (int v = 0; v < V; ++v) e[v] = ex[v].of(e[v]);
        if (a.ck && t < a.L && t % SPAN == 0) {
            float* ck = a.ck + (at.b * a.spans + t / SPAN) * a.dim + at.c;
            put<float, V>(ck, e, at.skip);
        }
#pragma unroll
        for (int j = 0; j < TS; ++j) {
            float o[V];
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const float p = cs.clears(j) ? 0.f : e[v];
                e[v] = step(al[j][v], p, add[j][v]);
                o[v] = masked && !cs.is_live(j) ? 0.f : e[v];
            }
            if (t + j < a.L) put<T, V>(out + (t + j) * a.dim, o, at.skip);
        }
    }
    if (a.last && at.w == 0 && at.tg == 0) put<float, V>(a.last + (int64_t)at.b * a.dim + at.c, h, at.skip);
}

template <typename T, int V, int LC, int TS, int W, bool SEQ>
__global__ void __launch_bounds__(W * 64) k_rec_backward(RecArgs a) {
    typedef Place<V, LC, TS, W> P;
    static_assert(P::TILE % SPAN == 0, "");
    __shared__ float tot[2][3][W][P::C];
    const P at(a);
    const int lane = threadIdx.x & 63;
    const T* x = static_cast<const T*>(a.x) + at.b * a.xb + at.c;
    const T* r = static_cast<const T*>(a.r) + at.b * a.rb + at.c;
    const T* i = static_cast<const T*>(a.i) + at.b * a.ib + at.c;
    const T* g = static_cast<const T*>(a.g) + at.b * a.gb + at.c;
    const int64_t o0 = at.b * a.L * a.dim + at.c;
    T* dx = static_cast<T*>(a.dx) + o0;
    T* dr = static_cast<T*>(a.dr) + o0;
    T* di = static_cast<T*>(a.di) + o0;
    const int32_t* seq = SEQ ? a.seq + at.b * a.L : nullptr;
    const float* ck = a.ck + at.b * a.spans * a.dim + at.c;
    float A[V], mu[V], dA[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        A[v] = a.A[at.c + v];
        mu[v] = a.glast ? a.glast[(int64_t)at.b * a.dim + at.c + v] : 0.f;
        dA[v] = 0.f;
    }
    Raw<T, V> nx[TS], nr[TS], ni[TS], ng[TS];
    Raw<float, V> nk;
    Steps<TS, SEQ> ns, cs;
    auto load = [&](int64_t t0) {
        const int64_t t = t0 + at.step;
#pragma unroll
        for (int j = 0; j < TS; ++j) {
            const int64_t u = min(t + j, a.L - 1);
            nx[j].load(x + u * a.xt);
            nr[j].load(r + u * a.rt);
            ni[j].load(i + u * a.it);
            ng[j].load(g + u * a.gt);
        }
        nk.load(ck + t0 / SPAN * a.dim);
        ns.load(seq, t, a.L);
    };
    int64_t t0 = (a.L - 1) / P::TILE * P::TILE;
    load(t0);
    int buf = 0;
    for (; t0 >= 0; t0 -= P::TILE, buf ^= 1) {
        const int64_t t = t0 + at.step;
        Raw<T, V> cx[TS], cr[TS], ci[TS], cg[TS];
#pragma unroll
        for (int j = 0; j < TS; ++j) { cx[j] = nx[j]; cr[j] = nr[j]; ci[j] = ni[j]; cg[j] = ng[j]; }
        cs = ns;
        float e[V];
#pragma unroll
        for (int v = 0; v < V; ++v) e[v] = nk.get(v);
        if (t0 >= P::TILE) load(t0 - P::TILE);
        cs.set(t, a.L);
        const bool masked = SEQ || t0 + P::TILE > a.L;
        auto dead = [&](int j) { return masked && !cs.is_live(j); };
        float al[TS][V], q[TS][V], s[TS][V], ib[TS][V];
        Map<SEQ> m[V];
        float M[V];
#pragma unroll
        for (int v = 0; v < V; ++v) {
            float S = 0.f, H = 0.f;
#pragma unroll
            for (int j = 0; j < TS; ++j) {
                float xv = cx[j].get(v);
                q[j][v] = sigmoid(cr[j].get(v));
                s[j][v] = sigmoid(ci[j].get(v));
                if (dead(j)) q[j][v] = s[j][v] = xv = 0.f;
                const float L = A[v] * q[j][v];
                al[j][v] = decay(L);
                float y;
                ib[j][v] = inv_beta(al[j][v], y);
                S += L;
                const float p = cs.clears(j) ? 0.f : H;
                H = step(al[j][v], p, y * ib[j][v] * s[j][v] * xv);
            }
            m[v].P = SEQ && cs.clear ? -1.f : __builtin_amdgcn_exp2f(S * LOG2E);
            m[v].H = H;
            float k = 0.f;
#pragma unroll
            for (int j = TS - 1; j >= 0; --j) {
                const float l = (dead(j) ? 0.f : cg[j].get(v)) + k;
                k = cs.clears(j) ? 0.f : step(al[j][v], l, 0.f);
            }
            M[v] = k;
        }
        Map<SEQ> up[V], down[V];
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const Map<SEQ> f = scan_up<LC, SEQ>(m[v], lane), k = scan_down<LC, SEQ>(Map<SEQ>{m[v].P, M[v]}, lane);
            up[v] = Map<SEQ>{__shfl_up(f.P, LC), __shfl_up(f.H, LC)};
            down[v] = Map<SEQ>{__shfl_down(k.P, LC), __shfl_down(k.H, LC)};
            if (at.tg == 0) {
                up[v] = Map<SEQ>{1.f, 0.f};
                tot[buf][0][at.w][at.col + v] = k.P;
                tot[buf][2][at.w][at.col + v] = k.H;
            }
            if (at.tg == P::G - 1) {
                down[v] = Map<SEQ>{1.f, 0.f};
                tot[buf][1][at.w][at.col + v] = f.H;
            }
        }
        lds_barrier();
        float k[V];
#pragma unroll
        for (int u = 0; u < W; ++u) {
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const int f = u, d = W - 1 - u;
                if (f < at.w) e[v] = Map<SEQ>{tot[buf][0][f][at.col + v], tot[buf][1][f][at.col + v]}.of(e[v]);
                if (d == at.w) k[v] = mu[v];
                mu[v] = Map<SEQ>{tot[buf][0][d][at.col + v], tot[buf][2][d][at.col + v]}.of(mu[v]);
            }
        }
        float lam[TS][V];
#pragma unroll
        for (int v = 0; v < V; ++v) {
            e[v] = up[v].of(e[v]);
            k[v] = down[v].of(k[v]);
#pragma unroll
            for (int j = TS - 1; j >= 0; --j) {
                lam[j][v] = (dead(j) ? 0.f : cg[j].get(v)) + k[v];
                k[v] = cs.clears(j) ? 0.f : step(al[j][v], lam[j][v], 0.f);
            }
        }
#pragma unroll
        for (int j = 0; j < TS; ++j) {
            float ox[V], orr[V], oi[V];
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const bool off = dead(j);
                const float xv = off ? 0.f : cx[j].get(v), p = cs.clears(j) ? 0.f : e[v];
                const float av = 1.f - al[j][v], beta = al[j][v] * (2.f - al[j][v]) * ib[j][v];
                const float sx = s[j][v] * xv;
                e[v] = step(al[j][v], p, beta * sx);
                ox[v] = lam[j][v] * beta * s[j][v];
                const float dL = lam[j][v] * av * (p - av * ib[j][v] * sx);
                oi[v] = off ? 0.f : ox[v] * xv * co_sigmoid(ci[j].get(v), s[j][v]);
                orr[v] = off ? 0.f : dL * (A[v] * q[j][v]) * co_sigmoid(cr[j].get(v), q[j][v]);
                dA[v] = fmaf(dL, q[j][v], dA[v]);
            }
            if (t + j < a.L) {
                put<T, V>(dx + (t + j) * a.dim, ox, at.skip);
                put<T, V>(dr + (t + j) * a.dim, orr, at.skip);
                put<T, V>(di + (t + j) * a.dim, oi, at.skip);
            }
        }
    }
    const int64_t row = (int64_t)at.b * a.dim + at.c;
    if (a.dh0 && at.w == 0 && at.tg == 0) put<float, V>(a.dh0 + row, mu, at.skip);
    // dA of this row: of the lanes of a channel, then of the wavefronts in their order
    lds_barrier();
#pragma unroll
    for (int v = 0; v < V; ++v) {
#pragma unroll
        for (int o = LC; o < 64; o <<= 1) dA[v] += __shfl_xor(dA[v], o);
        if (at.tg == 0) tot[0][0][at.w][at.col + v] = dA[v];
    }
    lds_barrier();
    if (at.w == 0 && at.tg == 0) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
            dA[v] = 0.f;
#pragma unroll
            for (int u = 0; u < W; ++u) dA[v] += tot[0][0][u][at.col + v];
        }
        put<float, V>(a.dA + row, dA, at.skip);
    }
}

// dA of the batch rows, in their order
__global__ void __launch_bounds__(64) k_rec_join(const float* part, float* dA, int64_t batch, int64_t dim) {
    const int64_t c = (int64_t)blockIdx.x * 64 + threadIdx.x;
    if (c >= dim) return;
    double s = 0;
#pragma unroll 8
    for (int64_t b = 0; b < batch; ++b) s += part[b * dim + c];
    dA[c] = (float)s;
}

// no steps: the state stays, and so does its gradient
__global__ void __launch_bounds__(256) k_rec_nothing(const float* from, float* to, int64_t n) {
    for (int64_t k = (int64_t)blockIdx.x * 256 + threadIdx.x; k < n; k += (int64_t)gridDim.x * 256)
        to[k] = from ? from[k] : 0.f;
}

// one step of every row
struct StepArgs {
    const void *x, *r, *i;
    const float *A, *state;
    float* next;
    void* out;
    int64_t xb, rb, ib;
    int dim;
};
template <typename T> __global__ void __launch_bounds__(64) k_rec_step(StepArgs a) {
    const int64_t b = blockIdx.y;
    const int c = blockIdx.x * 64 + threadIdx.x;
    if (c >= a.dim) return;
    const float q = sigmoid(to_f32(static_cast<const T*>(a.r)[b * a.rb + c]));
    const float s = sigmoid(to_f32(static_cast<const T*>(a.i)[b * a.ib + c]));
    const float xv = to_f32(static_cast<const T*>(a.x)[b * a.xb + c]), e = a.state[b * a.dim + c];
    const float al = decay(a.A[c] * q);
    float y;
    const float ib = inv_beta(al, y);
    const float h = step(al, e, y * ib * s * xv);
    a.next[b * a.dim + c] = h;
    static_cast<T*>(a.out)[b * a.dim + c] = from_f32<T>(h);
}

// ---------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------
template <typename T, int V, int LC, int TS, int W> void launch(RecArgs a, int64_t batch, bool back, hipStream_t s) {
    a.slabs = (a.dim + V * LC - 1) / (V * LC);
    const dim3 grid((unsigned)(batch * a.slabs)), block(W * 64);
    auto go = [&](auto k) { hipLaunchKernelGGL(k, grid, block, 0, s, a); };
    if (back) {
        if (a.seq) go(k_rec_backward<T, V, LC, TS, W, true>);
        else go(k_rec_backward<T, V, LC, TS, W, false>);
    } else {
        if (a.seq) go(k_rec_forward<T, V, LC, TS, W, true>);
        else go(k_rec_forward<T, V, LC, TS, W, false>);
    }
}
template <typename T> void run(const RecArgs& a, int64_t batch, bool back, hipStream_t s) {
    if (a.dim < 4) launch<T, 1, 4, 4, 4>(a, batch, back, s);
    else launch<T, 4, 16, 4, 4>(a, batch, back, s);
}

// what a call may ask for, whichever it is
int check_sizes(const char* who, int64_t batch, int64_t seqlen, int64_t dim, int dtype) {
    M2_REQUIRE(batch >= 0 && seqlen >= 0 && dim > 0 && dim < (1 << 30) && seqlen < (1ll << 40), M2_ERR_INVALID,
               "%s: bad sizes (batch %lld, seqlen %lld, dim %lld)", who, (long long)batch, (long long)seqlen,
               (long long)dim);
    M2_REQUIRE(dtype == M2_F32 || dtype == M2_BF16, M2_ERR_UNSUPPORTED, "%s: dtype %d", who, dtype);
    // (workgroups of the narrowest slabs)
    M2_REQUIRE(batch < (1ll << 30) && batch * ((dim + 3) / 4) < (1ll << 31), M2_ERR_UNSUPPORTED, "%s: too many rows", who);
    return M2_OK;
}

}  // namespace

namespace m2 {

int launch_gated_recurrence(const m2_gated_recurrence_args& a, hipStream_t s) {
    const char* who = "gated_linear_recurrence";
    if (int rc = check_sizes(who, a.batch, a.seqlen, a.dim, a.dtype)) return rc;
    const bool some = a.batch && a.seqlen;
    M2_REQUIRE(!some || (a.x && a.r && a.i && a.A && a.out), M2_ERR_INVALID, "%s: x, r, i, A and out are required", who);
    if (!some) {
        const int64_t n = a.batch * a.dim;
        if (n && a.final_states)
            hipLaunchKernelGGL(k_rec_nothing, dim3((unsigned)(n < 65536 ? (n + 255) / 256 : 256)), dim3(256), 0, s,
                               a.initial_states, a.final_states, n);
        return check_launch(who);
    }
    RecArgs k{};
    k.x = a.x; k.r = a.r; k.i = a.i; k.A = a.A; k.h0 = a.initial_states; k.seq = a.seq_idx;
    k.xb = a.x_stride_batch; k.xt = a.x_stride_time;
    k.rb = a.r_stride_batch; k.rt = a.r_stride_time;
    k.ib = a.i_stride_batch; k.it = a.i_stride_time;
    k.ck = a.span_states; k.L = a.seqlen; k.spans = (a.seqlen + SPAN - 1) / SPAN; k.dim = (int)a.dim;
    k.out = a.out; k.last = a.final_states;
    if (a.dtype == M2_F32) run<float>(k, a.batch, false, s);
    else run<bf16>(k, a.batch, false, s);
    return check_launch(who);
}

size_t gated_recurrence_grad_workspace(const m2_gated_recurrence_grad_args& a) {
    if (check_sizes("gated_linear_recurrence_grad", a.batch, a.seqlen, a.dim, a.dtype)) return 0;
    return 4 * (size_t)(a.batch > 1 ? a.batch : 1) * a.dim;
}

int launch_gated_recurrence_grad(const m2_gated_recurrence_grad_args& a, hipStream_t s) {
    const char* who = "gated_linear_recurrence_grad";
    if (int rc = check_sizes(who, a.batch, a.seqlen, a.dim, a.dtype)) return rc;
    M2_REQUIRE(a.batch > 0 && a.seqlen > 0, M2_ERR_INVALID, "%s: no steps", who);
    M2_REQUIRE(a.x && a.r && a.i && a.A && a.span_states && a.grad_out && a.grad_x && a.grad_r && a.grad_i && a.grad_A,
               M2_ERR_INVALID, "%s: x, r, i, A, span_states, grad_out and the gradients are required", who);
    const size_t need = gated_recurrence_grad_workspace(a);
    M2_REQUIRE(a.workspace && a.workspace_bytes >= need, M2_ERR_WORKSPACE,
               "%s: workspace of %zu bytes needed, %zu given", who, need, a.workspace_bytes);
    RecArgs k{};
    k.x = a.x; k.r = a.r; k.i = a.i; k.A = a.A; k.seq = a.seq_idx;
    k.xb = a.x_stride_batch; k.xt = a.x_stride_time;
    k.rb = a.r_stride_batch; k.rt = a.r_stride_time;
    k.ib = a.i_stride_batch; k.it = a.i_stride_time;
    k.ck = const_cast<float*>(a.span_states);
    k.L = a.seqlen; k.spans = (a.seqlen + SPAN - 1) / SPAN; k.dim = (int)a.dim;
    k.g = a.grad_out; k.gb = a.grad_out_stride_batch; k.gt = a.grad_out_stride_time;
    k.glast = a.grad_final_states;
    k.dx = a.grad_x; k.dr = a.grad_r; k.di = a.grad_i; k.dh0 = a.grad_initial_states;
    k.dA = a.batch == 1 ? a.grad_A : static_cast<float*>(a.workspace);
    if (a.dtype == M2_F32) run<float>(k, a.batch, true, s);
    else run<bf16>(k, a.batch, true, s);
    if (a.batch > 1)
        hipLaunchKernelGGL(k_rec_join, dim3((unsigned)((a.dim + 63) / 64)), dim3(64), 0, s, k.dA, a.grad_A, a.batch, a.dim);
    return check_launch(who);
}

int launch_gated_recurrence_update(const m2_gated_recurrence_update_args& a, hipStream_t s) {
    const char* who = "gated_linear_recurrence_update";
    if (int rc = check_sizes(who, a.batch, 1, a.dim, a.dtype)) return rc;
    M2_REQUIRE(a.batch <= 65535, M2_ERR_UNSUPPORTED, "%s: batch %lld", who, (long long)a.batch);
    M2_REQUIRE(a.batch == 0 || (a.x && a.r && a.i && a.A && a.state && a.new_state && a.out), M2_ERR_INVALID,
               "%s: x, r, i, A, state, new_state and out are required", who);
    if (a.batch == 0) return M2_OK;
    const StepArgs k{a.x, a.r, a.i, a.A, a.state, a.new_state, a.out, a.x_stride_batch, a.r_stride_batch,
                     a.i_stride_batch, (int)a.dim};
    const dim3 grid((unsigned)((a.dim + 63) / 64), (unsigned)a.batch);
    if (a.dtype == M2_F32) hipLaunchKernelGGL(k_rec_step<float>, grid, dim3(64), 0, s, k);
    else hipLaunchKernelGGL(k_rec_step<bf16>, grid, dim3(64), 0, s, k);
    return check_launch(who);
}

}  // namespace m2
