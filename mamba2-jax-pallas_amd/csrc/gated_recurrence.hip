// The gated linear recurrence over time and its gradient: independent per channel,
//
//   q = sigmoid(r), s = sigmoid(i), log a = A q (A <= 0), beta = sqrt(1 - a^2)
//   h[t] = a h[t-1] + beta s x[t]
//   l[t] = g[t] + m[t+1], m[t] = a l[t]        (l: the gradient of h[t], m: what of it goes on)
//   dx = l beta s;  di = dx x (1 - s);  dL = l (a h[t-1] - a^2 / beta s x);  dr = dL A q (1 - q)
//   dA = sum dL q;  dh0 = m[0]
//
// A thread runs TS consecutive steps of V channels; a run of steps is an affine map h -> P h + H, and the maps of the
// threads of a wavefront (by lane shifts) and then of the wavefronts (by LDS) are joined to the state that each thread's run
// begins with.  A workgroup has 64 channels, so that a step of a bf16 stream is a whole line of 128 bytes.
//
// Forward: bound by bytes, three streams read and one written, and nearly by vector instructions (41 to 45 an element, five of
// them exponentials, reciprocals and roots).  Workgroups take a segment each of a row's length, hold it in registers, and
// pass the states on between them, so that every input is read and every gate computed once, with the whole chip
// busy on a single row: 16384 x 2560 bf16 77 us (336 MB, 4.4 TB/s; 85-94 with the clearing before it, where a pass of its own
// for the states takes 119, and all of a slab by one workgroup 580), 8 x 2048 x 5120 147-161 us (671 MB, 4.2 to 4.6 TB/s).
// It leaves the state that enters every span of 32 steps (float32, a sixteenth of a bf16 stream) for the backward.
//
// Backward: a workgroup walks from the last tile to the first, three tiles in flight, computes the states of a tile again
// from the span's and joins both directions at once (a run's map backward, m -> P m + M, has the same P).  Where there are few
// slabs a first pass finds what enters the segments of each; where there are more than run at once, segments pass it on.
// 74 vector instructions and 14 bytes an element: 8 x 2048 x 5120 296-337 us (1216 MB, 3.6 to 4.1 TB/s: the kernel of one call
// after the other under a trace), 8 x 2048 x 4096, whose 512 slabs run at once, 255 with its join (973 MB, 3.8 TB/s).
//
// Everything is float32 but what is loaded and stored.  Where log a >= NEAR alpha = 1 - a is kept in place of a: near
// 1, where memories are long, a itself has too few bits (beta^2 = alpha (2 - alpha) loses none,
// and h - alpha h + b rounds by the step's own size only).  Below NEAR a itself is, for there 1 - a has lost its bits, and
// h + b would round what is added at the size of a state that is about to go.  Wavefronts with a channel whose A is below
// NEAR (FAR) take either form step by step; the others need the first alone.
//
// Where seq_idx changes the state is cleared: P = -1 marks a run that holds such a step, so that what
// came before (a NaN, say) is selected away and not multiplied by zero.  Negative seq_idx is
// padding: a = 1, nothing added, 0 stored; so are the steps past the end of the row.
#include <type_traits>

#include "m2_internal.h"

namespace {

constexpr float LOG2E = 1.4426950408889634f;
constexpr int SPAN = M2_RECURRENCE_SPAN;

// Buffer accesses: a scalar descriptor of what may be touched (from a base on, so many bytes), a 32-bit
// offset of the lane, one of the wavefront.  A step's address takes no vector instruction, and
// what lies past the end reads 0 and is not stored.  Addresses need be aligned as elements only.
typedef __amdgpu_buffer_rsrc_t Rsrc;
M2_DEV Rsrc rsrc(const void* p, uint32_t bytes) { return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, bytes, 0x00027000); }
constexpr uint32_t NOWHERE = 0xfffffff0u;      // an offset past every end

// V consecutive channels of a row, as loaded
template <typename T, int V> struct Raw;
template <> struct Raw<bf16, 2> {
    uint32_t v;
    M2_DEV void load(Rsrc r, uint32_t off, uint32_t soff) { v = __builtin_amdgcn_raw_buffer_load_b32(r, off, soff, 0); }
    M2_DEV void fill(float f) { v = pk_bf16(f, f); }
    M2_DEV float get(int i) const { return i ? bf16_hi(v) : bf16_lo(v); }
    template <int AUX> static M2_DEV void store(Rsrc r, uint32_t off, uint32_t soff, const float (&f)[2]) {
        __builtin_amdgcn_raw_buffer_store_b32(pk_bf16(f[0], f[1]), r, off, soff, AUX);
    }
};
template <> struct Raw<float, 2> {
    typedef uint32_t pair __attribute__((ext_vector_type(2)));
    pair v;
    M2_DEV void load(Rsrc r, uint32_t off, uint32_t soff) { v = __builtin_amdgcn_raw_buffer_load_b64(r, off, soff, 0); }
    M2_DEV void fill(float f) { v[0] = v[1] = __float_as_uint(f); }
    M2_DEV float get(int i) const { return __uint_as_float(v[i]); }
    template <int AUX> static M2_DEV void store(Rsrc r, uint32_t off, uint32_t soff, const float (&f)[2]) {
        __builtin_amdgcn_raw_buffer_store_b64(pair{__float_as_uint(f[0]), __float_as_uint(f[1])}, r, off, soff, AUX);
    }
};
template <> struct Raw<bf16, 1> {
    uint32_t v;
    M2_DEV void load(Rsrc r, uint32_t off, uint32_t soff) {
        v = (uint32_t)(uint16_t)__builtin_amdgcn_raw_buffer_load_b16(r, off, soff, 0) << 16;
    }
    M2_DEV void fill(float f) { v = __float_as_uint(f); }
    M2_DEV float get(int) const { return __uint_as_float(v); }
    template <int AUX> static M2_DEV void store(Rsrc r, uint32_t off, uint32_t soff, const float (&f)[1]) {
        __builtin_amdgcn_raw_buffer_store_b16((uint16_t)pk_bf16(f[0], f[0]), r, off, soff, AUX);
    }
};
template <> struct Raw<float, 1> {
    uint32_t v;
    M2_DEV void load(Rsrc r, uint32_t off, uint32_t soff) { v = __builtin_amdgcn_raw_buffer_load_b32(r, off, soff, 0); }
    M2_DEV void fill(float f) { v = __float_as_uint(f); }
    M2_DEV float get(int) const { return __uint_as_float(v); }
    template <int AUX> static M2_DEV void store(Rsrc r, uint32_t off, uint32_t soff, const float (&f)[1]) {
        __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(f[0]), r, off, soff, AUX);
    }
};

constexpr float INF = __builtin_inff();

// exp(-v), sigmoid(v) from it, and 1 - sigmoid(v), which keeps its bits where the sigmoid is near 1
M2_DEV float exp_neg(float v) { return __builtin_amdgcn_exp2f(v * -LOG2E); }
M2_DEV float sigmoid_of(float e) { return __builtin_amdgcn_rcpf(1.f + e); }
M2_DEV float co_sigmoid(float e, float s) { return e <= 1.f ? e * s : 1.f - s; }
// 1 - exp(L) from NEAR on, where 1 - exp would cancel: -L times a polynomial of degree 5, found by Remez's exchange and rounded
// to float32 with its constant at 1.  As it stands its relative error is 2^-27.1 at most (at NEAR), and 2^-23.3 with the
// roundings of its evaluation, as the series to L^8 / 8! has in two instructions more.
constexpr float NEAR = -0.5f;
M2_DEV float decay_near(float L) {
    float p = 0x1.2607a4p-10f;
    p = fmaf(p, L, 0x1.0c48c6p-7f);
    p = fmaf(p, L, 0x1.550688p-5f);
    p = fmaf(p, L, 0x1.555304p-3f);
    p = fmaf(p, L, 0x1.fffff4p-2f);
    p = fmaf(p, L, 1.f);
    return p * -L;
}
// What a, and a product of them, is at least: never 0, whose sign would tell nothing, and of which an infinite state would make
// a NaN
constexpr float LEAST = 0x1p-149f;
M2_DEV float at_least(float p) { return __builtin_amdgcn_fmed3f(p, LEAST, 1.f); }
// What is kept of a step's decay a = exp(L): k = alpha = 1 - a >= 0, or (of FAR, where L < NEAR) -a < 0; and y = 1 - a^2
M2_DEV void decay(float L, float& k, float& y) {
    k = decay_near(L);
    y = k * (2.f - k);
}
M2_DEV void decay_far(float L, float& k, float& y) {
    const float a = at_least(__builtin_amdgcn_exp2f(L * LOG2E));
    k = L < NEAR ? -a : k;
    y = L < NEAR ? fmaf(-a, a, 1.f) : y;
}
// of the steps of a thread; far: of some channel of the wavefront an L may be below NEAR
template <int TS, int V> M2_DEV void decays(const float (&L)[TS][V], bool far, float (&k)[TS][V], float (&y)[TS][V]) {
#pragma unroll
    for (int j = 0; j < TS; ++j)
#pragma unroll
        for (int v = 0; v < V; ++v) decay(L[j][v], k[j][v], y[j][v]);
    if (!far) return;
    asm volatile("");        // (a branch, not selects: the exponentials cost the others an eighth of their time)
#pragma unroll
    for (int j = 0; j < TS; ++j)
#pragma unroll
        for (int v = 0; v < V; ++v) decay_far(L[j][v], k[j][v], y[j][v]);
}
// f of either kind of steps: what the wavefronts without the second compute stays without selects (8 x 2048 x 5120: forward 161
// and, with selects, 170 us, backward 304 and 326; both ways of the whole kernels instead of these parts of them hold 123
// registers for 78)
template <class F> M2_DEV void by_decay(bool far, F&& f) {
    if (far) {
        asm volatile("; far");
        f(std::true_type());
    } else {
        asm volatile("; near");
        f(std::false_type());
    }
}
// A channel's A: one above 0 is no decay, and makes NaNs
M2_DEV float decay_rate(float A) { return A > 0.f ? __builtin_nanf("") : A; }
// alpha p, of an infinite p the largest number (p - alpha p is then p, not inf - inf)
M2_DEV float bounded(float p) {
    constexpr float MAX = 3.402823466e38f;
    return __builtin_amdgcn_fmed3f(p, -MAX, MAX);
}
// Of what is kept, k: a; a p; a p + b; a P of a map, whose P is finite
template <bool FAR> M2_DEV float factor(float k) { return FAR && k < 0.f ? -k : 1.f - k; }
template <bool FAR> M2_DEV float step(float k, float p) { return FAR && k < 0.f ? -k * p : fmaf(-k, bounded(p), p); }
template <bool FAR> M2_DEV float step(float k, float p, float b) {
    return FAR && k < 0.f ? fmaf(-k, p, b) : fmaf(-k, bounded(p), p + b);
}
// (the runs of steps with k > 0 are too short to end at 0)
template <bool FAR> M2_DEV float shrunk(float k, float P) { return FAR && k < 0.f ? at_least(-k * P) : fmaf(-k, P, P); }
// 1 / sqrt(y), y = 1 - a^2; 0 where a is 1 (below 1e-37 the hardware's root has no argument left)
M2_DEV float inv_beta(float y) { return fabsf(y) <= 1e-37f ? 0.f : __builtin_amdgcn_rsqf(y); }

// an affine map v -> P v + H; P = -1: the state is cleared in it, v -> H.  A product of many a's would end at 0,
// of which an infinite v makes a NaN: no P is less than LEAST (which adds 5e-7 at most, of the largest v).
template <bool SEQ> struct Map {
    float P, H;
    M2_DEV float of(float v) const { return SEQ && P < 0.f ? H : fmaf(P, v, H); }
    // this one behind `first`
    M2_DEV Map after(const Map& first) const {
        Map m;
        m.H = of(first.H);
        m.P = at_least(P * first.P);
        if constexpr (SEQ) m.P = P < 0.f || first.P < 0.f ? -1.f : m.P;
        return m;
    }
};

constexpr int TICKET = 32;       // a counter's line, in ints
struct RecArgs {
    const void *x, *r, *i;
    const float *A, *h0;
    const int32_t* seq;
    int64_t xb, xt, rb, rt, ib, it;      // strides of batch and time
    float* ck;                           // [batch][spans][dim]
    int64_t L, spans;
    int dim, slabs, segments;
    int chains;                          // slabs of all rows
    int* tickets;                        // [chains] at TICKET: how many segments went out, less one
    uint32_t* states;                    // [batch][segments][dim]: what each passes on
    // forward
    uint64_t* maps;                      // [batch][segments][dim]: (P, H) of each
    void* out;
    float* last;
    // backward
    int64_t seg;                         // steps of a segment: whole tiles
    float2* agg;                         // [batch][segments][dim]: (P, M) of each
    const void* g;
    int64_t gb, gt;
    const float* glast;
    void *dx, *dr, *di;
    float* dA;                           // [batch][segments][dim]
    float* dh0;
};

// Which channels and steps of a tile a thread has
template <int V, int LC, int TS, int W> struct Place {
    static constexpr int G = 64 / LC, TILE = G * W * TS, C = V * LC;
    int b, segment, c, col, tg, w, step, lane, slab;       // col: place in the slab, which begins at channel slab
    int64_t t0, end;                     // of the segment
    // A lane that would reach past the last channel has the last V, and stores of them those that no other lane
    // has: all (whole), the second alone (half, of an odd number of channels), none
    bool whole, half;
    // segment `seg` of a chain, of so many steps
    M2_DEV Place(const RecArgs& a, int chain, int seg, int64_t steps) { init(a, chain, seg, steps); }
    // Of the grid of segments that are independent: neighbouring slabs to one XCD where there is one segment (8 x 2048 x 5120
    // 332 us so, 355 in turn), to all in turn where there are more (3 x 4096 x 5120 310 and 292)
    M2_DEV Place(const RecArgs& a) {
        const int id = a.segments == 1 ? xcd_remap(blockIdx.x, gridDim.x) : blockIdx.x;
        const int of = __builtin_amdgcn_readfirstlane(id / a.slabs), row = of / a.segments;
        init(a, row * a.slabs + id - of * a.slabs, of - row * a.segments, a.seg);
    }
    M2_DEV void init(const RecArgs& a, int chain, int seg, int64_t steps) {
        lane = threadIdx.x & 63;
        b = __builtin_amdgcn_readfirstlane(chain / a.slabs);
        segment = seg;
        t0 = segment * steps;
        end = min(t0 + steps, a.L);
        w = wave_id();
        col = (lane % LC) * V;
        tg = lane / LC;
        slab = (chain - b * a.slabs) * C;
        const int from = slab + col;
        c = min(from, a.dim - V);
        whole = from == c;
        half = V == 2 && from == c + 1;
        step = (w * G + tg) * TS;
    }
    M2_DEV bool owns(int v) const { return whole || (half && v == V - 1); }
    template <typename E> M2_DEV void put(E* p, const E (&f)[V]) const {
#pragma unroll
        for (int v = 0; v < V; ++v)
            if (owns(v)) p[v] = f[v];
    }
    M2_DEV int64_t agg(const RecArgs& a, int s) const { return ((int64_t)b * a.segments + s) * a.dim + c; }
};

// A of a thread's channels -> whether some channel of the wavefront has one below NEAR (or a NaN)
template <int V, class P> M2_DEV bool decay_rates(const RecArgs& a, const P& at, float (&A)[V]) {
    bool far = false;
#pragma unroll
    for (int v = 0; v < V; ++v) {
        A[v] = decay_rate(a.A[at.c + v]);
        far |= !(A[v] >= NEAR);
    }
    return __any(far);
}

// The tile of one input or output that the walk is at
template <typename T, int V> struct Stream {
    const char* base;        // of the tile's first step
    uint32_t st, row;        // bytes between steps, of a row
    uint32_t off;            // of the lane's first step
    template <class P> M2_DEV Stream(const void* p, int64_t offset, int64_t stride, const RecArgs& a, const P& at)
        : base(static_cast<const char*>(p) + offset * (int64_t)sizeof(T)), st((uint32_t)(stride * sizeof(T))),
          row(a.dim * (uint32_t)sizeof(T)), off(at.step * st + at.c * (uint32_t)sizeof(T)) {}
    M2_DEV void move(int64_t steps) { base += steps * st; }
    // last: the row's last step, counted from the tile's first
    M2_DEV Rsrc tile(int last) const { return rsrc(base, last * st + row); }
    template <int TS> M2_DEV void load(Raw<T, V> (&r)[TS], int last) const {
        const Rsrc t = tile(last);
#pragma unroll
        for (int j = 0; j < TS; ++j) r[j].load(t, off, j * st);
    }
};
// NT: past the caches (buffer accesses' nt bit)
template <typename T, int V, bool NT> struct Output : Stream<T, V> {
    static constexpr int AUX = NT ? 2 : 0;
    uint32_t whole, half;    // where this lane stores all of its channels, or the last alone
    bool odd;
    template <class P> M2_DEV Output(const void* p, int64_t offset, const RecArgs& a, const P& at)
        : Stream<T, V>(p, offset, a.dim, a, at), whole(at.whole ? this->off : NOWHERE),
          half(at.half ? this->off + (uint32_t)sizeof(T) : NOWHERE), odd(V == 2 && (a.dim & 1)) {}
    M2_DEV void store(Rsrc t, int j, const float (&f)[V]) const {
        Raw<T, V>::template store<AUX>(t, whole, j * this->st, f);
        if (odd) {
            const float one[1] = {f[V - 1]};
            Raw<T, 1>::template store<AUX>(t, half, j * this->st, one);
        }
    }
};

// The steps of a tile that a thread has: bit j of live: inside the row and no padding; of clear: the
// state is cleared before it.  Lane l holds seq_idx of the wavefront's step l - 1 (one load for all its
// steps); ballots make the bits of them.
template <int TS, int G, bool SEQ> struct Steps {
    static constexpr int N = G * TS;     // of a wavefront
    static_assert(!SEQ || N < 32, "");
    int sq;
    uint32_t live, clear;
    // row: of the tile's first step; begins: that is the row's first
    template <class P> M2_DEV void load(const int32_t* row, bool begins, const P& at, int last) {
        if constexpr (SEQ) {
            const int more = begins ? 0 : 1;                 // the step before the tile is read too
            const Rsrc t = rsrc(row - more, 4 * (last + 1 + more));
            sq = __builtin_amdgcn_raw_buffer_load_b32(t, 4 * max(at.w * N + min(at.lane, N) - 1 + more, 0), 0, 0);
        }
    }
    // -> whether all steps of the wavefront are live
    template <class P> M2_DEV bool set(bool begins, const P& at, int last) {
        const int first = at.w * N, in = min(max(last + 1 - first, 0), N);       // the wavefront's steps inside the row
        uint32_t l = (1u << in) - 1, c = 0;
        if constexpr (SEQ) {
            int before;
            if constexpr (N < 16) before = __builtin_amdgcn_update_dpp(0, sq, 0x111, 0xf, 0xf, true);      // row_shr:1
            else before = __shfl_up(sq, 1);
            l &= (uint32_t)(__ballot(sq >= 0) >> 1);
            c = l & (uint32_t)(__ballot(sq != before) >> 1);
            if (begins && first == 0) c &= ~1u;
        }
        live = l >> (at.tg * TS);
        clear = (c >> (at.tg * TS)) & ((1u << TS) - 1);
        return l == (1u << N) - 1;
    }
    M2_DEV bool is_live(int j) const { return live >> j & 1; }
    M2_DEV bool clears(int j) const { return SEQ && (clear >> j & 1); }
};

// The maps of the lanes of each channel, joined in the order of their steps: m becomes the inclusive one,
// the exclusive one is returned.  D: 1 from the first step on, -1 from the last back.  (A lane's shift goes through the LDS pipe,
// which is idle; lanes without another one read any.)
template <int D, int O, bool SEQ> M2_DEV Map<SEQ> shifted(const Map<SEQ>& m, int lane) {
    const int from = (lane - D * O) * 4;
    return Map<SEQ>{__int_as_float(__builtin_amdgcn_ds_bpermute(from, __float_as_int(m.P))),
                    __int_as_float(__builtin_amdgcn_ds_bpermute(from, __float_as_int(m.H)))};
}
template <int D, int LC, int O, bool SEQ> M2_DEV void join(Map<SEQ>& m, int lane) {
    if constexpr (O < 64) {
        const Map<SEQ> e = shifted<D, O, SEQ>(m, lane), j = m.after(e);
        const bool has = D > 0 ? lane >= O : lane + O < 64;
        m.P = has ? j.P : m.P;
        m.H = has ? j.H : m.H;
        join<D, LC, 2 * O, SEQ>(m, lane);
    }
}
template <int D, int LC, bool SEQ> M2_DEV Map<SEQ> scan(Map<SEQ>& m, int lane) {
    join<D, LC, LC, SEQ>(m, lane);
    const Map<SEQ> e = shifted<D, LC, SEQ>(m, lane);
    const bool has = D > 0 ? lane >= LC : lane + LC < 64;
    return Map<SEQ>{has ? e.P : 1.f, has ? e.H : 0.f};
}

// ---------------------------------------------------------------------------
// forward
// ---------------------------------------------------------------------------
// A workgroup's segment is one tile, held in registers.  A segment's map needs its own inputs alone; the state that enters it
// is the one of an earlier segment of the chain (a row's slab of channels), carried on by the maps between.  Both are
// published, and a segment waits until the states and maps of the W segments before it reach its start.
//
// Every wait ends: segments are given out by the chain's counter, so whoever waits for a segment knows that its workgroup
// is running, and of those that run the first in its chain waits for nobody.  Equal inputs give equal bits: from whichever
// state it starts, a segment applies the same maps to it in the same order.
constexpr uint32_t UNKNOWN = 0xffffffffu;    // a NaN's bits; what is published has NaNs of one other kind
M2_DEV uint32_t known(float f) { return f != f ? 0x7fc00000u : __float_as_uint(f); }
template <typename E> M2_DEV E peek(const E* p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
template <typename E> M2_DEV void publish(E* p, E v) { __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

// How many segments of the chain went out before; `next` is shared
M2_DEV int take(const RecArgs& a, int chain, int& next) {
    if (threadIdx.x == 0)
        next = __hip_atomic_fetch_add(a.tickets + chain * TICKET, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + 1;
    lds_barrier();
    return __builtin_amdgcn_readfirstlane(next);
}

// everything unknown, every counter at -1
__global__ void __launch_bounds__(256) k_rec_clear(u32x4* p, int64_t n) {
    for (int64_t k = (int64_t)blockIdx.x * 256 + threadIdx.x; k < n; k += (int64_t)gridDim.x * 256)
        p[k] = u32x4{UNKNOWN, UNKNOWN, UNKNOWN, UNKNOWN};
}

// The state that enters a segment.  Lanes stand for the slab's channels here, a wavefront w for the segment w + 1 before.
template <int V, bool SEQ, class P, int W> struct Enter {
    struct Shared {
        float2 map[2][W][P::C];
        uint32_t state[2][W][P::C];
        uint32_t near[P::C];             // the state behind the segment before, if it was known at the start
    };
    int l, ch;
    uint32_t early;
    M2_DEV int64_t index(const RecArgs& a, const P& at, int seg) const { return ((int64_t)at.b * a.segments + seg) * a.dim + ch; }
    M2_DEV uint32_t initial(const RecArgs& a, const P& at) const { return a.h0 ? known(a.h0[(int64_t)at.b * a.dim + ch]) : 0; }
    M2_DEV void begin(const RecArgs& a, const P& at) {
        l = at.lane % P::C;
        ch = min(at.slab + l, a.dim - 1);
        if (at.w == 0) early = at.segment > 0 ? peek(a.states + index(a, at, at.segment - 1)) : initial(a, at);
    }
    // before a barrier
    M2_DEV void meet(const P& at, Shared& s) const {
        if (at.w == 0) s.near[l] = early;
    }
    // behind it, in all wavefronts
    M2_DEV void end(const RecArgs& a, const P& at, Shared& s, float (&h)[V]) const {
        auto place = [&](int v) { return max(at.c - at.slab + v, 0); };      // (below 0: of a lane that stores nothing there)
        if (__all(s.near[l] != UNKNOWN)) {
#pragma unroll
            for (int v = 0; v < V; ++v) h[v] = __uint_as_float(s.near[place(v)]);
            return;
        }
        const int seg = at.segment - 1 - at.w;
        uint64_t m = ~0ull;
        uint32_t st = seg < 0 ? initial(a, at) : UNKNOWN;      // (before the row's start: nobody gets that far)
        int buf = 0;
        for (;; buf ^= 1) {
            if (seg >= 0) {
                st = peek(a.states + index(a, at, seg));
                m = peek(a.maps + index(a, at, seg));
            }
            s.map[buf][at.w][l] = make_float2(__uint_as_float((uint32_t)m), __uint_as_float((uint32_t)(m >> 32)));
            s.state[buf][at.w][l] = st;
            lds_barrier();
            // a state, and maps from there on
            bool found = false, gap = false;
#pragma unroll
            for (int k = 0; k < W; ++k) {
                const bool is = s.state[buf][k][l] != UNKNOWN;
                found |= is && !gap;
                gap |= !is && __float_as_uint(s.map[buf][k][l].x) == UNKNOWN;
            }
            if (__all(found)) break;             // (all wavefronts have read the same)
            __builtin_amdgcn_s_sleep(4);
        }
#pragma unroll
        for (int v = 0; v < V; ++v) {
            h[v] = 0.f;
#pragma unroll
            for (int k = W - 1; k >= 0; --k) {
                const uint32_t is = s.state[buf][k][place(v)];
                const float2 p = s.map[buf][k][place(v)];
                h[v] = is != UNKNOWN ? __uint_as_float(is) : Map<SEQ>{p.x, p.y}.of(h[v]);
            }
        }
    }
};

template <typename T, int V, int LC, int TS, int W, bool SEQ, bool NT>
__global__ void __launch_bounds__(W * 64, 4) k_rec_forward(RecArgs a) {
    typedef Place<V, LC, TS, W> P;
    typedef Enter<V, SEQ, P, W> E;
    __shared__ float2 tot[W][P::C];
    __shared__ typename E::Shared look;
    __shared__ int next;
    const int chain = blockIdx.x % a.chains;
    const int segment = a.segments > 1 ? take(a, chain, next) : 0;
    const P at(a, chain, segment, P::TILE);
    const bool ends = segment == a.segments - 1;
    E en;
    en.begin(a, at);
    const Stream<T, V> sx(a.x, at.b * a.xb + at.t0 * a.xt, a.xt, a, at), sr(a.r, at.b * a.rb + at.t0 * a.rt, a.rt, a, at),
        si(a.i, at.b * a.ib + at.t0 * a.it, a.it, a, at);
    const Output<T, V, NT> so(a.out, (at.b * a.L + at.t0) * a.dim, a, at);
    const int last = (int)(at.end - 1 - at.t0);
    Raw<T, V> x[TS], r[TS], i[TS];
    Steps<TS, P::G, SEQ> s;
    sr.load(r, last);
    sx.load(x, last);
    si.load(i, last);
    s.load(SEQ ? a.seq + at.b * a.L + at.t0 : nullptr, segment == 0, at, last);
    float A[V];
    const bool far = decay_rates<V>(a, at, A);
    if ((SEQ || last != P::TILE - 1) && !s.set(segment == 0, at, last)) {
#pragma unroll
        for (int j = 0; j < TS; ++j)
            if (!s.is_live(j)) {             // a = 1, nothing added
                x[j].fill(0.f);
                r[j].fill(-INF);
                i[j].fill(0.f);
            }
    }
    // the gates, and the map of this thread's steps
    float k[TS][V], add[TS][V], L[TS][V];
#pragma unroll
    for (int j = 0; j < TS; ++j)
#pragma unroll
        for (int v = 0; v < V; ++v) L[j][v] = A[v] * sigmoid_of(exp_neg(r[j].get(v)));
    decays<TS, V>(L, far, k, add);
    Map<SEQ> m[V], ex[V];
#pragma unroll
    for (int j = 0; j < TS; ++j)
#pragma unroll
        for (int v = 0; v < V; ++v) add[j][v] = sigmoid_of(exp_neg(i[j].get(v))) * x[j].get(v) * __builtin_amdgcn_sqrtf(add[j][v]);
    by_decay(far, [&](auto is_far) {
        constexpr bool FAR = decltype(is_far)::value;
#pragma unroll
        for (int v = 0; v < V; ++v)
#pragma unroll
            for (int j = 0; j < TS; ++j) {
                m[v].P = j == 0 ? factor<FAR>(k[j][v]) : shrunk<FAR>(k[j][v], m[v].P);
                m[v].H = j == 0 ? add[j][v] : step<FAR>(k[j][v], s.clears(j) ? 0.f : m[v].H, add[j][v]);
            }
    });
#pragma unroll
    for (int v = 0; v < V; ++v) {
        if (SEQ && s.clear) m[v].P = -1.f;
        ex[v] = scan<1, LC, SEQ>(m[v], at.lane);
        if (at.tg == P::G - 1) tot[at.w][at.col + v] = make_float2(m[v].P, m[v].H);
    }
    en.meet(at, look);
    lds_barrier();
    auto of_wave = [&](int u, int v) {
        const float2 p = tot[u][at.col + v];
        return Map<SEQ>{p.x, p.y};
    };
    const bool one = at.w == 0 && at.tg == 0;
    Map<SEQ> all[V];             // of the segment
    if (one) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
            all[v] = of_wave(0, v);
#pragma unroll
            for (int u = 1; u < W; ++u) all[v] = of_wave(u, v).after(all[v]);
            if (!ends && at.owns(v))
                publish(a.maps + at.agg(a, segment) + v, (uint64_t)known(all[v].P) | (uint64_t)__float_as_uint(all[v].H) << 32);
        }
    }
    float h[V];
    en.end(a, at, look, h);
    if (one) {
        float o[V];
#pragma unroll
        for (int v = 0; v < V; ++v) {
            o[v] = all[v].of(h[v]);
            if (!ends && at.owns(v)) publish(a.states + at.agg(a, segment) + v, known(o[v]));
        }
        if (ends && a.last) at.put(a.last + (int64_t)at.b * a.dim + at.c, o);
    }
    for (int u = 0; u < at.w; ++u)
#pragma unroll
        for (int v = 0; v < V; ++v) h[v] = of_wave(u, v).of(h[v]);
#pragma unroll
    for (int v = 0; v < V; ++v) h[v] = ex[v].of(h[v]);
    if (a.ck && at.step % SPAN == 0 && at.step <= last)
        at.put(a.ck + (at.b * a.spans + (at.t0 + at.step) / SPAN) * a.dim + at.c, h);
    const Rsrc to = so.tile(last);
    by_decay(far, [&](auto is_far) {
        constexpr bool FAR = decltype(is_far)::value;
#pragma unroll
        for (int j = 0; j < TS; ++j) {
            float o[V];
#pragma unroll
            for (int v = 0; v < V; ++v) {
                h[v] = step<FAR>(k[j][v], s.clears(j) ? 0.f : h[v], add[j][v]);
                o[v] = SEQ && !s.is_live(j) ? 0.f : h[v];
            }
            so.store(to, j, o);
        }
    });
}

// ---------------------------------------------------------------------------
// backward
// ---------------------------------------------------------------------------
// The map of each segment but the first from its end back: of r and the upstream gradient alone
template <typename T, int V, int LC, int TS, int W, bool SEQ>
__global__ void __launch_bounds__(W * 64, 4) k_rec_back_agg(RecArgs a) {
    typedef Place<V, LC, TS, W> P;
    __shared__ float2 tot[3][W][P::C];
    const P at(a);
    if (at.segment == 0) return;
    const int64_t end = at.t0 + (at.end - 1 - at.t0) / P::TILE * P::TILE;
    Stream<T, V> sr(a.r, at.b * a.rb + end * a.rt, a.rt, a, at), sg(a.g, at.b * a.gb + end * a.gt, a.gt, a, at);
    const int32_t* seq = SEQ ? a.seq + at.b * a.L : nullptr;
    float A[V];
    Map<SEQ> mu[V];
#pragma unroll
    for (int v = 0; v < V; ++v) mu[v] = Map<SEQ>{1.f, 0.f};
    const bool far = decay_rates<V>(a, at, A);
    auto last_of = [&](int64_t t0) { return (int)min(at.end - 1 - t0, (int64_t)P::TILE - 1); };
    struct Tile {
        Raw<T, V> r[TS], g[TS];
        Steps<TS, P::G, SEQ> s;
    } one, two, three;
    auto load = [&](Tile& n, int64_t t0) {
        const int last = last_of(t0);
        sr.load(n.r, last);
        sg.load(n.g, last);
        n.s.load(seq + t0, t0 == 0, at, last);
        sr.move(-P::TILE);
        sg.move(-P::TILE);
    };
    auto tile = [&](Tile& c, Tile& n, int64_t t0, int buf) {
        const int last = last_of(t0);
        if (t0 - 2 * P::TILE >= at.t0) load(n, t0 - 2 * P::TILE);
        if ((SEQ || last != P::TILE - 1) && !c.s.set(t0 == 0, at, last)) {
#pragma unroll
            for (int j = 0; j < TS; ++j)
                if (!c.s.is_live(j)) {
                    c.r[j].fill(-INF);
                    c.g[j].fill(0.f);
                }
        }
        float kept[TS][V], y[TS][V], L[TS][V];
#pragma unroll
        for (int j = 0; j < TS; ++j)
#pragma unroll
            for (int v = 0; v < V; ++v) L[j][v] = A[v] * sigmoid_of(exp_neg(c.r[j].get(v)));
        decays<TS, V>(L, far, kept, y);
        Map<SEQ> k[V];
        by_decay(far, [&](auto is_far) {
            constexpr bool FAR = decltype(is_far)::value;
#pragma unroll
            for (int v = 0; v < V; ++v)
#pragma unroll
                for (int j = TS - 1; j >= 0; --j) {
                    k[v].P = j == TS - 1 ? factor<FAR>(kept[j][v]) : shrunk<FAR>(kept[j][v], k[v].P);
                    k[v].H = step<FAR>(kept[j][v], j == TS - 1 ? c.g[j].get(v) : c.g[j].get(v) + k[v].H);
                    if (c.s.clears(j)) k[v].H = 0.f;
                }
        });
#pragma unroll
        for (int v = 0; v < V; ++v) {
            if (SEQ && c.s.clear) k[v].P = -1.f;
            join<-1, LC, LC, SEQ>(k[v], at.lane);
            if (at.tg == 0) tot[buf][at.w][at.col + v] = make_float2(k[v].P, k[v].H);
        }
        lds_barrier();
#pragma unroll
        for (int u = W - 1; u >= 0; --u)
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const float2 p = tot[buf][u][at.col + v];
                mu[v] = Map<SEQ>{p.x, p.y}.after(mu[v]);
            }
    };
    load(one, end);
    if (end - P::TILE >= at.t0) load(two, end - P::TILE);
    for (int64_t t0 = end; t0 >= at.t0; t0 -= 3 * P::TILE) {
        tile(one, three, t0, 0);
        if (t0 - P::TILE < at.t0) break;
        tile(two, one, t0 - P::TILE, 1);
        if (t0 - 2 * P::TILE < at.t0) break;
        tile(three, two, t0 - 2 * P::TILE, 2);
    }
    if (at.w != 0 || at.tg != 0) return;
    float2 o[V];
#pragma unroll
    for (int v = 0; v < V; ++v) o[v] = make_float2(mu[v].P, mu[v].H);
    at.put(a.agg + at.agg(a, at.segment), o);
}

template <typename T, int V, int LC, int TS, int W, bool SEQ, bool NT>
__global__ void __launch_bounds__(W * 64, 2) k_rec_backward(RecArgs a) {
    typedef Place<V, LC, TS, W> P;
    static_assert(P::TILE % SPAN == 0, "");
    __shared__ float tot[3][3][W][P::C];
    __shared__ int next;
    const bool passed = a.tickets != nullptr;            // from segment to segment, else a.agg tells what enters each
    const int chain = xcd_remap(blockIdx.x % a.chains, a.chains);
    const P at = passed ? P(a, chain, a.segments - 1 - take(a, chain, next), a.seg) : P(a);
    const int64_t end = at.t0 + (at.end - 1 - at.t0) / P::TILE * P::TILE;
    Stream<T, V> sx(a.x, at.b * a.xb + end * a.xt, a.xt, a, at), sr(a.r, at.b * a.rb + end * a.rt, a.rt, a, at),
        si(a.i, at.b * a.ib + end * a.it, a.it, a, at), sg(a.g, at.b * a.gb + end * a.gt, a.gt, a, at);
    const int64_t o0 = (at.b * a.L + end) * a.dim;
    Output<T, V, NT> ox(a.dx, o0, a, at), orr(a.dr, o0, a, at), oi(a.di, o0, a, at);
    const int32_t* seq = SEQ ? a.seq + at.b * a.L : nullptr;
    const float* ck = a.ck + at.b * a.spans * a.dim + at.c;
    float A[V], mu[V], dA[V];
    const bool far = decay_rates<V>(a, at, A);
#pragma unroll
    for (int v = 0; v < V; ++v) {
        mu[v] = a.glast ? a.glast[(int64_t)at.b * a.dim + at.c + v] : 0.f;
        dA[v] = 0.f;
    }
    if (!passed)
#pragma unroll 16
    for (int u = a.segments - 1; u > at.segment; --u)
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const float2 p = a.agg[at.agg(a, u) + v];
            mu[v] = Map<SEQ>{p.x, p.y}.of(mu[v]);
        }
    auto last_of = [&](int64_t t0) { return (int)min(at.end - 1 - t0, (int64_t)P::TILE - 1); };
    struct Tile {
        Raw<T, V> x[TS], r[TS], i[TS], g[TS];
        float e[V];              // the state that enters the tile
        Steps<TS, P::G, SEQ> s;
    } one, two, three;
    auto load = [&](Tile& n, int64_t t0) {
        const int last = last_of(t0);
        sx.load(n.x, last);
        sr.load(n.r, last);
        si.load(n.i, last);
        sg.load(n.g, last);
#pragma unroll
        for (int v = 0; v < V; ++v) n.e[v] = ck[t0 / SPAN * a.dim + v];
        n.s.load(seq + t0, t0 == 0, at, last);
        sx.move(-P::TILE);
        sr.move(-P::TILE);
        si.move(-P::TILE);
        sg.move(-P::TILE);
    };
    auto tile = [&](Tile& c, Tile& n, int64_t t0, int buf) {
        const int last = last_of(t0);
        if (t0 - 2 * P::TILE >= at.t0) load(n, t0 - 2 * P::TILE);
        if ((SEQ || last != P::TILE - 1) && !c.s.set(t0 == 0, at, last)) {
#pragma unroll
            for (int j = 0; j < TS; ++j)
                if (!c.s.is_live(j)) {           // a = 1, nothing added
                    c.x[j].fill(0.f);
                    c.r[j].fill(-INF);
                    c.i[j].fill(0.f);
                    c.g[j].fill(0.f);
                }
        }
        float kept[TS][V], q[TS][V], s[TS][V], cq[TS][V], cosg[TS][V], ib[TS][V], beta[TS][V], L[TS][V];
#pragma unroll
        for (int j = 0; j < TS; ++j)
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const float eq = exp_neg(c.r[j].get(v)), es = exp_neg(c.i[j].get(v));
                q[j][v] = sigmoid_of(eq);
                s[j][v] = sigmoid_of(es);
                cq[j][v] = co_sigmoid(eq, q[j][v]);
                cosg[j][v] = co_sigmoid(es, s[j][v]);
                L[j][v] = A[v] * q[j][v];
            }
        decays<TS, V>(L, far, kept, beta);
#pragma unroll
        for (int j = 0; j < TS; ++j)
#pragma unroll
            for (int v = 0; v < V; ++v) {
                ib[j][v] = inv_beta(beta[j][v]);
                beta[j][v] *= ib[j][v];
            }
        // the maps of this thread's steps, forward and back (with the same P)
        Map<SEQ> up[V], down[V], f[V], b[V];
        by_decay(far, [&](auto is_far) {
            constexpr bool FAR = decltype(is_far)::value;
#pragma unroll
            for (int v = 0; v < V; ++v) {
#pragma unroll
                for (int j = 0; j < TS; ++j) {
                    const float add = beta[j][v] * s[j][v] * c.x[j].get(v);
                    f[v].P = j == 0 ? factor<FAR>(kept[j][v]) : shrunk<FAR>(kept[j][v], f[v].P);
                    f[v].H = j == 0 ? add : step<FAR>(kept[j][v], c.s.clears(j) ? 0.f : f[v].H, add);
                }
#pragma unroll
                for (int j = TS - 1; j >= 0; --j) {
                    b[v].H = step<FAR>(kept[j][v], j == TS - 1 ? c.g[j].get(v) : c.g[j].get(v) + b[v].H);
                    if (c.s.clears(j)) b[v].H = 0.f;
                }
            }
        });
#pragma unroll
        for (int v = 0; v < V; ++v) {
            if (SEQ && c.s.clear) f[v].P = -1.f;
            b[v].P = f[v].P;
            up[v] = scan<1, LC, SEQ>(f[v], at.lane);
            down[v] = scan<-1, LC, SEQ>(b[v], at.lane);
            if (at.tg == 0) {
                tot[buf][0][at.w][at.col + v] = b[v].P;
                tot[buf][2][at.w][at.col + v] = b[v].H;
            }
            if (at.tg == P::G - 1) tot[buf][1][at.w][at.col + v] = f[v].H;
        }
        lds_barrier();
        float k[V];
#pragma unroll
        for (int u = 0; u < W; ++u) {
            const int d = W - 1 - u;
            if (u < at.w) {
                asm volatile("");                // (branches: they are the wavefront's)
#pragma unroll
                for (int v = 0; v < V; ++v) c.e[v] = Map<SEQ>{tot[buf][0][u][at.col + v], tot[buf][1][u][at.col + v]}.of(c.e[v]);
            }
            if (d == at.w) {
                asm volatile("");
#pragma unroll
                for (int v = 0; v < V; ++v) k[v] = mu[v];
            }
#pragma unroll
            for (int v = 0; v < V; ++v) mu[v] = Map<SEQ>{tot[buf][0][d][at.col + v], tot[buf][2][d][at.col + v]}.of(mu[v]);
        }
        const Rsrc tx = ox.tile(last), tr = orr.tile(last), ti = oi.tile(last);
        by_decay(far, [&](auto is_far) {
            constexpr bool FAR = decltype(is_far)::value;
            float lam[TS][V];
#pragma unroll
            for (int v = 0; v < V; ++v) {
                c.e[v] = up[v].of(c.e[v]);
                k[v] = down[v].of(k[v]);
#pragma unroll
                for (int j = TS - 1; j >= 0; --j) {
                    lam[j][v] = c.g[j].get(v) + k[v];
                    k[v] = step<FAR>(kept[j][v], lam[j][v]);
                    if (c.s.clears(j)) k[v] = 0.f;
                }
            }
#pragma unroll
            for (int j = 0; j < TS; ++j) {
                float dx[V], dr[V], di[V];
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    const float xv = c.x[j].get(v), p = c.s.clears(j) ? 0.f : c.e[v];
                    const float av = factor<FAR>(kept[j][v]), sxv = s[j][v] * xv;
                    c.e[v] = step<FAR>(kept[j][v], p, beta[j][v] * sxv);
                    dx[v] = lam[j][v] * beta[j][v] * s[j][v];
                    di[v] = dx[v] * xv * cosg[j][v];
                    float dLq = lam[j][v] * av * fmaf(-av * ib[j][v], sxv, p) * q[j][v];
                    dr[v] = dLq * A[v] * cq[j][v];
                    // (what a padded row carries through may be no number)
                    if (SEQ && !c.s.is_live(j)) dx[v] = dr[v] = di[v] = dLq = 0.f;
                    dA[v] += dLq;
                }
                ox.store(tx, j, dx);
                orr.store(tr, j, dr);
                oi.store(ti, j, di);
            }
        });
        ox.move(-P::TILE);
        orr.move(-P::TILE);
        oi.move(-P::TILE);
    };
    load(one, end);
    if (end - P::TILE >= at.t0) load(two, end - P::TILE);
    if (passed && at.segment < a.segments - 1) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const uint32_t* p = a.states + at.agg(a, at.segment + 1) + v;
            uint32_t m = 0;                  // (of what is stored by another lane, or chain: any)
            while (__any(at.owns(v) && (m = peek(p)) == UNKNOWN)) __builtin_amdgcn_s_sleep(8);
            mu[v] = __uint_as_float(m);
        }
    }
    for (int64_t t0 = end; t0 >= at.t0; t0 -= 3 * P::TILE) {
        tile(one, three, t0, 0);
        if (t0 - P::TILE < at.t0) break;
        tile(two, one, t0 - P::TILE, 1);
        if (t0 - 2 * P::TILE < at.t0) break;
        tile(three, two, t0 - 2 * P::TILE, 2);
    }
    if (passed && at.segment > 0 && at.w == 0 && at.tg == 0)
#pragma unroll
        for (int v = 0; v < V; ++v)
            if (at.owns(v)) publish(a.states + at.agg(a, at.segment) + v, known(mu[v]));
    if (a.dh0 && at.segment == 0 && at.w == 0 && at.tg == 0) at.put(a.dh0 + (int64_t)at.b * a.dim + at.c, mu);
    // dA of this segment: of the lanes of a channel, then of the wavefronts in their order
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
        at.put(a.dA + at.agg(a, at.segment), dA);
    }
}

// dA of the segments of all rows, in their order
__global__ void __launch_bounds__(64) k_rec_join(const float* part, float* dA, int64_t parts, int64_t dim) {
    const int64_t c = (int64_t)blockIdx.x * 64 + threadIdx.x;
    if (c >= dim) return;
    double s = 0;
#pragma unroll 8
    for (int64_t b = 0; b < parts; ++b) s += part[b * dim + c];
    dA[c] = (float)s;
}

// no steps: the state stays, and so does its gradient
__global__ void __launch_bounds__(256) k_rec_nothing(const float* from, float* to, int64_t n) {
    for (int64_t k = (int64_t)blockIdx.x * 256 + threadIdx.x; k < n; k += (int64_t)gridDim.x * 256)
        to[k] = from ? from[k] : 0.f;
}

// One step of every row: 16 x 2560 bf16 2.4 us, a launch's own time (0.7 MB)
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
    const float q = sigmoid_of(exp_neg(to_f32(static_cast<const T*>(a.r)[b * a.rb + c])));
    const float s = sigmoid_of(exp_neg(to_f32(static_cast<const T*>(a.i)[b * a.ib + c])));
    const float xv = to_f32(static_cast<const T*>(a.x)[b * a.xb + c]), e = a.state[b * a.dim + c];
    const float L = decay_rate(a.A[c]) * q;
    float k, y;
    decay(L, k, y);
    decay_far(L, k, y);
    const float h = step<true>(k, e, __builtin_amdgcn_sqrtf(y) * s * xv);
    a.next[b * a.dim + c] = h;
    static_cast<T*>(a.out)[b * a.dim + c] = from_f32<T>(h);
}

// ---------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------
constexpr int LC = 32;
// Steps of a forward segment, 16 for each wavefront.  us for 64, 128, 256 of them: 160 chains x 4096 74, 86, 112; 240 131, 144,
// 145; 640 x 2048 165, 177, 180.  A chain's counter gives out a segment every 0.43 us, which bounds few chains: 40 x 16384
// 128, 95, 121; 16 x 16384 119, 60, 62; 8 x 16384 119, 58, 44.  One segment needs no counter: 2560 x 100 steps 38, 34, 69.
int forward_steps(int64_t batch, int64_t L, int64_t dim) {
    const int64_t chains = batch * ((dim + 2 * LC - 1) / (2 * LC));
    return L <= 128 || (chains >= 16 && chains < m2::cu_count() / 2) ? 128 : chains < 16 ? 256 : 64;
}
// counters, maps, states
struct ForwardPlan {
    int64_t segments;
    size_t maps, states, total;
};
ForwardPlan forward_plan(int64_t batch, int64_t L, int64_t dim) {
    const int steps = forward_steps(batch, L, dim);
    ForwardPlan p{(L + steps - 1) / steps};
    if (p.segments <= 1) return p;
    const size_t n = (size_t)batch * p.segments * dim;
    p.maps = 4 * TICKET * (size_t)batch * ((dim + 2 * LC - 1) / (2 * LC));
    p.states = p.maps + 8 * n;
    p.total = (p.states + 4 * n + 15) / 16 * 16;
    return p;
}
// Segments of the backward, and their steps.  Where the slabs alone leave CUs idle, as many as make five workgroups a CU,
// of 128 steps at least; a pass more over two of the inputs then finds what enters each.  One segment
// against many, us: 160 slabs x 4096 298 and 196; 240 309 and 306; 320 432 and 367; 480 x 2048 246 and 271.
// (The forward's way, each segment waiting for others, takes 222 for 40 slabs x 16384, 191 so; 640 x 2048 362 and 327: a
// segment's four inputs and its factors leave registers for two workgroups a CU, and none of them loads ahead.)
// Two workgroups a CU run at once.  Where the slabs are a few times as many, the last round of whole rows would leave CUs idle:
// up to four segments of 512 steps at least then pass on what goes from one to the next, given out like the forward's
// (a slab's next segment is due when all slabs' last ones went out, so hardly anybody waits).  One, two, four of them, us:
// 520 slabs x 1024 163, 143, 135; 640 x 2048 332, 308, 294; 800 x 1600 321, 299, 295; 1280 x 1024 301, 293, 302; 2560 x 512
// 281, 299, 335; 748 x 301 78, 85, 87.
struct BackPlan {
    int64_t seg;
    int segments;
    bool passed;
    size_t states, dA, total;                // counters or maps first
};
BackPlan back_plan(int64_t batch, int64_t L, int64_t dim) {
    constexpr int64_t UNIT = 128;
    const int64_t units = L > 0 ? (L + UNIT - 1) / UNIT : 1, slabs = batch * ((dim + 2 * LC - 1) / (2 * LC));
    const int64_t ncu = m2::cu_count();
    BackPlan p{};
    int64_t s = 1;
    if (slabs > 0 && slabs < ncu * 3 / 2) s = (5 * ncu + slabs - 1) / slabs;
    else if (slabs > 2 * ncu && slabs <= 8 * ncu) s = units / 4 < 4 ? units / 4 : 4;
    if (s > units) s = units;
    if (s < 1) s = 1;
    const int64_t per = (units + s - 1) / s;
    p.seg = per * UNIT;
    p.segments = (int)((units + per - 1) / per);
    p.passed = p.segments > 1 && slabs >= ncu * 3 / 2;
    const size_t n = (size_t)(batch > 1 ? batch : 1) * p.segments * dim;
    p.states = p.passed ? 4 * TICKET * (size_t)slabs : 0;
    p.dA = p.passed ? (p.states + 4 * n + 15) / 16 * 16 : 8 * n;
    p.total = p.dA + 4 * n;
    return p;
}
// counters and states of `bytes`, unknown
void clear(void* ws, size_t bytes, hipStream_t s) {
    const int64_t n = (int64_t)(bytes / 16);
    hipLaunchKernelGGL(k_rec_clear, dim3((unsigned)(n < (1 << 18) ? (n + 255) / 256 : 1024)), dim3(256), 0, s,
                       static_cast<u32x4*>(ws), n);
}

template <typename T, int V, bool SEQ, bool NT> void launch_forward(const RecArgs& a, int steps, hipStream_t s) {
    const dim3 grid((unsigned)((int64_t)a.chains * a.segments));
    auto go = [&](auto k, int w) { hipLaunchKernelGGL(k, grid, dim3(w * 64), 0, s, a); };
    if (steps == 64) go(k_rec_forward<T, V, LC, 8, 4, SEQ, NT>, 4);
    else if (steps == 128) go(k_rec_forward<T, V, LC, 8, 8, SEQ, NT>, 8);
    else go(k_rec_forward<T, V, LC, 8, 16, SEQ, NT>, 16);
}
template <typename T, int V, bool SEQ, bool NT> void launch_backward(const RecArgs& a, hipStream_t s) {
    const dim3 grid((unsigned)((int64_t)a.chains * a.segments));
    auto go = [&](auto k) { hipLaunchKernelGGL(k, grid, dim3(256), 0, s, a); };
    if (a.segments > 1 && !a.tickets) go(k_rec_back_agg<T, V, LC, 4, 4, SEQ>);
    go(k_rec_backward<T, V, LC, 4, 4, SEQ, NT>);
}
// steps: of a forward segment, or 0: backward
template <typename T> void run(RecArgs a, int64_t batch, int steps, hipStream_t s) {
    a.slabs = a.dim == 1 ? 1 : (a.dim + 2 * LC - 1) / (2 * LC);
    a.chains = (int)batch * a.slabs;
    // Results go past the caches where what is read and written does not fit the last of them (256 MB): they would take
    // the place of what is read next, or again.  us with and without: 16384 x 2560 forward 107 and 109, backward 197 and 211;
    // 8 x 2048 x 5120 176 and 181, 332 and 341.
    const bool nt = batch * a.L * a.dim * (int64_t)sizeof(T) * (steps ? 4 : 7) > (256ll << 20);
    auto go = [&](auto seq, auto many) {
        constexpr bool SEQ = decltype(seq)::value, NT = decltype(many)::value;
        if (steps) {
            if (a.dim == 1) launch_forward<T, 1, SEQ, false>(a, steps, s);
            else launch_forward<T, 2, SEQ, NT>(a, steps, s);
        } else {
            if (a.dim == 1) launch_backward<T, 1, SEQ, false>(a, s);
            else launch_backward<T, 2, SEQ, NT>(a, s);
        }
    };
    if (a.seq) {
        if (nt) go(std::true_type(), std::true_type());
        else go(std::true_type(), std::false_type());
    } else {
        if (nt) go(std::false_type(), std::true_type());
        else go(std::false_type(), std::false_type());
    }
}

// (a tile's offsets have 32 bits: at most 256 steps of 4 bytes)
constexpr int64_t MAX_STRIDE = 1 << 20;
bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
// rows of a step that are one, or behind each other
bool stride_ok(int64_t st, int64_t dim) { return st == 0 || (st >= dim && st <= MAX_STRIDE); }

// what a call may ask for, whichever it is
int check_sizes(const char* who, int64_t batch, int64_t seqlen, int64_t dim, int dtype) {
    M2_REQUIRE(batch >= 0 && seqlen >= 0 && dim > 0 && dim <= MAX_STRIDE && seqlen < (1ll << 32), M2_ERR_INVALID,
               "%s: bad sizes (batch %lld, seqlen %lld, dim %lld)", who, (long long)batch, (long long)seqlen,
               (long long)dim);
    M2_REQUIRE(dtype == M2_F32 || dtype == M2_BF16, M2_ERR_UNSUPPORTED, "%s: dtype %d", who, dtype);
    // (counts of threads: 32 bits)
    M2_REQUIRE(batch < (1ll << 22) && batch * ((dim + 63) / 64) < (1ll << 22), M2_ERR_UNSUPPORTED, "%s: too many rows", who);
    return M2_OK;
}

}  // namespace

namespace m2 {

size_t gated_recurrence_workspace(const m2_gated_recurrence_args& a) {
    if (check_sizes("gated_linear_recurrence", a.batch, a.seqlen, a.dim, a.dtype)) return 0;
    const size_t b = forward_plan(a.batch, a.seqlen, a.dim).total;
    return b ? b : 256;
}

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
    M2_REQUIRE(stride_ok(a.x_stride_time, a.dim) && stride_ok(a.r_stride_time, a.dim) && stride_ok(a.i_stride_time, a.dim),
               M2_ERR_INVALID, "%s: strides of time (0, or dim to %lld)", who, (long long)MAX_STRIDE);
    RecArgs k{};
    k.x = a.x; k.r = a.r; k.i = a.i; k.A = a.A; k.h0 = a.initial_states; k.seq = a.seq_idx;
    k.xb = a.x_stride_batch; k.xt = a.x_stride_time;
    k.rb = a.r_stride_batch; k.rt = a.r_stride_time;
    k.ib = a.i_stride_batch; k.it = a.i_stride_time;
    k.ck = a.span_states; k.L = a.seqlen; k.spans = (a.seqlen + SPAN - 1) / SPAN; k.dim = (int)a.dim;
    k.out = a.out; k.last = a.final_states;
    const int steps = forward_steps(a.batch, a.seqlen, a.dim);
    const ForwardPlan p = forward_plan(a.batch, a.seqlen, a.dim);
    M2_REQUIRE(a.batch * ((a.dim + 63) / 64) * p.segments * (4 * steps) < (1ll << 32), M2_ERR_UNSUPPORTED, "%s: too many steps", who);
    M2_REQUIRE(p.total == 0 || (a.workspace && a.workspace_bytes >= p.total), M2_ERR_WORKSPACE,
               "%s: workspace of %zu bytes needed, %zu given", who, p.total, a.workspace_bytes);
    M2_REQUIRE(p.total == 0 || al16(a.workspace), M2_ERR_WORKSPACE, "%s: workspace of 16-byte alignment needed", who);
    k.segments = (int)p.segments;
    if (p.segments > 1) {
        char* ws = static_cast<char*>(a.workspace);
        k.tickets = reinterpret_cast<int*>(ws);
        k.maps = reinterpret_cast<uint64_t*>(ws + p.maps);
        k.states = reinterpret_cast<uint32_t*>(ws + p.states);
        clear(ws, p.total, s);
    }
    if (a.dtype == M2_F32) run<float>(k, a.batch, steps, s);
    else run<bf16>(k, a.batch, steps, s);
    return check_launch(who);
}

size_t gated_recurrence_grad_workspace(const m2_gated_recurrence_grad_args& a) {
    if (check_sizes("gated_linear_recurrence_grad", a.batch, a.seqlen, a.dim, a.dtype)) return 0;
    return back_plan(a.batch, a.seqlen, a.dim).total;
}

int launch_gated_recurrence_grad(const m2_gated_recurrence_grad_args& a, hipStream_t s) {
    const char* who = "gated_linear_recurrence_grad";
    if (int rc = check_sizes(who, a.batch, a.seqlen, a.dim, a.dtype)) return rc;
    M2_REQUIRE(a.batch > 0 && a.seqlen > 0, M2_ERR_INVALID, "%s: no steps", who);
    M2_REQUIRE(a.x && a.r && a.i && a.A && a.span_states && a.grad_out && a.grad_x && a.grad_r && a.grad_i && a.grad_A,
               M2_ERR_INVALID, "%s: x, r, i, A, span_states, grad_out and the gradients are required", who);
    M2_REQUIRE(stride_ok(a.x_stride_time, a.dim) && stride_ok(a.r_stride_time, a.dim) && stride_ok(a.i_stride_time, a.dim) &&
                   stride_ok(a.grad_out_stride_time, a.dim),
               M2_ERR_INVALID, "%s: strides of time (0, or dim to %lld)", who, (long long)MAX_STRIDE);
    const BackPlan p = back_plan(a.batch, a.seqlen, a.dim);
    M2_REQUIRE(a.workspace && a.workspace_bytes >= p.total, M2_ERR_WORKSPACE,
               "%s: workspace of %zu bytes needed, %zu given", who, p.total, a.workspace_bytes);
    M2_REQUIRE(al16(a.workspace), M2_ERR_WORKSPACE, "%s: workspace of 16-byte alignment needed", who);
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
    k.segments = p.segments;
    k.seg = p.seg;
    const int64_t parts = a.batch * k.segments;
    char* ws = static_cast<char*>(a.workspace);
    if (p.passed) {
        k.tickets = reinterpret_cast<int*>(ws);
        k.states = reinterpret_cast<uint32_t*>(ws + p.states);
        clear(ws, p.dA, s);
    } else {
        k.agg = reinterpret_cast<float2*>(ws);
    }
    k.dA = parts == 1 ? a.grad_A : reinterpret_cast<float*>(ws + p.dA);
    if (a.dtype == M2_F32) run<float>(k, a.batch, 0, s);
    else run<bf16>(k, a.batch, 0, s);
    if (parts > 1)
        hipLaunchKernelGGL(k_rec_join, dim3((unsigned)((a.dim + 63) / 64)), dim3(64), 0, s, k.dA, a.grad_A, parts, a.dim);
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
