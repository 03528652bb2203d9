// embedding: out[n] = scale * weight[ids[n]], and its gradient
//   grad_weight[v] = scale * sum over {n : ids[n] == v} of grad[n]
// by sorted tokens.
//
// The lookup is a gather of whole rows: a wavefront per (row, column part), 16 bytes a
// lane, bound by HBM for many rows and by two dependent loads (id, row) for
// few.
//
// The gradient sorts (id, n) by id with a stable radix sort (equal ids keep the
// order of n), walks the sorted list in pieces of up to 32 entries, one
// workgroup each, with the sum of the current id's rows in registers, and
// writes each row of the result once.  An id whose entries cross pieces
// (frequent tokens) leaves one partial row per piece, which the workgroup of its
// first piece's join adds in order: no float atomics, so equal inputs give
// equal bits, and a token that is half of the batch is spread over as many
// workgroups as any others.  The rows that no id names (most of a large
// vocabulary) are zeroed by further workgroups of the same launch, from a bitmap
// that the sort leaves: every byte of the result is written once.  Bound by
// HBM: grad read once, the result written once.
#include "m2_internal.h"

namespace {

constexpr int SORT_THREADS = 256, SORT_ITEMS = 8, SORT_TILE = SORT_THREADS * SORT_ITEMS;
constexpr int SMALL_THREADS = 1024, SMALL_ITEMS = 4, SMALL_N = SMALL_THREADS * SMALL_ITEMS;
constexpr int MAX_BINS = 512;

M2_DEV int64_t load_id(const void* ids, int64_t i, int is64) {
    return is64 ? reinterpret_cast<const int64_t*>(ids)[i]
                : (int64_t) reinterpret_cast<const int32_t*>(ids)[i];
}

// V consecutive elements as floats (one 16-byte access where V fills it)
template <typename T, int V> struct Vec {
    float v[V];
    M2_DEV void load(const T* p) {
        if constexpr (V == 1) {
            v[0] = to_f32(*p);
        } else if constexpr (sizeof(T) == 2) {
            const u32x4 r = *reinterpret_cast<const u32x4*>(p);
#pragma unroll
            for (int i = 0; i < 4; ++i) { v[2 * i] = bf16_lo(r[i]); v[2 * i + 1] = bf16_hi(r[i]); }
        } else {
#pragma unroll
            for (int i = 0; i < V; i += 4) {
                const f32x4 r = *reinterpret_cast<const f32x4*>(p + i);
#pragma unroll
                for (int j = 0; j < 4; ++j) v[i + j] = r[j];
            }
        }
    }
    M2_DEV void store(T* p) const {
        if constexpr (V == 1) {
            *p = from_f32<T>(v[0]);
        } else if constexpr (sizeof(T) == 2) {
            u32x4 r;
#pragma unroll
            for (int i = 0; i < 4; ++i) r[i] = pk_bf16(v[2 * i], v[2 * i + 1]);
            *reinterpret_cast<u32x4*>(p) = r;
        } else {
#pragma unroll
            for (int i = 0; i < V; i += 4) {
                const f32x4 r = {v[i], v[i + 1], v[i + 2], v[i + 3]};
                *reinterpret_cast<f32x4*>(p + i) = r;
            }
        }
    }
};

// ---------------------------------------------------------------------------
// lookup
// ---------------------------------------------------------------------------
struct EmbedArgs {
    const void* ids;
    const void* w;
    void* out;
    int64_t n, vocab, ldw, ldo;
    int vecs;          // V-element pieces of a row
    int parts;         // column parts of a row, 64 * UN pieces each
    float scale;
    int id64;
};

constexpr int EMB_UN = 2;    // pieces per lane

template <typename T, int V>
__global__ void __launch_bounds__(256) k_embedding(EmbedArgs a) {
    const int64_t work = (int64_t)blockIdx.x * 4 + wave_id();
    const int64_t row = work / a.parts;
    if (row >= a.n) return;
    const int c0 = (int)(work % a.parts) * 64 * EMB_UN + (threadIdx.x & 63);
    const int64_t id = load_id(a.ids, row, a.id64);
    const bool ok = id >= 0 && id < a.vocab;
    const T* src = static_cast<const T*>(a.w) + (ok ? id : 0) * a.ldw;
    T* dst = static_cast<T*>(a.out) + row * a.ldo;
    Vec<T, V> v[EMB_UN];
#pragma unroll
    for (int u = 0; u < EMB_UN; ++u)
        if (c0 + 64 * u < a.vecs) v[u].load(src + (int64_t)(c0 + 64 * u) * V);
#pragma unroll
    for (int u = 0; u < EMB_UN; ++u) {
        if (c0 + 64 * u >= a.vecs) continue;
#pragma unroll
        for (int i = 0; i < V; ++i) v[u].v[i] = ok ? v[u].v[i] * a.scale : __builtin_nanf("");
        v[u].store(dst + (int64_t)(c0 + 64 * u) * V);
    }
}

// ---------------------------------------------------------------------------
// the sort: keys are ids, or `vocab` for the entries that take no part
// ---------------------------------------------------------------------------
struct SortArgs {
    const void* ids;
    const int32_t* keys_in;      // NULL in the first pass (keys come from ids)
    const int32_t* pos_in;
    int32_t* keys_out;
    int32_t* pos_out;
    int32_t* hist;               // [blocks][bins]
    uint32_t* used;              // bitmap of the ids that take part
    int64_t vocab, padding;
    int n, id64, shift, bits, nb, words;
};

M2_DEV int32_t key_of(const SortArgs& a, int i) {
    const int64_t id = load_id(a.ids, i, a.id64);
    return id >= 0 && id < a.vocab && id != a.padding ? (int32_t)id : (int32_t)a.vocab;
}

__global__ void __launch_bounds__(SORT_THREADS) k_sort_hist(SortArgs a) {
    __shared__ int h[MAX_BINS];
    const int bins = 1 << a.bits, t = threadIdx.x, b = blockIdx.x;
    if (!a.keys_in)
        for (int64_t w = (int64_t)b * SORT_THREADS + t; w < a.words; w += (int64_t)a.nb * SORT_THREADS)
            a.used[w] = 0;
    for (int d = t; d < bins; d += SORT_THREADS) h[d] = 0;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < SORT_ITEMS; ++j) {
        const int i = b * SORT_TILE + j * SORT_THREADS + t;
        if (i < a.n) {
            const int32_t k = a.keys_in ? a.keys_in[i] : key_of(a, i);
            atomicAdd(&h[(k >> a.shift) & (bins - 1)], 1);
        }
    }
    __syncthreads();
    for (int d = t; d < bins; d += SORT_THREADS) a.hist[b * bins + d] = h[d];
}

// The place of an entry among the entries of its wavefront with the same
// digit, and their number so far: lanes with equal digits find each other by
// one ballot per bit; the first of them advances the wavefront's counter.
M2_DEV int wave_rank(int digit, bool on, int bits, int* cnt) {
    const int lane = threadIdx.x & 63;
    uint64_t peers = __ballot(on);
    for (int b = 0; b < bits; ++b) {
        const bool one = (digit >> b) & 1;
        const uint64_t m = __ballot(one);
        peers &= one ? m : ~m;
    }
    const int leader = __ffsll((unsigned long long)peers) - 1;
    int old = 0;
    if (on && lane == leader) old = atomicAdd(&cnt[digit], __popcll(peers));
    old = __shfl(old, leader < 0 ? 0 : leader);
    return old + __popcll(peers & ((1ull << lane) - 1));
}

// Exclusive prefix sums of v over the workgroup's NT threads, in thread order
template <int NT> M2_DEV int block_excl(int v, int* tmp) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    int s = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int u = __shfl_up(s, o);
        if (lane >= o) s += u;
    }
    if (lane == 63) tmp[w] = s;
    __syncthreads();
    int base = 0;
    for (int j = 0; j < NT / 64; ++j) base += j < w ? tmp[j] : 0;
    __syncthreads();
    return base + s - v;
}

__global__ void __launch_bounds__(SORT_THREADS) k_sort_scatter(SortArgs a, int last) {
    constexpr int NW = SORT_THREADS / 64;
    __shared__ int cnt[NW][MAX_BINS];
    __shared__ int tmp[NW];
    const int bins = 1 << a.bits, t = threadIdx.x, b = blockIdx.x, w = wave_id(), lane = t & 63;
    int32_t key[SORT_ITEMS], pos[SORT_ITEMS];
    int rank[SORT_ITEMS];
    const int base = b * SORT_TILE + w * 64 * SORT_ITEMS + lane;
#pragma unroll
    for (int j = 0; j < SORT_ITEMS; ++j) {
        const int i = base + 64 * j;
        key[j] = i < a.n ? (a.keys_in ? a.keys_in[i] : key_of(a, i)) : 0;
        pos[j] = i < a.n && a.pos_in ? a.pos_in[i] : i;
    }
    for (int d = t; d < NW * MAX_BINS; d += SORT_THREADS) (&cnt[0][0])[d] = 0;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < SORT_ITEMS; ++j)
        rank[j] = wave_rank((key[j] >> a.shift) & (bins - 1), base + 64 * j < a.n, a.bits, cnt[w]);
    __syncthreads();
    // where each (digit, wavefront) of this block begins: the entries of smaller digits in
    // all blocks, of this digit in earlier blocks and in earlier wavefronts.  Thread t
    // owns digits D t .. D t + D - 1 (a fixed order for the prefix sum).
    constexpr int D = MAX_BINS / SORT_THREADS;
    int tot[D], before[D], mine = 0;
#pragma unroll
    for (int k = 0; k < D; ++k) {
        const int d = t * D + k;
        tot[k] = before[k] = 0;
        if (d < bins)
            for (int q = 0; q < a.nb; ++q) {
                const int c = a.hist[q * bins + d];
                tot[k] += c;
                before[k] += q < b ? c : 0;
            }
        mine += tot[k];
    }
    int start = block_excl<SORT_THREADS>(mine, tmp);
#pragma unroll
    for (int k = 0; k < D; ++k) {
        const int d = t * D + k;
        int s = start + before[k];
#pragma unroll
        for (int q = 0; q < NW; ++q) {
            const int c = cnt[q][d];
            cnt[q][d] = s;
            s += c;
        }
        start += tot[k];
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < SORT_ITEMS; ++j) {
        if (base + 64 * j >= a.n) continue;
        const int p = cnt[w][(key[j] >> a.shift) & (bins - 1)] + rank[j];
        a.keys_out[p] = key[j];
        a.pos_out[p] = pos[j];
        if (last && key[j] < a.vocab) atomicOr(&a.used[key[j] >> 5], 1u << (key[j] & 31));
    }
}

// Up to SMALL_N entries: every pass in one workgroup, the list in LDS between
// the passes (a.shift, a.bits: of every pass; passes in a.nb).
__global__ void __launch_bounds__(SMALL_THREADS) k_sort_small(SortArgs a) {
    constexpr int NW = SMALL_THREADS / 64;
    __shared__ int cnt[NW][MAX_BINS];
    __shared__ int32_t lk[SMALL_N], lp[SMALL_N];
    __shared__ int tmp[NW];
    const int bins = 1 << a.bits, t = threadIdx.x, w = wave_id(), lane = t & 63;
    for (int i = t; i < a.words; i += SMALL_THREADS) a.used[i] = 0;
    const int base = w * 64 * SMALL_ITEMS + lane;
    int32_t key[SMALL_ITEMS], pos[SMALL_ITEMS];
    int rank[SMALL_ITEMS];
#pragma unroll
    for (int j = 0; j < SMALL_ITEMS; ++j) {
        const int i = base + 64 * j;
        key[j] = i < a.n ? key_of(a, i) : 0;
        pos[j] = i;
    }
    for (int pass = 0; pass < a.nb; ++pass) {
        const int shift = pass * a.bits;
        for (int d = t; d < NW * MAX_BINS; d += SMALL_THREADS) (&cnt[0][0])[d] = 0;
        __syncthreads();
#pragma unroll
        for (int j = 0; j < SMALL_ITEMS; ++j)
            rank[j] = wave_rank((key[j] >> shift) & (bins - 1), base + 64 * j < a.n, a.bits, cnt[w]);
        __syncthreads();
        int tot = 0;
        if (t < bins)
#pragma unroll
            for (int q = 0; q < NW; ++q) tot += cnt[q][t];
        int s = block_excl<SMALL_THREADS>(tot, tmp);
        if (t < bins)
#pragma unroll
            for (int q = 0; q < NW; ++q) {
                const int c = cnt[q][t];
                cnt[q][t] = s;
                s += c;
            }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < SMALL_ITEMS; ++j) {
            if (base + 64 * j >= a.n) continue;
            const int p = cnt[w][(key[j] >> shift) & (bins - 1)] + rank[j];
            lk[p] = key[j];
            lp[p] = pos[j];
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < SMALL_ITEMS; ++j) {
            const int i = base + 64 * j;
            if (i < a.n) { key[j] = lk[i]; pos[j] = lp[i]; }
        }
    }
#pragma unroll
    for (int j = 0; j < SMALL_ITEMS; ++j) {
        const int i = base + 64 * j;
        if (i >= a.n) continue;
        a.keys_out[i] = key[j];
        a.pos_out[i] = pos[j];
        // after the zeroing of `used` above: the passes' barriers lie between
        if (key[j] < a.vocab) atomicOr(&a.used[key[j] >> 5], 1u << (key[j] & 31));
    }
}

// ---------------------------------------------------------------------------
// the sums
// ---------------------------------------------------------------------------
struct ReduceArgs {
    const int32_t* keys;
    const int32_t* pos;
    const uint32_t* used;
    const void* grad;
    void* out;
    float* part;             // [pieces][2][ldp]: of a row begun before the piece / left unfinished
    int64_t ldg, ldo, ldp, vocab;
    int n, piece, pieces;    // entries per piece
    int vecs, slabs;         // V-element pieces of a row, split over `slabs` workgroups
    int cols;                // elements of a row
    int nred, accumulate;    // workgroups that sum; the others zero rows
    float scale;
};

template <typename TO, int V>
M2_DEV void put_row(const ReduceArgs& a, int32_t key, int c, Vec<float, V> s) {
    TO* p = static_cast<TO*>(a.out) + (int64_t)key * a.ldo + (int64_t)c * V;
#pragma unroll
    for (int i = 0; i < V; ++i) s.v[i] *= a.scale;
    Vec<TO, V> o;
    if (a.accumulate) {
        o.load(p);
#pragma unroll
        for (int i = 0; i < V; ++i) s.v[i] += o.v[i];
    }
#pragma unroll
    for (int i = 0; i < V; ++i) o.v[i] = s.v[i];
    o.store(p);
}

// Rows without an id become zero: whole 16-byte pieces, single elements at the ends
// of a row that does not begin or end on one.
template <typename TO> M2_DEV void zero_row(TO* p, int n, int t, int nt) {
    constexpr int E = 16 / sizeof(TO);
    int head = (int)((16 - ((uintptr_t)p & 15)) & 15) / (int)sizeof(TO);
    head = head < n ? head : n;
    const int vecs = (n - head) / E;
    const u32x4 z = {0, 0, 0, 0};
    for (int i = t; i < vecs; i += nt) *reinterpret_cast<u32x4*>(p + head + i * E) = z;
    const int tail = head + vecs * E;
    if (t < head) p[t] = (TO)0.f;
    if (t < n - tail) p[tail + t] = (TO)0.f;
}

template <typename T, typename TO, int V>
__global__ void __launch_bounds__(512) k_embed_sum(ReduceArgs a) {
    constexpr int UN = V == 1 ? 8 : 4;
    const int t = threadIdx.x;
    if ((int)blockIdx.x >= a.nred) {
        // the rows of 32-bit words of the bitmap: a wavefront per row
        const int nw = blockDim.x >> 6;
        const int64_t stride = (int64_t)(gridDim.x - a.nred) * nw;
        for (int64_t r = (int64_t)(blockIdx.x - a.nred) * nw + wave_id(); r < a.vocab; r += stride)
            if (!((a.used[r >> 5] >> (r & 31)) & 1))
                zero_row(static_cast<TO*>(a.out) + r * a.ldo, a.cols, t & 63, 64);
        return;
    }
    const int p = blockIdx.x / a.slabs, slab = blockIdx.x % a.slabs;
    const int per = (a.vecs + a.slabs - 1) / a.slabs;
    const int c = slab * per + t;
    const bool on = t < per && c < a.vecs;
    const int e0 = p * a.piece, e1 = min(a.n, e0 + a.piece);
    const T* g = static_cast<const T*>(a.grad) + (int64_t)c * V;
    int32_t key = a.keys[e0];
    bool head = p > 0 && a.keys[e0 - 1] == key;      // the row began in an earlier piece
    Vec<float, V> s;
#pragma unroll
    for (int i = 0; i < V; ++i) s.v[i] = 0.f;
    auto flush = [&](bool more) {
        if (!on || key >= a.vocab) return;
        if (!head && !more) put_row<TO, V>(a, key, c, s);
        else s.store(a.part + ((int64_t)p * 2 + (head ? 0 : 1)) * a.ldp + (int64_t)c * V);
    };
    for (int e = e0; e < e1; e += UN) {
        Vec<T, V> v[UN];
        int32_t k[UN];
#pragma unroll
        for (int u = 0; u < UN; ++u) {
            const int q = min(e + u, e1 - 1);
            k[u] = a.keys[q];
            if (on) v[u].load(g + (int64_t)a.pos[q] * a.ldg);
        }
#pragma unroll
        for (int u = 0; u < UN; ++u) {
            if (e + u >= e1) break;
            if (k[u] != key) {
                flush(false);
                key = k[u];
                head = false;
#pragma unroll
                for (int i = 0; i < V; ++i) s.v[i] = 0.f;
            }
            if (on)
#pragma unroll
                for (int i = 0; i < V; ++i) s.v[i] += v[u].v[i];
        }
    }
    flush(e1 < a.n && a.keys[e1] == key);
}

// The rows that cross pieces: the piece in which such a row begins adds its
// partial rows in order.
template <typename TO, int V>
__global__ void __launch_bounds__(512) k_embed_join(ReduceArgs a) {
    const int p = blockIdx.x / a.slabs, slab = blockIdx.x % a.slabs, t = threadIdx.x;
    const int e0 = p * a.piece, e1 = min(a.n, e0 + a.piece);
    if (e1 >= a.n) return;
    const int32_t key = a.keys[e1 - 1];
    if (key >= a.vocab || a.keys[e1] != key) return;
    if (a.keys[e0] == key && p > 0 && a.keys[e0 - 1] == key) return;      // begun before this piece
    const int per = (a.vecs + a.slabs - 1) / a.slabs;
    const int c = slab * per + t;
    if (t >= per || c >= a.vecs) return;
    Vec<float, V> s;
    s.load(a.part + ((int64_t)p * 2 + 1) * a.ldp + (int64_t)c * V);
    int q = p + 1;
    // piece q holds more of the row; the last such piece is the first that does not end in it
    // before the list goes on with it
    while (true) {
        Vec<float, V> v;
        v.load(a.part + (int64_t)q * 2 * a.ldp + (int64_t)c * V);
#pragma unroll
        for (int i = 0; i < V; ++i) s.v[i] += v.v[i];
        const int64_t nx = (int64_t)(q + 1) * a.piece;
        if (nx >= a.n || a.keys[nx] != key) break;
        ++q;
    }
    put_row<TO, V>(a, key, c, s);
}

size_t align256(size_t v) { return (v + 255) & ~size_t(255); }

struct GradPlan {
    int bits, passes, nb, piece, pieces, words;
    int64_t ldp;
    bool small;
    size_t keys[2], pos[2], hist, used, part, total;
};

GradPlan grad_plan(const m2_embedding_grad_args& a) {
    GradPlan p{};
    int kb = 1;
    while ((1ll << kb) <= a.vocab) ++kb;          // keys 0 .. vocab
    p.passes = (kb + 8) / 9;
    p.bits = (kb + p.passes - 1) / p.passes;
    p.small = a.n <= SMALL_N;
    p.nb = (int)((a.n + SORT_TILE - 1) / SORT_TILE);
    // entries per piece: about 512 pieces, so that every CU has two, of 4 to 32
    // entries (longer pieces leave fewer partial rows, shorter ones more
    // workgroups to a small batch)
    int64_t e = a.n / 512;
    p.piece = e < 4 ? 4 : e > 32 ? 32 : (int)e;
    p.pieces = (int)((a.n + p.piece - 1) / p.piece);
    p.words = (int)((a.vocab + 31) / 32);
    p.ldp = (a.dim + 7) / 8 * 8;
    size_t at = 0;
    auto take = [&](size_t bytes) { const size_t r = at; at += align256(bytes); return r; };
    for (int i = 0; i < 2; ++i) { p.keys[i] = take(4 * (size_t)a.n); p.pos[i] = take(4 * (size_t)a.n); }
    p.hist = take(4 * (size_t)p.nb << p.bits);
    p.used = take(4 * (size_t)p.words);
    p.part = take((size_t)p.pieces * 2 * p.ldp * 4);
    p.total = at;
    return p;
}

int check_grad(const m2_embedding_grad_args& a) {
    const char* who = "embedding_grad";
    M2_REQUIRE(a.n >= 0 && a.n < (1ll << 31) - 4096 && a.vocab > 0 && a.vocab < (1ll << 27) && a.dim > 0 &&
                   a.dim < (1ll << 30),
               M2_ERR_INVALID, "%s: bad sizes (n %lld, vocab %lld, dim %lld)", who, (long long)a.n,
               (long long)a.vocab, (long long)a.dim);
    return M2_OK;
}

template <typename T, typename TO, int V>
void launch_sums(const ReduceArgs& r, unsigned fill, int threads, hipStream_t s) {
    hipLaunchKernelGGL((k_embed_sum<T, TO, V>), dim3(r.nred + fill), dim3(threads), 0, s, r);
    if (r.pieces > 1)
        hipLaunchKernelGGL((k_embed_join<TO, V>), dim3(r.nred), dim3(threads), 0, s, r);
}

}  // namespace

namespace m2 {

static bool al16(const void* p) { return ((uintptr_t)p & 15) == 0; }

int launch_embedding(const m2_embedding_args& a, hipStream_t s) {
    const char* who = "embedding";
    M2_REQUIRE(a.n >= 0 && a.vocab > 0 && a.dim > 0 && a.dim < (1ll << 30), M2_ERR_INVALID,
               "%s: bad sizes (n %lld, vocab %lld, dim %lld)", who, (long long)a.n, (long long)a.vocab,
               (long long)a.dim);
    M2_REQUIRE(a.dtype == M2_F32 || a.dtype == M2_BF16, M2_ERR_UNSUPPORTED, "%s: dtype %d", who, a.dtype);
    M2_REQUIRE(a.id_dtype == M2_I32 || a.id_dtype == M2_I64, M2_ERR_UNSUPPORTED, "%s: id dtype %d", who,
               a.id_dtype);
    M2_REQUIRE(a.ldw >= a.dim && a.ldo >= a.dim, M2_ERR_INVALID, "%s: row strides", who);
    if (a.n == 0) return M2_OK;
    M2_REQUIRE(a.ids && a.weight && a.out, M2_ERR_INVALID, "%s: ids, weight and out are required", who);
    const int es = (int)m2_dtype_size(a.dtype), ev = 16 / es;
    const bool vec = a.dim % ev == 0 && a.ldw % ev == 0 && a.ldo % ev == 0 && al16(a.weight) && al16(a.out);
    EmbedArgs k{a.ids, a.weight, a.out, a.n, a.vocab, a.ldw, a.ldo, 0, 0, a.scale, a.id_dtype == M2_I64};
    k.vecs = (int)(vec ? a.dim / ev : a.dim);
    k.parts = (k.vecs + 64 * EMB_UN - 1) / (64 * EMB_UN);
    const int64_t blocks = (a.n * k.parts + 3) / 4;
    M2_REQUIRE(blocks < (1ll << 31), M2_ERR_UNSUPPORTED, "%s: too many rows", who);
    const dim3 grid((unsigned)blocks), thr(256);
    if (a.dtype == M2_BF16) {
        if (vec) hipLaunchKernelGGL((k_embedding<bf16, 8>), grid, thr, 0, s, k);
        else hipLaunchKernelGGL((k_embedding<bf16, 1>), grid, thr, 0, s, k);
    } else {
        if (vec) hipLaunchKernelGGL((k_embedding<float, 4>), grid, thr, 0, s, k);
        else hipLaunchKernelGGL((k_embedding<float, 1>), grid, thr, 0, s, k);
    }
    return check_launch(who);
}

size_t embedding_grad_workspace(const m2_embedding_grad_args& a) {
    if (check_grad(a)) return 0;
    const size_t n = grad_plan(a).total;
    return n ? n : 256;
}

int launch_embedding_grad(const m2_embedding_grad_args& a, hipStream_t s) {
    const char* who = "embedding_grad";
    if (int rc = check_grad(a)) return rc;
    for (int d : {a.grad_dtype, a.out_dtype})
        M2_REQUIRE(d == M2_F32 || d == M2_BF16, M2_ERR_UNSUPPORTED, "%s: dtype %d", who, d);
    M2_REQUIRE(a.id_dtype == M2_I32 || a.id_dtype == M2_I64, M2_ERR_UNSUPPORTED, "%s: id dtype %d", who,
               a.id_dtype);
    M2_REQUIRE(a.ldg >= a.dim && a.ldo >= a.dim, M2_ERR_INVALID, "%s: row strides", who);
    M2_REQUIRE(a.out && (a.n == 0 || (a.ids && a.grad)), M2_ERR_INVALID, "%s: ids, grad and out are required",
               who);
    const GradPlan p = grad_plan(a);
    M2_REQUIRE(a.workspace && a.workspace_bytes >= (p.total ? p.total : 256), M2_ERR_WORKSPACE,
               "%s: workspace of %zu bytes needed, %zu given", who, p.total, a.workspace_bytes);
    if (a.n == 0 && a.accumulate) return M2_OK;
    char* ws = static_cast<char*>(a.workspace);
    auto at = [&](size_t o) { return reinterpret_cast<int32_t*>(ws + o); };
    SortArgs k{};
    k.ids = a.ids; k.used = reinterpret_cast<uint32_t*>(ws + p.used); k.hist = at(p.hist);
    k.vocab = a.vocab; k.padding = a.padding_idx; k.n = (int)a.n; k.id64 = a.id_dtype == M2_I64;
    k.bits = p.bits; k.words = p.words;
    int cur = 0;
    if (p.small) {
        // one launch (also for n == 0, which only clears the bitmap)
        k.nb = p.passes;
        k.keys_out = at(p.keys[0]); k.pos_out = at(p.pos[0]);
        hipLaunchKernelGGL(k_sort_small, dim3(1), dim3(SMALL_THREADS), 0, s, k);
    } else {
        k.nb = p.nb;
        for (int pass = 0; pass < p.passes; ++pass) {
            k.shift = pass * p.bits;
            k.keys_out = at(p.keys[cur]); k.pos_out = at(p.pos[cur]);
            hipLaunchKernelGGL(k_sort_hist, dim3(p.nb), dim3(SORT_THREADS), 0, s, k);
            hipLaunchKernelGGL(k_sort_scatter, dim3(p.nb), dim3(SORT_THREADS), 0, s, k,
                               (int)(pass == p.passes - 1));
            k.keys_in = k.keys_out; k.pos_in = k.pos_out;
            cur ^= 1;
        }
        cur ^= 1;
    }
    if (int rc = check_launch(who)) return rc;
    const int gs = (int)m2_dtype_size(a.grad_dtype), os = (int)m2_dtype_size(a.out_dtype);
    const int ev = gs == 2 ? 8 : 4;
    const bool vec = a.dim % 8 == 0 && a.ldg % 8 == 0 && a.ldo % 8 == 0 && al16(a.grad) && al16(a.out);
    ReduceArgs r{};
    r.keys = at(p.keys[cur]); r.pos = at(p.pos[cur]); r.used = k.used;
    r.grad = a.grad; r.out = a.out; r.part = reinterpret_cast<float*>(ws + p.part);
    r.ldg = a.ldg; r.ldo = a.ldo; r.ldp = p.ldp; r.vocab = a.vocab;
    r.n = (int)a.n; r.piece = p.piece; r.pieces = p.pieces; r.accumulate = a.accumulate;
    r.scale = a.scale; r.cols = (int)a.dim;
    const int V = vec ? 8 : 1;
    r.vecs = (int)(a.dim / V);
    r.slabs = (r.vecs + 511) / 512;
    const int per = (r.vecs + r.slabs - 1) / r.slabs;
    const int threads = (per + 63) / 64 * 64;
    M2_REQUIRE((int64_t)p.pieces * r.slabs < (1ll << 30), M2_ERR_UNSUPPORTED, "%s: too large", who);
    r.nred = p.pieces * r.slabs;
    const int64_t rows = (a.vocab + threads / 64 - 1) / (threads / 64);
    const unsigned fill = a.accumulate ? 0u : (unsigned)(rows < 4096 ? rows : 4096);
    if (r.nred + fill == 0) return M2_OK;
#define M2_SUMS(T, TO)                                         \
    do {                                                       \
        if (vec) launch_sums<T, TO, 8>(r, fill, threads, s);   \
        else launch_sums<T, TO, 1>(r, fill, threads, s);       \
    } while (0)
    if (gs == 2 && os == 2) M2_SUMS(bf16, bf16);
    else if (gs == 2) M2_SUMS(bf16, float);
    else if (os == 2) M2_SUMS(float, bf16);
    else M2_SUMS(float, float);
#undef M2_SUMS
    return check_launch(who);
}

}  // namespace m2
