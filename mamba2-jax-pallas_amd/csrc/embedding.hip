// embedding: out[n] = scale * weight[ids[n]], and its gradient
//   grad_weight[v] = scale * sum over {n : ids[n] == v} of grad[n]
// by sorted tokens.
//
// The lookup is a gather of whole rows: a wavefront per (row, column part), 16 bytes a
// lane, bound by HBM for many rows and by two dependent loads (id, row) for
// few: 16384 x 2560 bf16 25 us, 16 rows 2.8 us of GPU time in a call of 9.5.
//
// The gradient sorts (id, n) by id with a stable radix sort (equal ids keep the
// order of n), walks the sorted list in pieces of up to 32 entries, one
// workgroup each, with the sum of the current id's rows in registers, and
// writes each row that an id names once.  An id whose entries cross pieces
// (frequent tokens) leaves one partial row per piece, which a second kernel
// adds in order: no float atomics, so equal inputs give equal bits, and a token
// that is half of the batch is spread over as many workgroups as any others.
// The sort keeps one workgroup (of up to 16384 entries) or some (512 at most) busy; the rest of the
// chip meanwhile writes the zeros, which are most of a large vocabulary's gradient.  The rows that ids name are written twice that way, at
// most n rows; zeroing the others alone would have to wait for the sort.  Bound
// by HBM: grad read once, the result written once and those rows again.
//
// Up to 256 entries need neither sort nor partial rows: one launch, in which every entry
// looks for its id among the others and the first of an id adds up all of them, while
// further workgroups write the zeros of the rows that no id names (64 x 512 bf16 over 8000:
// 12.4 us a call, 17.5 with sort and join).
#include "m2_internal.h"

#include <type_traits>

namespace {

constexpr int SORT_THREADS = 256, SORT_ITEMS = 8, SORT_TILE = SORT_THREADS * SORT_ITEMS;
constexpr int SMALL_THREADS = 1024, SMALL_POS = 14, SMALL_N = 1 << SMALL_POS;
constexpr int MAX_BINS = 512;
// Workgroups of a pass over many entries: each counts, then moves, a contiguous run of tiles.  Every
// one of them adds up the counts of all, which is half a gigabyte read from the L2 at most; with a
// workgroup for each tile it would grow with the square of the entries.
constexpr int SORT_BLOCKS = 512;

M2_DEV int64_t load_id(const void* ids, int64_t i, int is64) {
    return is64 ? reinterpret_cast<const int64_t*>(ids)[i]
                : (int64_t) reinterpret_cast<const int32_t*>(ids)[i];
}

// V consecutive elements as floats, aligned as elements only
template <typename T, int V> struct Vec {
    float v[V];
    M2_DEV void load(const T* p) {
        if constexpr (V == 1) {
            v[0] = to_f32(*p);
        } else if constexpr (sizeof(T) == 2 && V == 8) {
            const u32x4 r = load16(p);
#pragma unroll
            for (int i = 0; i < 4; ++i) { v[2 * i] = bf16_lo(r[i]); v[2 * i + 1] = bf16_hi(r[i]); }
        } else if constexpr (sizeof(T) == 2) {
#pragma unroll
            for (int i = 0; i < V; ++i) v[i] = to_f32(p[i]);
        } else {
#pragma unroll
            for (int i = 0; i < V; i += 4) {
                const u32x4 r = load16(p + i);
#pragma unroll
                for (int j = 0; j < 4; ++j) v[i + j] = __uint_as_float(r[j]);
            }
        }
    }
    M2_DEV void store(T* p) const {
        if constexpr (V == 1) {
            *p = from_f32<T>(v[0]);
        } else if constexpr (sizeof(T) == 2 && V == 8) {
            store16(p, u32x4{pk_bf16(v[0], v[1]), pk_bf16(v[2], v[3]), pk_bf16(v[4], v[5]), pk_bf16(v[6], v[7])});
        } else if constexpr (sizeof(T) == 2) {
            typedef uint32_t Any __attribute__((ext_vector_type(2), aligned(2)));
            *reinterpret_cast<Any*>(p) = Any{pk_bf16(v[0], v[1]), pk_bf16(v[2], v[3])};
        } else {
#pragma unroll
            for (int i = 0; i < V; i += 4)
                store16(p + i, __builtin_bit_cast(u32x4, f32x4{v[i], v[i + 1], v[i + 2], v[i + 3]}));
        }
    }
};
// A row of cols elements in pieces of V (V == 1 where the row is shorter than 8): piece
// c begins at column at(c); the last one ends with the row, and its first skip(c) elements
// are its neighbour's too (computed twice, equal).
template <int V> M2_DEV int piece_at(int c, int cols) { return min(c * V, cols - V); }

// ---------------------------------------------------------------------------
// lookup
// ---------------------------------------------------------------------------
struct EmbedArgs {
    const void* ids;
    const void* w;
    void* out;
    int64_t n, vocab, ldw, ldo;
    int cols, vecs;    // elements of a row, V-element pieces of it
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
    const bool ok = id >= 0 && id < a.vocab;             // if not, row 0 is read and NaN written
    const T* src = static_cast<const T*>(a.w) + (ok ? id : 0) * a.ldw;
    T* dst = static_cast<T*>(a.out) + row * a.ldo;
    Vec<T, V> v[EMB_UN];
#pragma unroll
    for (int u = 0; u < EMB_UN; ++u)
        if (c0 + 64 * u < a.vecs) v[u].load(src + piece_at<V>(c0 + 64 * u, a.cols));
#pragma unroll
    for (int u = 0; u < EMB_UN; ++u) {
        if (c0 + 64 * u >= a.vecs) continue;
#pragma unroll
        for (int i = 0; i < V; ++i) v[u].v[i] = ok ? v[u].v[i] * a.scale : __builtin_nanf("");
        v[u].store(dst + piece_at<V>(c0 + 64 * u, a.cols));
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
    int64_t vocab, padding;
    int n, id64, shift, bits, nb;
    int tiles;                   // of SORT_TILE entries

    // of workgroup b: [tile(b), tile(b + 1))
    M2_DEV int tile(int b) const { return (int)((int64_t)tiles * b / nb); }
};

M2_DEV int32_t key_of(const SortArgs& a, int i) {
    const int64_t id = load_id(a.ids, i, a.id64);
    return id >= 0 && id < a.vocab && id != a.padding ? (int32_t)id : (int32_t)a.vocab;
}

// Zeros of the result, written by the workgroups that a sort's launch has to spare: rows
// [r0, r1), a contiguous range of bytes where the rows lie without gaps.
struct FillArgs {
    char* out;
    int64_t r0, r1, ldo, row;    // bytes
    int flat;                    // ldo == row, 16-byte aligned
    int nt;                      // past the caches
};
// Non-temporal zeros leave grad where its producer put it, in the 256 MB cache that they would
// fill, but run at HBM's rate, others at the cache's: 16384 x 2560 bf16 over 50288 (grad a
// third of the result) 82 us against 101, 2047 x 768 f32 over 50277 (a 25th) 46 against
// 34; the two meet at about an eighth.  Bytes of a workgroup: 64 KB with, 256 KB without.
constexpr int64_t FILL_BYTES = 64 << 10;

M2_DEV void fill(const FillArgs& f, int block, int blocks) {
    const u32x4 z = {0, 0, 0, 0};
    if (f.flat) {
        const int64_t b0 = f.r0 * f.row, n = (f.r1 - f.r0) * f.row / 16;
        u32x4* p = reinterpret_cast<u32x4*>(f.out + b0);
        const int64_t i0 = n * block / blocks, i1 = n * (block + 1) / blocks;
        if (f.nt) {
#pragma unroll 4
            for (int64_t i = i0 + threadIdx.x; i < i1; i += blockDim.x) __builtin_nontemporal_store(z, p + i);
        } else {
#pragma unroll 4
            for (int64_t i = i0 + threadIdx.x; i < i1; i += blockDim.x) p[i] = z;
        }
        // what 16-byte pieces leave of the last row
        if (block == 0 && threadIdx.x < (int)(((f.r1 - f.r0) * f.row - n * 16) >> 1))
            reinterpret_cast<uint16_t*>(p + n)[threadIdx.x] = 0;
        return;
    }
    const int nw = blockDim.x >> 6, lane = threadIdx.x & 63;
    for (int64_t r = f.r0 + (int64_t)block * nw + wave_id(); r < f.r1; r += (int64_t)blocks * nw) {
        char* p = f.out + r * f.ldo;
        // single elements (of 2 bytes) up to a 16-byte boundary and behind the last one
        int64_t head = (16 - ((uintptr_t)p & 15)) & 15;
        head = head < f.row ? head : f.row;
        const int64_t vecs = (f.row - head) >> 4, tail = head + vecs * 16;
        for (int64_t i = lane; i < vecs; i += 64) *reinterpret_cast<u32x4*>(p + head + i * 16) = z;
        if (2 * lane < head) reinterpret_cast<uint16_t*>(p)[lane] = 0;
        if (2 * lane < f.row - tail) reinterpret_cast<uint16_t*>(p + tail)[lane] = 0;
    }
}

__global__ void __launch_bounds__(SORT_THREADS) k_sort_hist(SortArgs a, FillArgs f) {
    __shared__ int h[MAX_BINS];
    const int bins = 1 << a.bits, t = threadIdx.x, b = blockIdx.x;
    if (b >= a.nb) return fill(f, b - a.nb, gridDim.x - a.nb);
    for (int d = t; d < bins; d += SORT_THREADS) h[d] = 0;
    __syncthreads();
    for (int tile = a.tile(b); tile < a.tile(b + 1); ++tile) {
#pragma unroll
        for (int j = 0; j < SORT_ITEMS; ++j) {
            const int i = tile * SORT_TILE + j * SORT_THREADS + t;
            if (i < a.n) {
                const int32_t k = a.keys_in ? a.keys_in[i] : key_of(a, i);
                atomicAdd(&h[(k >> a.shift) & (bins - 1)], 1);
            }
        }
    }
    __syncthreads();
    for (int d = t; d < bins; d += SORT_THREADS) a.hist[b * bins + d] = h[d];
}

// The lanes with this lane's digit of BITS bits, by one ballot per bit (lanes that are not `on`
// are nobody's).
template <int BITS> M2_DEV uint64_t wave_peers(int digit, bool on) {
    const uint64_t all = __ballot(on);
    uint32_t lo = (uint32_t)all, hi = (uint32_t)(all >> 32);
#pragma unroll
    for (int b = 0; b < BITS; ++b) {
        const int one = (digit << (31 - b)) >> 31;          // 0 or all bits
        const uint64_t m = __ballot(one != 0);
        lo &= ~((uint32_t)m ^ (uint32_t)one);
        hi &= ~((uint32_t)(m >> 32) ^ (uint32_t)one);
    }
    return (uint64_t)hi << 32 | lo;
}
// The places of a thread's IT entries among those of their wavefront with the same digit, in
// the order of j and of the lanes; their numbers are left in cnt.  Three passes, so that
// the LDS accesses of all entries are under way together.
template <int BITS, int IT, typename D, typename ON>
M2_DEV void wave_ranks(D digit, ON on, int* cnt, int (&rank)[IT]) {
    const int lane = threadIdx.x & 63;
    const uint64_t below = (1ull << lane) - 1;
    int first[IT];
#pragma unroll
    for (int j = 0; j < IT; ++j) {
        const uint64_t peers = wave_peers<BITS>(digit(j), on(j));
        first[j] = peers ? __ffsll((unsigned long long)peers) - 1 : 0;
        rank[j] = __popcll(peers & below);
        // the first of the lanes counts them all
        if (on(j) && rank[j] == 0) rank[j] = atomicAdd(&cnt[digit(j)], __popcll(peers)) << 6;
    }
#pragma unroll
    for (int j = 0; j < IT; ++j) {
        const int base = __shfl(rank[j], first[j]) >> 6;
        rank[j] = base + (lane == first[j] ? 0 : rank[j]);
    }
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

__global__ void __launch_bounds__(SORT_THREADS) k_sort_scatter(SortArgs a, FillArgs f) {
    constexpr int NW = SORT_THREADS / 64;
    __shared__ int cnt[NW][MAX_BINS];
    __shared__ int tmp[NW];
    const int bins = 1 << a.bits, t = threadIdx.x, b = blockIdx.x, w = wave_id(), lane = t & 63;
    if (b >= a.nb) return fill(f, b - a.nb, gridDim.x - a.nb);
    int32_t key[SORT_ITEMS], pos[SORT_ITEMS];
    int rank[SORT_ITEMS];
    int tile = a.tile(b), base = 0;
    const int end = a.tile(b + 1);
    auto load = [&]() {
        base = tile * SORT_TILE + w * 64 * SORT_ITEMS + lane;
#pragma unroll
        for (int j = 0; j < SORT_ITEMS; ++j) {
            const int i = base + 64 * j, at = min(i, a.n - 1);      // used below n
            key[j] = a.keys_in ? a.keys_in[at] : key_of(a, at);
            pos[j] = a.pos_in ? a.pos_in[at] : i;
        }
    };
    load();
    // where each digit of this block begins: the entries of smaller digits in all blocks and
    // of this digit in earlier blocks.  Thread t owns digits D t .. D t + D - 1 (a fixed order
    // for the prefix sum).
    constexpr int D = MAX_BINS / SORT_THREADS;
    int next[D], tot[D], mine = 0;
#pragma unroll
    for (int k = 0; k < D; ++k) {
        const int d = t * D + k;
        tot[k] = next[k] = 0;
        if (d < bins)
#pragma unroll 8
            for (int q = 0; q < a.nb; ++q) {
                const int c = a.hist[q * bins + d];
                tot[k] += c;
                next[k] += q < b ? c : 0;
            }
        mine += tot[k];
    }
    int start = block_excl<SORT_THREADS>(mine, tmp);
#pragma unroll
    for (int k = 0; k < D; ++k) {
        next[k] += start;
        start += tot[k];
    }
    for (;;) {
        for (int d = t; d < NW * MAX_BINS; d += SORT_THREADS) (&cnt[0][0])[d] = 0;
        __syncthreads();
        wave_ranks<9, SORT_ITEMS>([&](int j) { return (key[j] >> a.shift) & (bins - 1); },
                                  [&](int j) { return base + 64 * j < a.n; }, cnt[w], rank);
        __syncthreads();
        // where each (digit, wavefront) of this tile begins
#pragma unroll
        for (int k = 0; k < D; ++k) {
#pragma unroll
            for (int q = 0; q < NW; ++q) {
                const int c = cnt[q][t * D + k];
                cnt[q][t * D + k] = next[k];
                next[k] += c;
            }
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < SORT_ITEMS; ++j) {
            if (base + 64 * j >= a.n) continue;
            const int p = cnt[w][(key[j] >> a.shift) & (bins - 1)] + rank[j];
            a.keys_out[p] = key[j];
            a.pos_out[p] = pos[j];
        }
        if (++tile >= end) return;
        load();
        __syncthreads();             // everybody has its places
    }
}

// Up to SMALL_N entries of a vocabulary below 2^18: every pass in one workgroup, the list
// in LDS between the passes, an entry in one word (key, position).  a.nb passes of BITS bits;
// 16384 entries are 16 words a thread.  One workgroup on one CU, bound by its vector
// instructions (the ballots): 26 us at 16384 entries of 16 bits, 5 at 1000; the whole
// gradient of 8192 x 64 takes 24.5 us (32.5 with 16 words a thread), of 16384 x 64 43, and
// of 20000 x 64 by the sort over many workgroups 41.
template <int IT, int BITS>
__global__ void __launch_bounds__(SMALL_THREADS) k_sort_small(SortArgs a, FillArgs f) {
    constexpr int NW = SMALL_THREADS / 64;
    __shared__ int cnt[NW][MAX_BINS];
    __shared__ uint32_t list[SMALL_THREADS * IT];
    __shared__ int tmp[NW];
    if (blockIdx.x > 0) return fill(f, blockIdx.x - 1, gridDim.x - 1);
    constexpr int bins = 1 << BITS;
    const int t = threadIdx.x, w = wave_id();
    const int base = w * 64 * IT + (t & 63);
    uint32_t e[IT];
    int rank[IT];
#pragma unroll
    for (int j = 0; j < IT; ++j) {
        const int i = base + 64 * j;
        e[j] = (uint32_t)key_of(a, min(i, a.n - 1)) << SMALL_POS | (uint32_t)i;      // used below n
    }
    for (int pass = 0; pass < a.nb; ++pass) {
        const int shift = SMALL_POS + pass * BITS;
        for (int d = t; d < NW * bins; d += SMALL_THREADS) cnt[d >> BITS][d & (bins - 1)] = 0;
        __syncthreads();
        wave_ranks<BITS, IT>([&](int j) { return (int)(e[j] >> shift) & (bins - 1); },
                             [&](int j) { return base + 64 * j < a.n; }, cnt[w], rank);
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
        for (int j = 0; j < IT; ++j)
            if (base + 64 * j < a.n) list[cnt[w][(e[j] >> shift) & (bins - 1)] + rank[j]] = e[j];
        __syncthreads();
#pragma unroll
        for (int j = 0; j < IT; ++j) e[j] = list[base + 64 * j];
    }
#pragma unroll
    for (int j = 0; j < IT; ++j) {
        const int i = base + 64 * j;
        if (i >= a.n) continue;
        a.keys_out[i] = (int32_t)(e[j] >> SMALL_POS);
        a.pos_out[i] = (int32_t)(e[j] & (SMALL_N - 1));
    }
}

// ---------------------------------------------------------------------------
// the sums
// ---------------------------------------------------------------------------
struct ReduceArgs {
    const int32_t* keys;
    const int32_t* pos;
    const void* grad;
    void* out;
    float* part;             // [pieces][2][ldp]: of a row begun before the piece / left unfinished
    int64_t ldg, ldo, ldp, vocab;
    int n, piece, pieces;    // entries per piece
    int cols, vecs, slabs;   // elements of a row, V-element pieces of it, split over `slabs` workgroups
    int accumulate;
    float scale;
};

template <typename TO, int V>
M2_DEV void put_row(const ReduceArgs& a, int32_t key, int c, Vec<float, V> s) {
    const int col = piece_at<V>(c, a.cols), skip = c * V - col;
    TO* p = static_cast<TO*>(a.out) + (int64_t)key * a.ldo + col;
#pragma unroll
    for (int i = 0; i < V; ++i) s.v[i] *= a.scale;
    if (a.accumulate && skip) {          // the neighbour adds the others
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (i >= skip) p[i] = from_f32<TO>(s.v[i] + to_f32(p[i]));
        return;
    }
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

constexpr int MAX_PIECE = 32;

template <typename T, typename TO, int V>
__global__ void __launch_bounds__(512) k_embed_sum(ReduceArgs a) {
    const int t = threadIdx.x, lane = t & 63;
    const int p = blockIdx.x / a.slabs, slab = blockIdx.x % a.slabs;
    const int per = (a.vecs + a.slabs - 1) / a.slabs;
    const int c = slab * per + t;
    const bool on = t < per && c < a.vecs;
    const int e0 = p * a.piece, cnt = min(a.n - e0, a.piece);
    // the piece's entries, one a lane (every wavefront has them all)
    const int q = e0 + min(lane, cnt - 1);
    const int32_t keys = a.keys[q], pos = a.pos[q];
    const int32_t before = p > 0 ? a.keys[e0 - 1] : -1, after = e0 + cnt < a.n ? a.keys[e0 + cnt] : -1;
    const int col = piece_at<V>(on ? c : 0, a.cols);
    const T* g = static_cast<const T*>(a.grad) + col;
    int32_t key = __builtin_amdgcn_readlane(keys, 0);
    bool head = before == key;            // the row began in an earlier piece
    Vec<float, V> s;
#pragma unroll
    for (int i = 0; i < V; ++i) s.v[i] = 0.f;
    auto flush = [&](bool more) {
        if (!on || key >= a.vocab) return;
        if (!head && !more) put_row<TO, V>(a, key, c, s);
        else s.store(a.part + ((int64_t)p * 2 + (head ? 0 : 1)) * a.ldp + col);
    };
    auto add = [&](int e, auto count) {
        constexpr int UN = decltype(count)::value;
        Vec<T, V> v[UN];
#pragma unroll
        for (int u = 0; u < UN; ++u) v[u].load(g + (int64_t)__builtin_amdgcn_readlane(pos, e + u) * a.ldg);
#pragma unroll
        for (int u = 0; u < UN; ++u) {
            const int32_t k = __builtin_amdgcn_readlane(keys, e + u);
            if (k != key) {
                flush(false);
                key = k;
                head = false;
#pragma unroll
                for (int i = 0; i < V; ++i) s.v[i] = 0.f;
            }
#pragma unroll
            for (int i = 0; i < V; ++i) s.v[i] += v[u].v[i];
        }
    };
    int e = 0;
    for (; e + 8 <= cnt; e += 8) add(e, std::integral_constant<int, 8>());
    if (e + 4 <= cnt) { add(e, std::integral_constant<int, 4>()); e += 4; }
    for (; e < cnt; ++e) add(e, std::integral_constant<int, 1>());
    flush(after == key);
}

// The rows that cross pieces: the piece in which such a row begins adds its
// partial rows in order.
// A frequent token's partial rows are a chain of loads that one workgroup waits for:
// narrow column parts and 16 rows in flight.
constexpr int JOIN_THREADS = 256;
template <typename TO, int V>
__global__ void __launch_bounds__(JOIN_THREADS) k_embed_join(ReduceArgs a) {
    const int p = blockIdx.x / a.slabs, slab = blockIdx.x % a.slabs, t = threadIdx.x;
    const int e0 = p * a.piece, e1 = min(a.n, e0 + a.piece);
    if (e1 >= a.n) return;
    const int32_t key = a.keys[e1 - 1], first = a.keys[e0], before = p > 0 ? a.keys[e0 - 1] : -1;
    if (key >= a.vocab || a.keys[e1] != key) return;
    if (first == key && before == key) return;      // begun before this piece
    const int c = slab * JOIN_THREADS + t;
    // pieces p + 1 .. p + m begin with the row
    int m = 0;
    for (int q0 = p + 1; q0 < a.pieces; q0 += 64) {
        const int64_t at = (int64_t)(q0 + (t & 63)) * a.piece;
        const uint64_t same = __ballot(at < a.n && a.keys[at] == key);
        const int run = ~same ? __ffsll((unsigned long long)~same) - 1 : 64;
        m += run;
        if (run < 64) break;
    }
    if (c >= a.vecs) return;
    Vec<float, V> s;
    const int col = piece_at<V>(c, a.cols);
    s.load(a.part + ((int64_t)p * 2 + 1) * a.ldp + col);
    const float* from = a.part + (int64_t)(p + 1) * 2 * a.ldp + col;
    auto add = [&](auto count) {
        constexpr int UN = decltype(count)::value;
        Vec<float, V> v[UN];
#pragma unroll
        for (int u = 0; u < UN; ++u) v[u].load(from + (int64_t)u * 2 * a.ldp);
#pragma unroll
        for (int u = 0; u < UN; ++u)
#pragma unroll
            for (int i = 0; i < V; ++i) s.v[i] += v[u].v[i];
        from += (int64_t)UN * 2 * a.ldp;
        m -= UN;
    };
    while (m >= 16) add(std::integral_constant<int, 16>());
    while (m >= 4) add(std::integral_constant<int, 4>());
    while (m > 0) add(std::integral_constant<int, 1>());
    put_row<TO, V>(a, key, c, s);
}

// ---------------------------------------------------------------------------
// few entries: the whole gradient in one launch
// ---------------------------------------------------------------------------
constexpr int FEW_N = 256, FEW_THREADS = 256, FEW_ROWS = 4096;
struct FewArgs {
    const void* ids;
    int64_t padding;
    int64_t row_bytes, ld_bytes;
    int id64, nred, rows;    // workgroups that sum; rows that one of the others zeroes
};

template <typename T, typename TO, int V>
__global__ void __launch_bounds__(FEW_THREADS) k_embed_few(ReduceArgs a, FewArgs f) {
    __shared__ uint8_t named[FEW_ROWS];
    const int t = threadIdx.x, lane = t & 63;
    auto key_at = [&](int i) {
        const int64_t id = load_id(f.ids, i, f.id64);
        return id >= 0 && id < a.vocab && id != f.padding ? (int32_t)id : -1;
    };
    if ((int)blockIdx.x >= f.nred) {
        const int64_t r0 = (int64_t)(blockIdx.x - f.nred) * f.rows;
        const int rows = (int)min((int64_t)f.rows, a.vocab - r0);
        for (int i = t; i < rows; i += FEW_THREADS) named[i] = 0;
        __syncthreads();
        if (t < a.n) {
            const int64_t r = key_at(t) - r0;
            if (r >= 0 && r < rows) named[r] = 1;
        }
        __syncthreads();
        // 16-byte pieces, the last one of a row ends with it; rows shorter than that by their
        // 2-byte elements
        char* out = static_cast<char*>(a.out) + r0 * f.ld_bytes;
        const int bytes = f.row_bytes < 16 ? 2 : 16;
        const uint32_t per = (uint32_t)((f.row_bytes + bytes - 1) / bytes);
        const uint32_t all = per * rows;
        for (uint32_t i = t; i < all; i += FEW_THREADS) {
            const uint32_t r = i / per, c = i - r * per;
            if (named[r]) continue;
            char* p = out + r * f.ld_bytes + min((int64_t)c * bytes, f.row_bytes - bytes);
            if (bytes == 16) store16(p, u32x4{0, 0, 0, 0});
            else *reinterpret_cast<uint16_t*>(p) = 0;
        }
        return;
    }
    const int e = blockIdx.x / a.slabs, slab = blockIdx.x % a.slabs;
    const int32_t key = key_at(e);
    if (key < 0) return;
    uint64_t same[FEW_N / 64];            // entries with this id
#pragma unroll
    for (int j = 0; j < FEW_N / 64; ++j) {
        const int i = 64 * j + lane;
        same[j] = __ballot(i < a.n && key_at(i) == key);
    }
    // an earlier entry has it: that one's workgroup adds them all
#pragma unroll
    for (int j = 0; j < FEW_N / 64; ++j)
        if (64 * j <= e && (same[j] & ((e >> 6) == j ? (1ull << (e & 63)) - 1 : ~0ull))) return;
    const int c = slab * FEW_THREADS + t;
    if (c >= a.vecs) return;
    const T* g = static_cast<const T*>(a.grad) + piece_at<V>(c, a.cols);
    Vec<float, V> s;
#pragma unroll
    for (int i = 0; i < V; ++i) s.v[i] = 0.f;
#pragma unroll
    for (int j = 0; j < FEW_N / 64; ++j) {
        uint64_t m = same[j];
        while (m) {
            constexpr int UN = 4;
            Vec<T, V> v[UN];
            int k = 0;
#pragma unroll
            for (int u = 0; u < UN; ++u)
                if (m) {
                    const int at = 64 * j + __ffsll((unsigned long long)m) - 1;
                    m &= m - 1;
                    v[u].load(g + (int64_t)at * a.ldg);
                    k = u + 1;
                }
#pragma unroll
            for (int u = 0; u < UN; ++u)
                if (u < k)
#pragma unroll
                    for (int i = 0; i < V; ++i) s.v[i] += v[u].v[i];
        }
    }
    put_row<TO, V>(a, key, c, s);
}

size_t align256(size_t v) { return (v + 255) & ~size_t(255); }

struct GradPlan {
    int bits, passes, tiles, nb, piece, pieces;
    int64_t ldp;
    bool small;
    size_t keys[2], pos[2], hist, part, total;
};

GradPlan grad_plan(const m2_embedding_grad_args& a) {
    GradPlan p{};
    int kb = 1;
    while ((1ll << kb) <= a.vocab) ++kb;          // keys 0 .. vocab
    p.passes = (kb + 8) / 9;
    p.bits = (kb + p.passes - 1) / p.passes;
    p.small = a.n <= SMALL_N && kb <= 32 - SMALL_POS;
    p.tiles = (int)((a.n + SORT_TILE - 1) / SORT_TILE);
    p.nb = p.tiles < SORT_BLOCKS ? p.tiles : SORT_BLOCKS;
    // entries per piece: about 512 pieces, so that every CU has two, of 4 to 32
    // entries (longer pieces leave fewer partial rows, shorter ones more
    // workgroups to a small batch)
    int64_t e = a.n / 512;
    p.piece = e < 4 ? 4 : e > MAX_PIECE ? MAX_PIECE : (int)e;
    p.pieces = (int)((a.n + p.piece - 1) / p.piece);
    p.ldp = (a.dim + 7) / 8 * 8;
    size_t at = 0;
    auto take = [&](size_t bytes) { const size_t r = at; at += align256(bytes); return r; };
    for (int i = 0; i < 2; ++i) { p.keys[i] = take(4 * (size_t)a.n); p.pos[i] = take(4 * (size_t)a.n); }
    p.hist = take(4 * (size_t)p.nb << p.bits);
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
    M2_REQUIRE(a.n <= FEW_N || (int64_t)grad_plan(a).pieces * (a.dim / 256 + 1) < (1ll << 30), M2_ERR_UNSUPPORTED,
               "%s: too large (n %lld, dim %lld)", who, (long long)a.n, (long long)a.dim);
    return M2_OK;
}

template <typename T, typename TO, int V>
void launch_sums(const ReduceArgs& r, int threads, hipStream_t s) {
    hipLaunchKernelGGL((k_embed_sum<T, TO, V>), dim3((unsigned)(r.pieces * r.slabs)), dim3(threads), 0, s, r);
    if (r.pieces > 1) {
        constexpr int JV = V == 1 ? 1 : 4;
        ReduceArgs j = r;
        j.vecs = (r.cols + JV - 1) / JV;
        j.slabs = (j.vecs + JOIN_THREADS - 1) / JOIN_THREADS;
        hipLaunchKernelGGL((k_embed_join<TO, JV>), dim3((unsigned)(r.pieces * j.slabs)), dim3(JOIN_THREADS), 0, s,
                           j);
    }
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
    const int ev = 16 / (int)m2_dtype_size(a.dtype);
    const bool vec = a.dim >= ev;
    EmbedArgs k{a.ids, a.weight, a.out, a.n, a.vocab, a.ldw, a.ldo, (int)a.dim, 0, 0, a.scale, a.id_dtype == M2_I64};
    k.vecs = (int)(vec ? (a.dim + ev - 1) / ev : a.dim);
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
    return a.n <= FEW_N ? 256 : grad_plan(a).total;
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
    const size_t need = embedding_grad_workspace(a);
    M2_REQUIRE(a.workspace && a.workspace_bytes >= need, M2_ERR_WORKSPACE,
               "%s: workspace of %zu bytes needed, %zu given", who, need, a.workspace_bytes);
    if (a.n == 0 && a.accumulate) return M2_OK;
    if (a.n <= FEW_N) {
        ReduceArgs r{};
        const bool vec = a.dim >= 8;
        const int64_t osz = (int64_t)m2_dtype_size(a.out_dtype);
        r.grad = a.grad; r.out = a.out; r.ldg = a.ldg; r.ldo = a.ldo; r.vocab = a.vocab;
        r.n = (int)a.n; r.cols = (int)a.dim; r.accumulate = a.accumulate; r.scale = a.scale;
        r.vecs = (int)(vec ? (a.dim + 7) / 8 : a.dim);
        r.slabs = (r.vecs + FEW_THREADS - 1) / FEW_THREADS;
        FewArgs f{a.ids, a.padding_idx, a.dim * osz, a.ldo * osz, a.id_dtype == M2_I64, (int)a.n * r.slabs, 0};
        const int64_t rows = (FILL_BYTES + f.row_bytes - 1) / f.row_bytes;
        f.rows = (int)(rows < FEW_ROWS ? rows : FEW_ROWS);
        const int64_t zero = a.accumulate ? 0 : (a.vocab + f.rows - 1) / f.rows;
        const dim3 grid((unsigned)(f.nred + zero)), thr(FEW_THREADS);
#define M2_FEW(T, TO)                                                                              \
    do {                                                                                           \
        if (vec) hipLaunchKernelGGL((k_embed_few<T, TO, 8>), grid, thr, 0, s, r, f);               \
        else hipLaunchKernelGGL((k_embed_few<T, TO, 1>), grid, thr, 0, s, r, f);                   \
    } while (0)
        if (a.grad_dtype == M2_BF16 && a.out_dtype == M2_BF16) M2_FEW(bf16, bf16);
        else if (a.grad_dtype == M2_BF16) M2_FEW(bf16, float);
        else if (a.out_dtype == M2_BF16) M2_FEW(float, bf16);
        else M2_FEW(float, float);
#undef M2_FEW
        return check_launch(who);
    }
    char* ws = static_cast<char*>(a.workspace);
    auto at = [&](size_t o) { return reinterpret_cast<int32_t*>(ws + o); };
    SortArgs k{};
    k.ids = a.ids; k.hist = at(p.hist);
    k.vocab = a.vocab; k.padding = a.padding_idx; k.n = (int)a.n; k.id64 = a.id_dtype == M2_I64;
    k.bits = p.bits;
    const int64_t osz = (int64_t)m2_dtype_size(a.out_dtype);
    FillArgs f{static_cast<char*>(a.out), 0, 0, a.ldo * osz, a.dim * osz, 0, 0};
    f.nt = 8 * a.n * (int64_t)m2_dtype_size(a.grad_dtype) >= a.vocab * osz;
    const int64_t fill_bytes = f.nt ? FILL_BYTES : 4 * FILL_BYTES;
    f.flat = a.ldo == a.dim && al16(a.out);
    // workgroups that write the zeros of rows r0 .. r1: a multiple of 16 rows keeps the next
    // part of a flat range on a 16-byte boundary
    const int parts = p.small ? 1 : 2 * p.passes;
    auto zeros = [&](int i, int64_t most) -> unsigned {
        if (a.accumulate) return 0;
        f.r0 = a.vocab * i / parts / 16 * 16;
        f.r1 = i + 1 == parts ? a.vocab : a.vocab * (i + 1) / parts / 16 * 16;
        const int64_t b = ((f.r1 - f.r0) * f.row + fill_bytes - 1) / fill_bytes;
        return (unsigned)(b < most ? b : most);
    };
    int cur = 0;
    if (p.small) {
        // one launch
        k.nb = p.passes;
        k.keys_out = at(p.keys[0]); k.pos_out = at(p.pos[0]);
        const dim3 grid(1 + zeros(0, 8192)), thr(SMALL_THREADS);
        auto sort = [&](auto bits) {
            constexpr int B = decltype(bits)::value;
            auto run = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, thr, 0, s, k, f); };
            if (a.n <= SMALL_THREADS) run(k_sort_small<1, B>);
            else if (a.n <= 2 * SMALL_THREADS) run(k_sort_small<2, B>);
            else if (a.n <= 4 * SMALL_THREADS) run(k_sort_small<4, B>);
            else if (a.n <= 8 * SMALL_THREADS) run(k_sort_small<8, B>);
            else if (a.n <= 12 * SMALL_THREADS) run(k_sort_small<12, B>);
            else run(k_sort_small<16, B>);
        };
        // bits and words a thread as constants: the ballots are most of the time, and those of
        // absent bits and entries cost as much
        if (p.bits <= 7) sort(std::integral_constant<int, 7>());
        else if (p.bits == 8) sort(std::integral_constant<int, 8>());
        else sort(std::integral_constant<int, 9>());
    } else {
        k.nb = p.nb;
        k.tiles = p.tiles;
        for (int pass = 0; pass < p.passes; ++pass) {
            k.shift = pass * p.bits;
            k.keys_out = at(p.keys[cur]); k.pos_out = at(p.pos[cur]);
            unsigned z = zeros(2 * pass, 8192);
            hipLaunchKernelGGL(k_sort_hist, dim3(p.nb + z), dim3(SORT_THREADS), 0, s, k, f);
            z = zeros(2 * pass + 1, 8192);
            hipLaunchKernelGGL(k_sort_scatter, dim3(p.nb + z), dim3(SORT_THREADS), 0, s, k, f);
            k.keys_in = k.keys_out; k.pos_in = k.pos_out;
            cur ^= 1;
        }
        cur ^= 1;
    }
    if (int rc = check_launch(who)) return rc;
    const int gs = (int)m2_dtype_size(a.grad_dtype), os = (int)m2_dtype_size(a.out_dtype);
    const bool vec = a.dim >= 8;
    ReduceArgs r{};
    r.keys = at(p.keys[cur]); r.pos = at(p.pos[cur]);
    r.grad = a.grad; r.out = a.out; r.part = reinterpret_cast<float*>(ws + p.part);
    r.ldg = a.ldg; r.ldo = a.ldo; r.ldp = p.ldp; r.vocab = a.vocab;
    r.n = (int)a.n; r.piece = p.piece; r.pieces = p.pieces; r.accumulate = a.accumulate;
    r.scale = a.scale;
    const int V = vec ? 8 : 1;
    r.cols = (int)a.dim;
    r.vecs = (int)((a.dim + V - 1) / V);
    r.slabs = (r.vecs + 511) / 512;
    const int per = (r.vecs + r.slabs - 1) / r.slabs;
    const int threads = (per + 63) / 64 * 64;
#define M2_SUMS(T, TO)                                         \
    do {                                                       \
        if (vec) launch_sums<T, TO, 8>(r, threads, s);   \
        else launch_sums<T, TO, 1>(r, threads, s);       \
    } while (0)
    if (gs == 2 && os == 2) M2_SUMS(bf16, bf16);
    else if (gs == 2) M2_SUMS(bf16, float);
    else if (os == 2) M2_SUMS(float, bf16);
    else M2_SUMS(float, float);
#undef M2_SUMS
    return check_launch(who);
}

}  // namespace m2
