// clip_grad_norm: the 2-norm over all values of many tensors, and the tensors
// times min(1, max_norm / (norm + eps)).
//
// Bound by HBM: every tensor is read for the norm and read again and written for the
// result (the scale is not known before the last value is).  The tensors' table goes to
// the workspace through kernel arguments, 136 at a time (a copy from the host would
// neither be captured into a graph nor run without waiting); then one launch
// reads everything and one scales it, so that one large embedding and a hundred small
// vectors take one pass.  The workgroups share the tensors' pieces of 16 KB evenly,
// a contiguous range each.  The squares are summed in float64 per thread (the vector
// units do that well above the rate at which HBM brings the values in): no square
// overflows and long sums lose nothing, and the order is fixed, so equal inputs give equal
// bits.  Every workgroup of the second pass adds the first one's sums up by itself,
// and walks its pieces in the opposite order: what the first pass read last is still in the
// 256 MB last-level cache.  130m float32 gradients (515 MB, 218 tensors): 300 us; 1.3b bf16
// (2.7 GB): 1.5 ms, 5.4 TB/s of the three transfers.
#include "m2_internal.h"

namespace {

constexpr int NT = 256;               // threads of a workgroup
constexpr int BATCH = 136;            // table entries that travel with one launch (below 4 KB)
constexpr int PIECE_BYTES = 16 << 10;
constexpr int MAXWG = 2048;           // 8 workgroups on each CU

struct Entry {
    const void* in;
    void* out;
    int64_t n;
    int64_t first;                    // number of pieces before this tensor
    int64_t bf;
};
struct Batch {
    const void* in[BATCH];
    void* out[BATCH];
    int64_t n[BATCH];                 // ~n: bf16
    uint32_t first[BATCH];            // behind base
    int64_t base;
    int count;
};
struct PassArgs {
    const Entry* table;
    int64_t count, pieces;
    double* part;                     // sums of the first pass, one a workgroup
    float* norm;                      // out
    float max_norm, eps;
    int parts;
};

__global__ void __launch_bounds__(256) k_table(Batch b, Entry* to) {
    const int i = threadIdx.x;
    if (i >= b.count) return;
    const int64_t n = b.n[i];
    to[i] = Entry{b.in[i], b.out[i], n < 0 ? ~n : n, b.base + b.first[i], n < 0};
}

M2_DEV double block_sum(double v, double* red) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    double s = 0;
#pragma unroll
    for (int j = 0; j < NT / 64; ++j) s += red[j];
    __syncthreads();
    return s;
}

// The tensor that piece p belongs to: the number of tensors that begin at or before it
M2_DEV int64_t find(const PassArgs& a, int64_t p, int* red) {
    int c = 0;
    for (int64_t i = threadIdx.x; i < a.count; i += NT) c += a.table[i].first <= p;
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) c += __shfl_xor(c, o);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = c;
    __syncthreads();
    int s = 0;
#pragma unroll
    for (int j = 0; j < NT / 64; ++j) s += red[j];
    return __builtin_amdgcn_readfirstlane(s - 1);
}

// Elements [i0, i1) of a tensor: single ones up to a 16-byte boundary of `p`, whole
// 16-byte pieces, single ones at the end.  f1(i): one element; fv(i): E of them.
template <int E, typename F1, typename FV>
M2_DEV void walk(const void* p, int es, int64_t i0, int64_t i1, F1 f1, FV fv) {
    const int t = threadIdx.x;
    const uintptr_t b = (uintptr_t)p + i0 * es;
    int64_t head = (int64_t)((16 - (b & 15)) & 15) / es;
    if (head > i1 - i0) head = i1 - i0;
    const int64_t a0 = i0 + head;
    const int nv = (int)((i1 - a0) / E);
    if (t < head) f1(i0 + t);
#pragma unroll 4
    for (int v = t; v < nv; v += NT) fv(a0 + (int64_t)v * E);
    const int64_t tail = a0 + (int64_t)nv * E;
    if (tail + t < i1) f1(tail + t);
}

__global__ void __launch_bounds__(NT) k_sumsq(PassArgs a) {
    __shared__ double red[NT / 64];
    __shared__ int found[NT / 64];
    const int64_t p0 = a.pieces * blockIdx.x / gridDim.x, p1 = a.pieces * (blockIdx.x + 1) / gridDim.x;
    double s = 0;
    int64_t ti = find(a, p0, found);
    Entry e = a.table[ti];
    int64_t end = ti + 1 < a.count ? a.table[ti + 1].first : a.pieces;
    for (int64_t p = p0; p < p1; ++p) {
        if (p >= end) {
            e = a.table[++ti];
            end = ti + 1 < a.count ? a.table[ti + 1].first : a.pieces;
        }
        if (e.bf) {
            const int64_t i0 = (p - e.first) * (PIECE_BYTES / 2), i1 = min(e.n, i0 + PIECE_BYTES / 2);
            const bf16* x = static_cast<const bf16*>(e.in);
            walk<8>(x, 2, i0, i1,
                    [&](int64_t i) { const double v = (float)x[i]; s = fma(v, v, s); },
                    [&](int64_t i) {
                        const u32x4 r = *reinterpret_cast<const u32x4*>(x + i);
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const double lo = bf16_lo(r[j]), hi = bf16_hi(r[j]);
                            s = fma(lo, lo, s);
                            s = fma(hi, hi, s);
                        }
                    });
        } else {
            const int64_t i0 = (p - e.first) * (PIECE_BYTES / 4), i1 = min(e.n, i0 + PIECE_BYTES / 4);
            const float* x = static_cast<const float*>(e.in);
            walk<4>(x, 4, i0, i1, [&](int64_t i) { const double v = x[i]; s = fma(v, v, s); },
                    [&](int64_t i) {
                        const f32x4 r = *reinterpret_cast<const f32x4*>(x + i);
#pragma unroll
                        for (int j = 0; j < 4; ++j) { const double v = r[j]; s = fma(v, v, s); }
                    });
        }
    }
    s = block_sum(s, red);
    if (threadIdx.x == 0) a.part[blockIdx.x] = s;
}

// the norm, from the workgroups' sums in a fixed order
M2_DEV float norm_of(const PassArgs& a, double* red) {
    double s = 0;
    for (int i = threadIdx.x; i < a.parts; i += NT) s += a.part[i];
    return (float)sqrt(block_sum(s, red));
}
__global__ void __launch_bounds__(NT) k_norm(PassArgs a) {
    __shared__ double red[NT / 64];
    const float norm = norm_of(a, red);
    if (threadIdx.x == 0) *a.norm = norm;
}

// PAST: the results past the caches
template <bool PAST> __global__ void __launch_bounds__(NT) k_scale(PassArgs a) {
    __shared__ double red[NT / 64];
    __shared__ int found[NT / 64];
    const float norm = norm_of(a, red);
    if (blockIdx.x == 0 && threadIdx.x == 0) *a.norm = norm;
    float c = a.max_norm / (norm + a.eps);
    c = c >= 1.f ? 1.f : c;                    // a norm that is not a number stays one here
    // the opposite order of k_sumsq
    const int b = gridDim.x - 1 - blockIdx.x;
    const int64_t p0 = a.pieces * b / gridDim.x, p1 = a.pieces * (b + 1) / gridDim.x;
    if (p0 >= p1) return;
    int64_t ti = find(a, p1 - 1, found);
    Entry e = a.table[ti];
    for (int64_t p = p1 - 1; p >= p0; --p) {
        if (p < e.first) e = a.table[--ti];
        if (c == 1.f && e.in == e.out) continue;      // in place, nothing to do
        // input and output on the same 16-byte phase: whole pieces of both
        const bool same = (((uintptr_t)e.in ^ (uintptr_t)e.out) & 15) == 0;
        if (e.bf) {
            const int64_t i0 = (p - e.first) * (PIECE_BYTES / 2), i1 = min(e.n, i0 + PIECE_BYTES / 2);
            const bf16* x = static_cast<const bf16*>(e.in);
            bf16* y = static_cast<bf16*>(e.out);
            walk<8>(x, 2, i0, i1, [&](int64_t i) { y[i] = (bf16)((float)x[i] * c); },
                    [&](int64_t i) {
                        const u32x4 r = *reinterpret_cast<const u32x4*>(x + i);
                        u32x4 o;
#pragma unroll
                        for (int j = 0; j < 4; ++j) o[j] = pk_bf16(bf16_lo(r[j]) * c, bf16_hi(r[j]) * c);
                        if (!same) store16(y + i, o);
                        else if constexpr (PAST) __builtin_nontemporal_store(o, reinterpret_cast<u32x4*>(y + i));
                        else *reinterpret_cast<u32x4*>(y + i) = o;
                    });
        } else {
            const int64_t i0 = (p - e.first) * (PIECE_BYTES / 4), i1 = min(e.n, i0 + PIECE_BYTES / 4);
            const float* x = static_cast<const float*>(e.in);
            float* y = static_cast<float*>(e.out);
            walk<4>(x, 4, i0, i1, [&](int64_t i) { y[i] = x[i] * c; },
                    [&](int64_t i) {
                        f32x4 r = *reinterpret_cast<const f32x4*>(x + i);
#pragma unroll
                        for (int j = 0; j < 4; ++j) r[j] *= c;
                        if (!same) store16(y + i, __builtin_bit_cast(u32x4, r));
                        else if constexpr (PAST) __builtin_nontemporal_store(r, reinterpret_cast<f32x4*>(y + i));
                        else *reinterpret_cast<f32x4*>(y + i) = r;
                    });
        }
    }
}

// workspace: the first pass's sums, then the table
size_t need(int64_t count) { return MAXWG * 8 + (size_t)count * sizeof(Entry) + 256; }

}  // namespace

namespace m2 {

size_t clip_grad_norm_workspace(const m2_clip_grad_norm_args& a) {
    if (a.count < 0 || a.count > (1 << 24)) {
        set_error(M2_ERR_INVALID, "clip_grad_norm: bad count %lld", (long long)a.count);
        return 0;
    }
    return need(a.count);
}

int launch_clip_grad_norm(const m2_clip_grad_norm_args& a, hipStream_t s) {
    const char* who = "clip_grad_norm";
    M2_REQUIRE(a.count >= 0 && a.count <= (1 << 24) && (a.tensors || a.count == 0) && a.norm, M2_ERR_INVALID,
               "%s: tensors and norm are required", who);
    M2_REQUIRE(a.workspace && a.workspace_bytes >= need(a.count), M2_ERR_WORKSPACE,
               "%s: workspace of %zu bytes needed, %zu given", who, need(a.count), a.workspace_bytes);
    M2_REQUIRE(!a.clip || (a.max_norm >= 0.f && a.eps >= 0.f), M2_ERR_INVALID, "%s: max_norm %g, eps %g", who,
               a.max_norm, a.eps);
    for (int64_t i = 0; i < a.count; ++i) {
        const m2_tensor_ref& r = a.tensors[i];
        M2_REQUIRE(r.dtype == M2_F32 || r.dtype == M2_BF16, M2_ERR_UNSUPPORTED, "%s: tensor %lld: dtype %lld",
                   who, (long long)i, (long long)r.dtype);
        const uintptr_t es = m2_dtype_size((int32_t)r.dtype);
        M2_REQUIRE(r.n >= 0 && r.n < (1ll << 44) &&
                       (r.n == 0 || (r.in && (uintptr_t)r.in % es == 0 &&
                                     (!a.clip || (r.out && (uintptr_t)r.out % es == 0)))),
                   M2_ERR_INVALID, "%s: tensor %lld: bad pointer or size", who, (long long)i);
    }
    PassArgs p{};
    p.part = static_cast<double*>(a.workspace);
    Entry* table = reinterpret_cast<Entry*>(static_cast<char*>(a.workspace) + MAXWG * 8);
    p.table = table; p.norm = a.norm; p.max_norm = a.max_norm; p.eps = a.eps;
    // tensors without elements are passed over
    Batch b;
    b.count = 0;
    auto send = [&]() {
        hipLaunchKernelGGL(k_table, dim3(1), dim3(256), 0, s, b, table + p.count);
        p.count += b.count;
        b.count = 0;
    };
    for (int64_t i = 0; i < a.count; ++i) {
        const m2_tensor_ref& r = a.tensors[i];
        if (r.n == 0) continue;
        const int64_t per = r.dtype == M2_BF16 ? PIECE_BYTES / 2 : PIECE_BYTES / 4;
        if (b.count == BATCH || (b.count && p.pieces - b.base > (int64_t)UINT32_MAX)) send();
        if (b.count == 0) b.base = p.pieces;
        const int k = b.count++;
        b.in[k] = r.in;
        b.out[k] = r.out;
        b.n[k] = r.dtype == M2_BF16 ? ~r.n : r.n;
        b.first[k] = (uint32_t)(p.pieces - b.base);
        p.pieces += (r.n + per - 1) / per;
    }
    if (b.count) send();
    p.parts = (int)(p.pieces < MAXWG ? p.pieces : MAXWG);
    if (p.parts) hipLaunchKernelGGL(k_sumsq, dim3(p.parts), dim3(NT), 0, s, p);
    // tensors and results that do not both fit the last-level cache: the results go past it, and
    // what the first pass read stays (515 MB: 352 to 317 us; 2.7 GB: 1586 to 1542)
    const bool past = p.pieces > (128 << 20) / PIECE_BYTES;
    if (a.clip && p.parts && past) hipLaunchKernelGGL(k_scale<true>, dim3(p.parts), dim3(NT), 0, s, p);
    else if (a.clip && p.parts) hipLaunchKernelGGL(k_scale<false>, dim3(p.parts), dim3(NT), 0, s, p);
    else hipLaunchKernelGGL(k_norm, dim3(1), dim3(NT), 0, s, p);
    return check_launch(who);
}

}  // namespace m2
