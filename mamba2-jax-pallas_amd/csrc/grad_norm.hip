// clip_grad_norm: the 2-norm over all values of many tensors, and the tensors
// times min(1, max_norm / (norm + eps)).
//
// Bound by HBM: every tensor is read for the norm and read again and written for the
// result (the scale is not known before the last value is).  The tensors
// travel as a table in the kernel's arguments, up to 96 per launch; a
// launch's workgroups share its elements evenly whatever the tensors' sizes
// (pieces of 16384 elements, a contiguous range of pieces per workgroup), so one large
// embedding and a hundred small vectors take one pass.  The squares
// are summed in float64 per thread (the vector units do that well
// above the rate at which HBM brings the values in): no square overflows and long
// sums lose nothing, and the order is fixed, so equal inputs give equal
// bits.  The second pass walks the pieces in the opposite order: what the first pass read
// last is still in the 256 MB last-level cache.
#include "m2_internal.h"

namespace {

constexpr int NT = 256;               // threads of a workgroup
constexpr int MAXT = 96;              // tensors per launch (the table stays below 4 KB)
constexpr int PIECE = 16384;          // elements
constexpr int MAXWG = 2048;           // workgroups per launch

struct Table {
    const void* in[MAXT];
    void* out[MAXT];
    int64_t n[MAXT];
    int first[MAXT + 1];              // first piece of each tensor
    uint8_t bf[MAXT];
    int count;
};

struct PassArgs {
    double* part;                     // this launch's partial sums
    const float* norm;                // [norm, scale] (second pass)
};

M2_DEV double block_sum(double v, double* red) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    double s = 0;
    for (int j = 0; j < (int)(blockDim.x >> 6); ++j) s += red[j];
    __syncthreads();
    return s;
}

// The tensor that piece p belongs to
M2_DEV int find(const Table& tb, int p) {
    int lo = 0, hi = tb.count - 1;
    while (lo < hi) {
        const int m = (lo + hi + 1) >> 1;
        if (tb.first[m] <= p) lo = m; else hi = m - 1;
    }
    return lo;
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

__global__ void __launch_bounds__(NT) k_sumsq(Table tb, PassArgs a) {
    __shared__ double red[NT / 64];
    const int np = tb.first[tb.count];
    const int per = (np + gridDim.x - 1) / gridDim.x;
    const int p0 = blockIdx.x * per, p1 = min(np, p0 + per);
    double s = 0;
    int ti = p0 < p1 ? find(tb, p0) : 0;
    for (int p = p0; p < p1; ++p) {
        while (p >= tb.first[ti + 1]) ++ti;
        const int64_t i0 = (int64_t)(p - tb.first[ti]) * PIECE;
        const int64_t i1 = min(tb.n[ti], i0 + PIECE);
        if (tb.bf[ti]) {
            const bf16* x = static_cast<const bf16*>(tb.in[ti]);
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
            const float* x = static_cast<const float*>(tb.in[ti]);
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

// norm and the factor, in `out` (caller) and `ws` = [norm, factor]
__global__ void __launch_bounds__(1024) k_norm(const double* part, int n, float max_norm, float eps,
                                               float* out, float* ws) {
    __shared__ double red[16];
    double s = 0;
    for (int i = threadIdx.x; i < n; i += 1024) s += part[i];
    s = block_sum(s, red);
    if (threadIdx.x == 0) {
        const float norm = (float)sqrt(s);
        const float c = max_norm / (norm + eps);
        *out = norm;
        ws[0] = norm;
        ws[1] = c >= 1.f ? 1.f : c;          // a norm that is not a number stays one here
    }
}

__global__ void __launch_bounds__(NT) k_scale(Table tb, PassArgs a) {
    const float c = a.norm[1];
    const int np = tb.first[tb.count];
    const int per = (np + gridDim.x - 1) / gridDim.x;
    // the opposite order of k_sumsq
    const int b = gridDim.x - 1 - blockIdx.x;
    const int p0 = b * per, p1 = min(np, p0 + per);
    int ti = p0 < p1 ? find(tb, p1 - 1) : 0;
    for (int p = p1 - 1; p >= p0; --p) {
        while (p < tb.first[ti]) --ti;
        if (c == 1.f && tb.in[ti] == tb.out[ti]) continue;      // in place, nothing to do
        const int64_t i0 = (int64_t)(p - tb.first[ti]) * PIECE;
        const int64_t i1 = min(tb.n[ti], i0 + PIECE);
        // input and output on the same 16-byte phase: whole pieces of both
        const bool same = (((uintptr_t)tb.in[ti] ^ (uintptr_t)tb.out[ti]) & 15) == 0;
        if (tb.bf[ti]) {
            const bf16* x = static_cast<const bf16*>(tb.in[ti]);
            bf16* y = static_cast<bf16*>(tb.out[ti]);
            walk<8>(x, 2, i0, i1, [&](int64_t i) { y[i] = (bf16)((float)x[i] * c); },
                    [&](int64_t i) {
                        const u32x4 r = *reinterpret_cast<const u32x4*>(x + i);
                        u32x4 o;
#pragma unroll
                        for (int j = 0; j < 4; ++j) o[j] = pk_bf16(bf16_lo(r[j]) * c, bf16_hi(r[j]) * c);
                        if (same) {
                            *reinterpret_cast<u32x4*>(y + i) = o;
                        } else {
                            const uint16_t* q = reinterpret_cast<const uint16_t*>(&o);
#pragma unroll
                            for (int j = 0; j < 8; ++j) reinterpret_cast<uint16_t*>(y)[i + j] = q[j];
                        }
                    });
        } else {
            const float* x = static_cast<const float*>(tb.in[ti]);
            float* y = static_cast<float*>(tb.out[ti]);
            walk<4>(x, 4, i0, i1, [&](int64_t i) { y[i] = x[i] * c; },
                    [&](int64_t i) {
                        f32x4 r = *reinterpret_cast<const f32x4*>(x + i);
#pragma unroll
                        for (int j = 0; j < 4; ++j) r[j] *= c;
                        if (same) {
                            *reinterpret_cast<f32x4*>(y + i) = r;
                        } else {
#pragma unroll
                            for (int j = 0; j < 4; ++j) y[i + j] = r[j];
                        }
                    });
        }
    }
}

// workspace: [norm, factor] in 256 bytes, then the partial sums of each launch
size_t need(int64_t count) { return 256 + (size_t)((count + MAXT - 1) / MAXT + 1) * MAXWG * 8; }

}  // namespace

namespace m2 {

size_t clip_grad_norm_workspace(const m2_clip_grad_norm_args& a) {
    if (a.count < 0 || a.count > (1 << 24)) {
        set_error(M2_ERR_INVALID, "clip_grad_norm: bad count %lld", (long long)a.count);
        return 0;
    }
    return need(a.count);
}

// fills the table from tensor i on (tensors without elements are passed over);
// returns the number of pieces
static int64_t fill(const m2_clip_grad_norm_args& a, int64_t& i, Table& tb) {
    tb.count = 0;
    int64_t np = 0;
    for (; i < a.count && tb.count < MAXT; ++i) {
        const m2_tensor_ref& r = a.tensors[i];
        if (r.n == 0) continue;
        const int64_t k = (r.n + PIECE - 1) / PIECE;
        if (np + k >= (1ll << 31) - 1) break;
        tb.in[tb.count] = r.in;
        tb.out[tb.count] = r.out;
        tb.n[tb.count] = r.n;
        tb.bf[tb.count] = r.dtype == M2_BF16;
        tb.first[tb.count++] = (int)np;
        np += k;
    }
    tb.first[tb.count] = (int)np;
    return np;
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
    float* nw = static_cast<float*>(a.workspace);
    double* part = reinterpret_cast<double*>(static_cast<char*>(a.workspace) + 256);
    Table tb;
    int64_t parts = 0;
    for (int64_t i = 0; i < a.count;) {
        const int64_t np = fill(a, i, tb);
        if (np == 0) break;
        const unsigned grid = (unsigned)(np < MAXWG ? np : MAXWG);
        hipLaunchKernelGGL(k_sumsq, dim3(grid), dim3(NT), 0, s, tb, PassArgs{part + parts, nullptr});
        parts += grid;
    }
    hipLaunchKernelGGL(k_norm, dim3(1), dim3(1024), 0, s, part, (int)parts, a.max_norm, a.eps, a.norm, nw);
    if (a.clip) {
        for (int64_t i = 0; i < a.count;) {
            const int64_t np = fill(a, i, tb);
            if (np == 0) break;
            const unsigned grid = (unsigned)(np < MAXWG ? np : MAXWG);
            hipLaunchKernelGGL(k_scale, dim3(grid), dim3(NT), 0, s, tb, PassArgs{nullptr, nw});
        }
    }
    return check_launch(who);
}

}  // namespace m2
