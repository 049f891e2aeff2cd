// The global norm over many gradient tensors, clipping by it, and the Adam step that clips on the way.
//
//   norm = sqrt(sum over all tensors and values of g^2);  c = 1 if norm <= max_norm, max_norm / norm above it, NaN if not finite
//   clip: out = g c                       (tf.clip_by_global_norm, which Keras' optimizers call for global_clipnorm)
//   Adam: the step of train.hip on g c    (Keras semantics)
//
// Squares and sums are float64: the largest float32 squared is 1e77, so no finite gradient overflows and none underflows, and the
// order of the sum is fixed by the sizes alone.  c stays float64 up to the product with g: max_norm / norm can lie below
// float32's range.
//
// Bound by HBM: g is read once for the norm and once more by what applies it.  At 18.5 M values (the Dense gradient) clipping into
// other buffers takes 49 us (222 MB, 4.5 TB/s), the clipped Adam step 117 us (591 MB, 5.05 TB/s, what a large copy reaches); in
// the step g c never reaches memory.
//
// The tensors' addresses and lengths travel by value in the launch's arguments (no copy to the device, nothing to keep alive,
// safe to capture); a launch takes up to kTensors of them, longer lists take several.  Seen as one concatenation, the values
// are split evenly over the workgroups whatever the tensors' sizes are.
#include "common.h"
#include <algorithm>
#include <cmath>

namespace {

typedef __bf16 bf16;

constexpr int kTensors = 64;
constexpr int kThreads = 256, kBlocks = 1024;                                   // four workgroups to a CU; the same on every device: it is the order of the sum

struct Lists {
    void *a[kTensors], *b[kTensors], *c[kTensors], *d[kTensors];   // norm: g; clip: g, out; Adam: p, g, m, v
    long long start[kTensors + 1];                                 // values before tensor t in this launch
    unsigned long long half;                                       // bit t: tensor t holds bf16
    int n;
};

__device__ inline double block_sum(double v, double *lds) {
    for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d, 64);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    double sum = 0.0;
    for (int w = 0; w < (int)blockDim.x >> 6; ++w) sum += lds[w];
    return sum;
}

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4_m __attribute__((ext_vector_type(4), aligned(4)));         // as it lies in memory: views of a bucket start anywhere
typedef __bf16 bf16x4_m __attribute__((ext_vector_type(4), aligned(2)));

// calls f(t, lo, hi) for every tensor that has values in this workgroup's share of the concatenation
template <class F>
__device__ inline void my_share(const Lists &ls, const F &f) {
    const long long total = ls.start[ls.n], per = (total + gridDim.x * 16ll - 1) / (gridDim.x * 16ll) * 16;
    const long long lo = per * blockIdx.x, hi = lo + per < total ? lo + per : total;
    if (lo >= hi) return;
    int t = 0;
    for (int step = kTensors / 2; step > 0; step >>= 1)
        if (t + step < ls.n && ls.start[t + step] <= lo) t += step;
    for (; t < ls.n && ls.start[t] < hi; ++t) {
        const long long a = lo > ls.start[t] ? lo : ls.start[t], b = hi < ls.start[t + 1] ? hi : ls.start[t + 1];
        f(t, a - ls.start[t], b - ls.start[t]);
    }
}

// calls four(j) for groups of four values from lo on, UN of them a thread before the next (their loads in flight together), and
// one(j) for the last values
template <int UN, class Four, class One>
__device__ inline void by_fours(long long lo, long long hi, const Four &four, const One &one) {
    const int W = 4 * blockDim.x;
    const long long whole = lo + ((hi - lo) & ~3ll);
    long long j = lo + 4 * threadIdx.x;
    for (; j + (UN - 1) * W < whole; j += UN * W) {
        typename Four::Values v[UN];
#pragma unroll
        for (int u = 0; u < UN; ++u) v[u] = four.load(j + u * W);
#pragma unroll
        for (int u = 0; u < UN; ++u) four.use(j + u * W, v[u]);
    }
    for (; j < whole; j += W) four.use(j, four.load(j));
    if (whole + threadIdx.x < hi) one(whole + threadIdx.x);
}

__device__ inline f32x4 load4(const float *p) { return *(const f32x4_m *)p; }
__device__ inline f32x4 load4(const bf16 *p) {
    const bf16x4_m v = *(const bf16x4_m *)p;
    return f32x4{(float)v[0], (float)v[1], (float)v[2], (float)v[3]};
}
__device__ inline void store4(float *p, f32x4 v) { *(f32x4_m *)p = v; }
__device__ inline void store4(bf16 *p, f32x4 v) { *(bf16x4_m *)p = bf16x4_m{(bf16)v[0], (bf16)v[1], (bf16)v[2], (bf16)v[3]}; }
__device__ inline float scaled(float g, double c) { return (float)((double)g * c); }

template <class T>
struct Square {
    typedef f32x4 Values;
    const T *g;
    double *sum;
    __device__ Values load(long long j) const { return load4(g + j); }
    __device__ void use(long long, const Values &v) const {
#pragma unroll
        for (int e = 0; e < 4; ++e) *sum += (double)v[e] * (double)v[e];
    }
};

template <class T>
struct Scale {
    typedef f32x4 Values;
    const T *g;
    T *out;
    double c;
    __device__ Values load(long long j) const { return load4(g + j); }
    __device__ void use(long long j, Values v) const {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = scaled(v[e], c);
        store4(out + j, v);
    }
};

struct Adam {
    struct Values {
        f32x4 p, g, m, v;
    };
    float *p, *m, *v;
    const float *g;
    double c;
    float rate, b1, b2, c1, c2, eps;
    __device__ Values load(long long j) const { return {load4(p + j), load4(g + j), load4(m + j), load4(v + j)}; }
    __device__ void step(float &pj, float gj, float &mj, float &vj) const {
        gj = scaled(gj, c);
        mj = b1 * mj + c1 * gj;
        vj = b2 * vj + c2 * (gj * gj);
        pj -= rate * mj / (sqrtf(vj) + eps);
    }
    __device__ void use(long long j, Values x) const {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            float pe = x.p[e], me = x.m[e], ve = x.v[e];
            step(pe, x.g[e], me, ve);
            x.p[e] = pe;
            x.m[e] = me;
            x.v[e] = ve;
        }
        store4(p + j, x.p);
        store4(m + j, x.m);
        store4(v + j, x.v);
    }
};

template <class T>
__device__ inline void square_share(const T *g, long long lo, long long hi, double &sum) {
    by_fours<4>(lo, hi, Square<T>{g, &sum}, [&](long long j) { sum += (double)(float)g[j] * (double)(float)g[j]; });
}

template <class T>
__device__ inline void scale_share(const T *g, T *out, double c, long long lo, long long hi) {
    by_fours<4>(lo, hi, Scale<T>{g, out, c}, [&](long long j) { out[j] = (T)scaled((float)g[j], c); });
}

// the coefficient of a norm
__device__ inline double shrink(double norm, double max_norm) {
    if (!(norm < __builtin_huge_val())) return __builtin_nan("");
    return norm <= max_norm ? 1.0 : max_norm / norm;
}

__device__ inline void square_all(const Lists &ls, void *const *list, double &sum) {
    my_share(ls, [&](int t, long long lo, long long hi) {
        if (ls.half >> t & 1) square_share((const bf16 *)list[t], lo, hi, sum);
        else square_share((const float *)list[t], lo, hi, sum);
    });
}

__device__ inline void scale_all(const Lists &ls, double c) {
    my_share(ls, [&](int t, long long lo, long long hi) {
        if (c == 1.0 && ls.a[t] == ls.b[t]) return;                    // in place and within the norm: the values are the result
        if (ls.half >> t & 1) scale_share((const bf16 *)ls.a[t], (bf16 *)ls.b[t], c, lo, hi);
        else scale_share((const float *)ls.a[t], (float *)ls.b[t], c, lo, hi);
    });
}

struct AdamArgs {
    float rate, b1, b2, c1, c2, eps;
};

__device__ inline void adam_all(const Lists &ls, const AdamArgs &a, double c) {
    my_share(ls, [&](int t, long long lo, long long hi) {
        const Adam f = {(float *)ls.a[t], (float *)ls.c[t], (float *)ls.d[t], (const float *)ls.b[t], c, a.rate, a.b1, a.b2, a.c1, a.c2, a.eps};
        by_fours<1>(lo, hi, f, [&](long long j) { f.step(f.p[j], f.g[j], f.m[j], f.v[j]); });
    });
}

__global__ __launch_bounds__(kThreads) void norm_kernel(const Lists ls, double *__restrict__ part) {
    __shared__ double lds[16];
    double sum = 0.0;
    square_all(ls, ls.a, sum);
    sum = block_sum(sum, lds);
    if (threadIdx.x == 0) part[blockIdx.x] = sum;
}

// the norm and the coefficient from the partial sums, by every workgroup for itself; workgroup 0 also stores the norm
__device__ inline double coefficient(const double *__restrict__ part, int parts, double max_norm, float *norm, double *lds) {
    double sum = 0.0;
    for (int j = threadIdx.x; j < parts; j += blockDim.x) sum += part[j];
    const double n = sqrt(block_sum(sum, lds));
    if (blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)n;
    return shrink(n, max_norm);
}

__global__ __launch_bounds__(kThreads) void norm_finish_kernel(const double *__restrict__ part, int parts, float *norm) {
    __shared__ double lds[16];
    coefficient(part, parts, 1.0, norm, lds);
}

__global__ __launch_bounds__(kThreads) void clip_kernel(const Lists ls, const double *__restrict__ part, int parts, double max_norm,
                                                        float *norm) {
    __shared__ double lds[16];
    scale_all(ls, coefficient(part, parts, max_norm, norm, lds));
}

__global__ __launch_bounds__(kThreads) void adam_clip_kernel(const Lists ls, const double *__restrict__ part, int parts,
                                                             double max_norm, float *norm, const AdamArgs a) {
    __shared__ double lds[16];
    adam_all(ls, a, coefficient(part, parts, max_norm, norm, lds));
}

// Few values: one workgroup does all of it in one launch, the second reading of g from its cache.
enum Then { kNorm, kClip, kAdam };
template <Then THEN>
__global__ __launch_bounds__(1024) void small_kernel(const Lists ls, double max_norm, float *norm, const AdamArgs a) {
    __shared__ double lds[16];
    double sum = 0.0;
    square_all(ls, THEN == kAdam ? ls.b : ls.a, sum);
    const double n = sqrt(block_sum(sum, lds));                        // (behind its barriers every value has been read)
    if (threadIdx.x == 0) *norm = (float)n;
    if (THEN == kClip) scale_all(ls, shrink(n, max_norm));
    if (THEN == kAdam) adam_all(ls, a, shrink(n, max_norm));
}

int blocks_for(long long total) {
    const long long want = (total + 4095) / 4096;
    return (int)(want < 1 ? 1 : want > kBlocks ? kBlocks : want);
}

// No tensor that is written may share memory with another one (a value scaled twice, or read after it was scaled): all address
// ranges in order, each against the ranges that reach furthest before it.  Bit l of `written`: list l is written; list 1 may
// lie exactly on list 0 where `in_place`.  The norm (tensor number -1) is written too.
int check_overlap(const char *what, int n, const int64_t *counts, const int *dtypes, void *const *const *lists, int n_lists,
                  unsigned written, bool in_place, const float *norm) {
    struct Range {
        uintptr_t lo, hi;
        int t;
        bool w;
    };
    Range *r = (Range *)malloc(sizeof(Range) * ((size_t)n * n_lists + 1));
    TY1_REQUIRE(r, "%s: out of host memory", what);
    size_t k = 0;
    r[k++] = {(uintptr_t)norm, (uintptr_t)(norm + 1), -1, true};
    for (int l = 0; l < n_lists; ++l)
        for (int t = 0; t < n; ++t) {
            if (counts[t] == 0 || (in_place && l == 0 && lists[1][t] == lists[0][t])) continue;
            const uintptr_t lo = (uintptr_t)lists[l][t];
            r[k++] = {lo, lo + (uintptr_t)counts[t] * (dtypes && dtypes[t] == TY1_BF16 ? 2 : 4), t, (written >> l & 1) != 0};
        }
    std::sort(r, r + k, [](const Range &a, const Range &b) { return a.lo < b.lo; });
    uintptr_t read_to = 0, written_to = 0;
    bool bad = false;
    int at = 0;
    for (size_t j = 0; j < k && !bad; ++j) {
        bad = r[j].lo < written_to || (r[j].w && r[j].lo < read_to);
        at = r[j].t;
        uintptr_t &to = r[j].w ? written_to : read_to;
        if (r[j].hi > to) to = r[j].hi;
    }
    free(r);
    TY1_REQUIRE(!bad, "%s: tensor %d (-1: the norm) shares memory with another tensor of the call", what, at);
    return 0;
}

size_t partials(int n) { return ((size_t)n + kTensors - 1) / kTensors * kBlocks; }

// The norm and the scratch memory: alignments, and no partial sum may be written over a value that is still to be read.
int check_scratch(const char *what, int n, const int64_t *counts, const int *dtypes, void *const *const *lists, int n_lists,
                  const float *norm, const void *ws, size_t ws_bytes) {
    const size_t need = partials(n) * sizeof(double);
    TY1_REQUIRE(norm && ws && ws_bytes >= need, "%s: null pointer or workspace too small", what);
    TY1_REQUIRE(((uintptr_t)norm & 3) == 0 && ((uintptr_t)ws & 7) == 0, "%s: norm not aligned to 4 bytes or workspace not aligned to 8", what);
    const uintptr_t lo = (uintptr_t)ws, hi = lo + need, at = (uintptr_t)norm;
    TY1_REQUIRE(at + 4 <= lo || at >= hi, "%s: the workspace shares memory with the norm", what);
    for (int l = 0; l < n_lists; ++l)
        for (int t = 0; t < n; ++t) {
            const uintptr_t a = (uintptr_t)lists[l][t], b = a + (uintptr_t)counts[t] * (dtypes && dtypes[t] == TY1_BF16 ? 2 : 4);
            TY1_REQUIRE(counts[t] == 0 || b <= lo || a >= hi, "%s: the workspace shares memory with tensor %d", what, t);
        }
    return 0;
}

// lists of n host pointers: element sizes and addresses have to fit
int check_lists(const char *what, int n, const int64_t *counts, const int *dtypes, void *const *const *lists, int n_lists) {
    TY1_REQUIRE(n >= 1 && counts, "%s: no tensors", what);
    for (int l = 0; l < n_lists; ++l) TY1_REQUIRE(lists[l], "%s: null list", what);
    for (int t = 0; t < n; ++t) {
        TY1_REQUIRE(counts[t] >= 0, "%s: tensor %d has %lld values", what, t, (long long)counts[t]);
        TY1_REQUIRE(!dtypes || dtypes[t] == TY1_F32 || dtypes[t] == TY1_BF16, "%s: tensor %d has type %d", what, t, dtypes[t]);
        const uintptr_t align = dtypes && dtypes[t] == TY1_BF16 ? 2 : 4;
        for (int l = 0; l < n_lists; ++l)
            TY1_REQUIRE(counts[t] == 0 || (lists[l][t] && ((uintptr_t)lists[l][t] & (align - 1)) == 0), "%s: tensor %d: null or misaligned pointer", what, t);
    }
    return 0;
}

// fills ls with tensors t0, t0 + 1, ... -> how many list entries were consumed
int fill(Lists &ls, int t0, int n, const int64_t *counts, const int *dtypes, void *const *const *lists, int n_lists) {
    ls.n = 0;
    ls.half = 0;
    ls.start[0] = 0;
    int t = t0;
    for (; t < n && ls.n < kTensors; ++t) {
        if (counts[t] == 0) continue;
        void **dst[4] = {ls.a, ls.b, ls.c, ls.d};
        for (int l = 0; l < n_lists; ++l) dst[l][ls.n] = lists[l][t];
        if (dtypes && dtypes[t] == TY1_BF16) ls.half |= 1ull << ls.n;
        ls.start[ls.n + 1] = ls.start[ls.n] + counts[t];
        ++ls.n;
    }
    return t - t0;
}

// True with ls filled where one workgroup does it all.  One launch against two, in a graph: the norm 3.4 against 4.9 us and
// clipping 5.3 against 6.6 at 16384 values; the Adam step 6.8 against 7.8 at 8192 and 9.2 against 7.8 at 16384.
constexpr long long kSmall = 16384, kSmallAdam = 8192;
bool fill_small(Lists &ls, int n, const int64_t *counts, const int *dtypes, void *const *const *lists, int n_lists, long long limit) {
    return fill(ls, 0, n, counts, dtypes, lists, n_lists) == n && ls.start[ls.n] <= limit;
}

// the squares of one list, launch by launch -> number of partial sums in ws
int launch_norm(int n, const int64_t *counts, const int *dtypes, void *const *list, double *part, hipStream_t s) {
    int parts = 0;
    Lists ls;
    for (int t = 0; t < n;) {
        t += fill(ls, t, n, counts, dtypes, &list, 1);
        if (ls.n == 0) break;
        const int blocks = blocks_for(ls.start[ls.n]);
        norm_kernel<<<dim3(blocks), dim3(kThreads), 0, s>>>(ls, part + parts);
        parts += blocks;
    }
    return parts;
}

}  // namespace

extern "C" int ty1_grad_norm_workspace_bytes(int n, size_t *bytes) {
    TY1_REQUIRE(bytes && n >= 1, "ty1_grad_norm_workspace_bytes: bad arguments");
    *bytes = partials(n) * sizeof(double);
    return 0;
}

extern "C" int ty1_grad_norm(void *const *grads, const int64_t *counts, const int *dtypes, int n, float *norm, void *workspace,
                             size_t workspace_bytes, ty1_stream_t stream) {
    if (check_lists("ty1_grad_norm", n, counts, dtypes, &grads, 1)) return 1;
    if (check_scratch("ty1_grad_norm", n, counts, dtypes, &grads, 1, norm, workspace, workspace_bytes)) return 1;
    hipStream_t s = (hipStream_t)stream;
    ty1::ProfScope prof("grad_norm", s);
    Lists ls;
    if (fill_small(ls, n, counts, dtypes, &grads, 1, kSmall)) {
        small_kernel<kNorm><<<dim3(1), dim3(1024), 0, s>>>(ls, 1.0, norm, AdamArgs());
        return ty1::check_launch("ty1_grad_norm");
    }
    const int parts = launch_norm(n, counts, dtypes, grads, (double *)workspace, s);
    norm_finish_kernel<<<dim3(1), dim3(kThreads), 0, s>>>((const double *)workspace, parts, norm);
    return ty1::check_launch("ty1_grad_norm");
}

extern "C" int ty1_clip_grad_norm(void *const *grads, void *const *outs, const int64_t *counts, const int *dtypes, int n,
                                  double max_norm, float *norm, void *workspace, size_t workspace_bytes, ty1_stream_t stream) {
    void *const *lists[2] = {grads, outs};
    if (check_lists("ty1_clip_grad_norm", n, counts, dtypes, lists, 2)) return 1;
    TY1_REQUIRE(max_norm > 0.0, "ty1_clip_grad_norm: max_norm=%g must be positive", max_norm);
    if (check_scratch("ty1_clip_grad_norm", n, counts, dtypes, lists, 2, norm, workspace, workspace_bytes)) return 1;
    if (check_overlap("ty1_clip_grad_norm", n, counts, dtypes, lists, 2, 2u, true, norm)) return 1;
    hipStream_t s = (hipStream_t)stream;
    ty1::ProfScope prof("clip_grad_norm", s);
    Lists ls;
    if (fill_small(ls, n, counts, dtypes, lists, 2, kSmall)) {
        small_kernel<kClip><<<dim3(1), dim3(1024), 0, s>>>(ls, max_norm, norm, AdamArgs());
        return ty1::check_launch("ty1_clip_grad_norm");
    }
    const int parts = launch_norm(n, counts, dtypes, grads, (double *)workspace, s);
    int t = 0;
    do {
        t += fill(ls, t, n, counts, dtypes, lists, 2);
        clip_kernel<<<dim3(blocks_for(ls.start[ls.n])), dim3(kThreads), 0, s>>>(ls, (const double *)workspace, parts, max_norm, norm);
    } while (t < n);
    return ty1::check_launch("ty1_clip_grad_norm");
}

extern "C" int ty1_adam_step_clip_f32(void *const *p, void *const *g, void *const *m, void *const *v, const int64_t *counts, int n,
                                      double max_norm, double lr, double beta1, double beta2, double eps, int64_t t, float *norm,
                                      void *workspace, size_t workspace_bytes, ty1_stream_t stream) {
    void *const *lists[4] = {p, g, m, v};
    if (check_lists("ty1_adam_step_clip", n, counts, nullptr, lists, 4)) return 1;
    TY1_REQUIRE(max_norm > 0.0, "ty1_adam_step_clip: max_norm=%g must be positive", max_norm);
    TY1_REQUIRE(t >= 1, "ty1_adam_step_clip: bad t=%lld", (long long)t);
    TY1_REQUIRE(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0, "ty1_adam_step_clip: betas %g, %g must lie in [0, 1)", beta1, beta2);
    if (check_scratch("ty1_adam_step_clip", n, counts, nullptr, lists, 4, norm, workspace, workspace_bytes)) return 1;
    if (check_overlap("ty1_adam_step_clip", n, counts, nullptr, lists, 4, 13u, false, norm)) return 1;
    const double lr_t = lr * std::sqrt(1.0 - std::pow(beta2, (double)t)) / (1.0 - std::pow(beta1, (double)t));
    hipStream_t s = (hipStream_t)stream;
    ty1::ProfScope prof("adam_step_clip", s);
    const AdamArgs a = {(float)lr_t, (float)beta1, (float)beta2, (float)(1.0 - beta1), (float)(1.0 - beta2), (float)eps};
    Lists ls;
    if (fill_small(ls, n, counts, nullptr, lists, 4, kSmallAdam)) {
        small_kernel<kAdam><<<dim3(1), dim3(1024), 0, s>>>(ls, max_norm, norm, a);
        return ty1::check_launch("ty1_adam_step_clip_f32");
    }
    const int parts = launch_norm(n, counts, nullptr, g, (double *)workspace, s);
    int k = 0;
    do {
        k += fill(ls, k, n, counts, nullptr, lists, 4);
        adam_clip_kernel<<<dim3(blocks_for(ls.start[ls.n])), dim3(kThreads), 0, s>>>(ls, (const double *)workspace, parts, max_norm, norm, a);
    } while (k < n);
    return ty1::check_launch("ty1_adam_step_clip_f32");
}
