// Low-rank adapters of many requests beside the shared Dense layer, and their gradients.
//
//   forward    h[n][r] = sum_k x[n][k] A[i][r][k],   out[n][u] (+)= scale[i] sum_r h[n][r] B[i][r][u],   i = index[n]
//   backward   g[n][r] = scale[i] sum_u dz[n][u] B[i][r][u]
//              dA[i][r][k] = sum_{n: index[n] = i} g[n][r] x[n][k]
//              dB[i][r][u] = scale[i] sum_{n: index[n] = i} h[n][r] dz[n][u]
//              dx[n][k] = sum_r g[n][r] A[i][r][k]
//
// With A as [L][R][K] and B as [L][R][U] three kernels serve all of it: contract the long axis of a row against its adapter
// (x.A^T and dz.B^T), expand the rank (h.B and g.A), and contract the rows of one adapter (g^T.x and h^T.dz).  All sums are
// float32; bf16 operands are widened as they are read.
#include "common.h"

namespace {

typedef __bf16 bf16;

__device__ inline float widen(float v) { return v; }
__device__ inline float widen(bf16 v) { return (float)v; }

// one workgroup per row: h[n][r] = sum_k x[n][k] m[i][r][k]; no adapter: zero, index behind the bank: NaN
template <class TX, class TM>
__global__ __launch_bounds__(256) void contract_kernel(const TX *__restrict__ x, const TM *__restrict__ m,
                                                       const int *__restrict__ index, float *__restrict__ h, int K, int L, int R,
                                                       long long ldx, long long ldm, long long sm) {
    __shared__ float red[4];
    const int n = blockIdx.x, i = index[n], lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int r = 0; r < R; ++r) {
        float sum = 0.f;
        if (i >= 0 && i < L)
            for (int k = threadIdx.x; k < K; k += 256) sum += widen(x[n * ldx + k]) * widen(m[i * sm + r * ldm + k]);
        for (int d = 32; d > 0; d >>= 1) sum += __shfl_xor(sum, d, 64);
        if (lane == 0) red[wave] = sum;
        __syncthreads();
        if (threadIdx.x == 0) h[(long long)n * R + r] = i >= L ? __builtin_nanf("") : red[0] + red[1] + red[2] + red[3];
        __syncthreads();
    }
}

// one thread per output: out[n][u] (+)= scale[i] sum_r h[n][r] m[i][r][u]
template <class TM>
__global__ __launch_bounds__(256) void expand_kernel(const float *__restrict__ h, const TM *__restrict__ m,
                                                     const int *__restrict__ index, const float *__restrict__ scale,
                                                     float *__restrict__ out, int U, int L, int R, long long ldm, long long sm,
                                                     long long ldo, int accumulate) {
    const int n = blockIdx.x, i = index[n];
    for (int u = blockIdx.y * 256 + threadIdx.x; u < U; u += gridDim.y * 256) {
        float v = i >= L ? __builtin_nanf("") : 0.f;
        if (i >= 0 && i < L) {
            for (int r = 0; r < R; ++r) v += h[(long long)n * R + r] * widen(m[i * sm + r * ldm + u]);
            v *= scale[i];
        }
        float *o = out + n * ldo + u;
        if (!accumulate) *o = v;
        else if (i >= 0) *o += v;
    }
}

// one thread per gradient: out[i][r][k] = scale[i] sum_{n of adapter i} g[n][r] x[n][k]
template <class TX>
__global__ __launch_bounds__(256) void rows_kernel(const float *__restrict__ g, const TX *__restrict__ x,
                                                   const int *__restrict__ index, const float *__restrict__ scale,
                                                   float *__restrict__ out, int N, int K, int R, long long ldx, long long ldo,
                                                   long long so) {
    const int i = blockIdx.z, r = blockIdx.y, k = blockIdx.x * 256 + threadIdx.x;
    if (k >= K) return;
    float sum = 0.f;
    for (int n = 0; n < N; ++n)
        if (index[n] == i) sum += g[(long long)n * R + r] * widen(x[n * ldx + k]);
    out[i * so + r * ldo + k] = sum * scale[i];
}

constexpr int kMaxRank = 128, kMaxAdapters = 4096;

int check_sizes(const char *what, int N, int K, int U, int L, int R) {
    TY1_REQUIRE(N >= 0 && K > 0 && U > 0, "%s: bad dimensions N=%d K=%d U=%d", what, N, K, U);
    TY1_REQUIRE(L >= 1 && L <= kMaxAdapters, "%s: %d adapters, 1 to %d are supported", what, L, kMaxAdapters);
    TY1_REQUIRE(R >= 1 && R <= kMaxRank, "%s: rank %d, 1 to %d are supported", what, R, kMaxRank);
    return 0;
}

size_t workspace(int N, int R) { return (size_t)N * R * 8 + 256; }

// a tensor that is written: its rows must not overlap
bool apart(int64_t ld, int rows, int64_t stride, int slabs, int cols) {
    if (rows > 1 && ld < cols) return false;
    return slabs <= 1 || stride >= (rows > 1 ? ld * (rows - 1) : 0) + cols;
}

template <class T>
int forward(const char *what, const T *x, const T *a, const T *b, const int32_t *index, const float *scale, float *out, float *h,
            int N, int K, int U, int L, int R, int64_t ldx, int64_t lda, int64_t sa, int64_t ldb, int64_t sb, int64_t ldo,
            int accumulate, void *ws, size_t ws_bytes, ty1_stream_t stream) {
    if (check_sizes(what, N, K, U, L, R)) return 1;
    if (N == 0) return 0;
    TY1_REQUIRE(x && a && b && index && scale && out, "%s: null pointer", what);
    TY1_REQUIRE((((uintptr_t)index | (uintptr_t)scale | (uintptr_t)out | (uintptr_t)h) & 3) == 0 &&
                    (((uintptr_t)x | (uintptr_t)a | (uintptr_t)b) & (sizeof(T) - 1)) == 0, "%s: pointers not aligned to their type", what);
    TY1_REQUIRE(ldx >= 0 && lda >= 0 && sa >= 0 && ldb >= 0 && sb >= 0, "%s: negative strides", what);
    TY1_REQUIRE(apart(ldo, N, 0, 1, U), "%s: ldo=%lld makes the rows of out overlap", what, (long long)ldo);
    TY1_REQUIRE(ws && ((uintptr_t)ws & 15) == 0 && ws_bytes >= workspace(N, R), "%s: workspace null, not 16-byte aligned, or %zu bytes where %zu are needed", what,
                ws_bytes, workspace(N, R));
    hipStream_t s = (hipStream_t)stream;
    ty1::ProfScope prof("adapter_forward", s);
    float *hh = h ? h : (float *)ws;
    contract_kernel<<<dim3(N), dim3(256), 0, s>>>(x, a, index, hh, K, L, R, ldx, lda, sa);
    expand_kernel<<<dim3(N, U < 4096 ? (U + 255) / 256 : 16), dim3(256), 0, s>>>(hh, b, index, scale, out, U, L, R, ldb, sb, ldo, accumulate);
    return ty1::check_launch(what);
}

template <class T>
int backward(const char *what, const float *dz, const T *x, const T *a, const T *b, const int32_t *index, const float *scale,
             const float *h, float *da, float *db, float *dx, int N, int K, int U, int L, int R, int64_t lddz, int64_t ldx,
             int64_t lda, int64_t sa, int64_t ldb, int64_t sb, int64_t ldda, int64_t sda, int64_t lddb, int64_t sdb,
             int64_t lddx, void *ws, size_t ws_bytes, ty1_stream_t stream) {
    if (check_sizes(what, N, K, U, L, R)) return 1;
    TY1_REQUIRE(da && db && scale && (N == 0 || (dz && x && a && b && index)), "%s: null pointer", what);
    TY1_REQUIRE((((uintptr_t)index | (uintptr_t)scale | (uintptr_t)dz | (uintptr_t)h | (uintptr_t)da | (uintptr_t)db | (uintptr_t)dx) & 3) == 0 &&
                    (((uintptr_t)x | (uintptr_t)a | (uintptr_t)b) & (sizeof(T) - 1)) == 0, "%s: pointers not aligned to their type", what);
    TY1_REQUIRE(lddz >= 0 && ldx >= 0 && lda >= 0 && sa >= 0 && ldb >= 0 && sb >= 0, "%s: negative strides", what);
    TY1_REQUIRE(apart(ldda, R, sda, L, K) && apart(lddb, R, sdb, L, U) && (!dx || apart(lddx, N, 0, 1, K)), "%s: strides make the rows of a gradient overlap", what);
    TY1_REQUIRE(ws && ((uintptr_t)ws & 15) == 0 && ws_bytes >= workspace(N, R), "%s: workspace null, not 16-byte aligned, or %zu bytes where %zu are needed", what,
                ws_bytes, workspace(N, R));
    hipStream_t s = (hipStream_t)stream;
    ty1::ProfScope prof("adapter_backward", s);
    float *g = (float *)ws, *hh = g + (size_t)N * R;
    if (N > 0) {
        contract_kernel<<<dim3(N), dim3(256), 0, s>>>(dz, b, index, g, U, L, R, lddz, ldb, sb);
        if (!h) contract_kernel<<<dim3(N), dim3(256), 0, s>>>(x, a, index, hh, K, L, R, ldx, lda, sa);
        if (dx) expand_kernel<<<dim3(N, K < 4096 ? (K + 255) / 256 : 16), dim3(256), 0, s>>>(g, a, index, scale, dx, K, L, R, lda, sa, lddx, 0);
    }
    rows_kernel<<<dim3((K + 255) / 256, R, L), dim3(256), 0, s>>>(g, x, index, scale, da, N, K, R, ldx, ldda, sda);
    rows_kernel<<<dim3((U + 255) / 256, R, L), dim3(256), 0, s>>>(h ? h : hh, dz, index, scale, db, N, U, R, lddz, lddb, sdb);
    return ty1::check_launch(what);
}

}  // namespace

extern "C" int ty1_adapter_workspace_bytes(int N, int K, int U, int L, int R, int backward, size_t *bytes) {
    TY1_REQUIRE(bytes, "ty1_adapter_workspace_bytes: null result pointer");
    (void)backward;
    if (check_sizes("ty1_adapter_workspace_bytes", N, K, U, L, R)) return 1;
    *bytes = workspace(N, R);
    return 0;
}

extern "C" int ty1_adapter_forward_f32(const float *x, const float *a, const float *b, const int32_t *index, const float *scale,
                                       float *out, float *h, int N, int K, int U, int L, int R, int64_t ldx, int64_t lda,
                                       int64_t sa, int64_t ldb, int64_t sb, int64_t ldo, int accumulate, void *workspace,
                                       size_t workspace_bytes, ty1_stream_t stream) {
    return forward<float>("ty1_adapter_forward_f32", x, a, b, index, scale, out, h, N, K, U, L, R, ldx, lda, sa, ldb, sb, ldo,
                          accumulate, workspace, workspace_bytes, stream);
}

extern "C" int ty1_adapter_forward_bf16(const void *x, const void *a, const void *b, const int32_t *index, const float *scale,
                                        float *out, float *h, int N, int K, int U, int L, int R, int64_t ldx, int64_t lda,
                                        int64_t sa, int64_t ldb, int64_t sb, int64_t ldo, int accumulate, void *workspace,
                                        size_t workspace_bytes, ty1_stream_t stream) {
    return forward<bf16>("ty1_adapter_forward_bf16", (const bf16 *)x, (const bf16 *)a, (const bf16 *)b, index, scale, out, h, N, K,
                         U, L, R, ldx, lda, sa, ldb, sb, ldo, accumulate, workspace, workspace_bytes, stream);
}

extern "C" int ty1_adapter_backward_f32(const float *dz, const float *x, const float *a, const float *b, const int32_t *index,
                                        const float *scale, const float *h, float *da, float *db, float *dx, int N, int K, int U,
                                        int L, int R, int64_t lddz, int64_t ldx, int64_t lda, int64_t sa, int64_t ldb, int64_t sb,
                                        int64_t ldda, int64_t sda, int64_t lddb, int64_t sdb, int64_t lddx, void *workspace,
                                        size_t workspace_bytes, ty1_stream_t stream) {
    return backward<float>("ty1_adapter_backward_f32", dz, x, a, b, index, scale, h, da, db, dx, N, K, U, L, R, lddz, ldx, lda, sa,
                           ldb, sb, ldda, sda, lddb, sdb, lddx, workspace, workspace_bytes, stream);
}

extern "C" int ty1_adapter_backward_bf16(const float *dz, const void *x, const void *a, const void *b, const int32_t *index,
                                         const float *scale, const float *h, float *da, float *db, float *dx, int N, int K, int U,
                                         int L, int R, int64_t lddz, int64_t ldx, int64_t lda, int64_t sa, int64_t ldb, int64_t sb,
                                         int64_t ldda, int64_t sda, int64_t lddb, int64_t sdb, int64_t lddx, void *workspace,
                                         size_t workspace_bytes, ty1_stream_t stream) {
    return backward<bf16>("ty1_adapter_backward_bf16", dz, (const bf16 *)x, (const bf16 *)a, (const bf16 *)b, index, scale, h, da,
                          db, dx, N, K, U, L, R, lddz, ldx, lda, sa, ldb, sb, ldda, sda, lddb, sdb, lddx, workspace,
                          workspace_bytes, stream);
}
