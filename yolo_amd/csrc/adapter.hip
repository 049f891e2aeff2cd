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
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
// the same, as they lie in memory: rows start at any element (units = 1470, sliced buffers), and one 16-byte load takes them
// from any address the element type allows
typedef float f32x4_m __attribute__((ext_vector_type(4), aligned(4)));
typedef __bf16 bf16x8_m __attribute__((ext_vector_type(8), aligned(2)));
typedef __bf16 bf16x4_m __attribute__((ext_vector_type(4), aligned(2)));

constexpr int kMaxRank = 128, kMaxAdapters = 4096;
constexpr int kSelfPlan = 256;            // rows up to which every workgroup finds its tile by itself (one thread per row)

// ---------------------------------------------------------------------------------------------------------------- tiles
// The rows of a batch come in any order of adapters; a tile is up to TM rows of ONE adapter, so that the adapter's weights are
// read once for all of them.  Rows without an adapter (index < 0 or >= L) form a class of their own, L, whose tiles are only
// filled in.  Up to kSelfPlan rows a workgroup works its tile out from the index (below 1 us, and no launch); above, one
// workgroup sorts the rows once (plan_kernel) and the others read the list.
struct Plan {
    const int *index;          // (N)
    int N, L;
    const int *perm;           // (N) rows, stably sorted by class        | null: N <= kSelfPlan
    const int *offs;           // (L + 1) first place of each class in perm
    const int4 *tiles;         // {class, first place, rows, -}
    const int *ntiles;
};

__device__ inline int class_of(int i, int L) { return i < 0 || i >= L ? L : i; }

struct alignas(16) TileLds {
    int cls[kSelfPlan];
    int rows[64];
    int wave_leaders[4];
    int adapter, first;
};

// tile t -> its class and number of rows (0: there is no tile t); lds.rows holds them.  All 256 threads call it.
template <int TM>
__device__ inline int find_tile(const Plan &p, int t, TileLds &lds, int &adapter) {
    const int tid = threadIdx.x;
    if (p.perm) {
        if (t >= *p.ntiles) return 0;
        const int4 tile = p.tiles[t];
        if (tid < tile.z) lds.rows[tid] = p.perm[tile.y + tid];
        adapter = tile.x;
        __syncthreads();
        return tile.z;
    }
    // a row leads a tile when the rows of its class before it are a multiple of TM; tile t belongs to the t-th leader
    const int cls = tid < p.N ? class_of(p.index[tid], p.L) : -1;
    lds.cls[tid] = cls;
    if (tid == 0) lds.adapter = -1;
    __syncthreads();
    int before = 0;
    for (int m = 0; m < p.N; m += 4) {
        const int4 c = *reinterpret_cast<const int4 *>(lds.cls + m);
        before += (c.x == cls && m < tid) + (c.y == cls && m + 1 < tid) + (c.z == cls && m + 2 < tid) + (c.w == cls && m + 3 < tid);
    }
    const bool leads = cls >= 0 && before % TM == 0;
    const unsigned long long vote = __ballot(leads);
    if ((tid & 63) == 0) lds.wave_leaders[tid >> 6] = __popcll(vote);
    __syncthreads();
    int place = __popcll(vote & ((1ull << (tid & 63)) - 1));
    for (int w = 0; w < tid >> 6; ++w) place += lds.wave_leaders[w];
    if (leads && place == t) {
        lds.adapter = cls;
        lds.first = before;
    }
    __syncthreads();
    adapter = lds.adapter;
    const int slot = before - lds.first;
    const bool mine = adapter >= 0 && cls == adapter && slot >= 0 && slot < TM;
    if (mine) lds.rows[slot] = tid;
    return __syncthreads_count(mine);
}

// One workgroup sorts the rows by class (a stable counting sort, so that an adapter's rows stay in ascending order) and cuts
// the classes into tiles.  Each wave owns a contiguous segment of the rows: counts them by class in LDS, the counts turn into
// first places (class by class, segment by segment), and each wave puts its rows down in order, equal classes within 64 rows
// ranked by ballots over the bits of the class.
__global__ __launch_bounds__(1024) void plan_kernel(const int *__restrict__ index, int N, int L, int waves, int bits, int TM,
                                                    int *__restrict__ perm, int *__restrict__ offs, int4 *__restrict__ tiles,
                                                    int *__restrict__ ntiles) {
    extern __shared__ int hist[];                     // [waves][L + 1]
    __shared__ long long scan[16];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, C = L + 1;
    const int per = ((N + waves - 1) / waves + 63) & ~63;
    const long long lo = (long long)wave * per, hi = lo + per < N ? lo + per : N;
    for (int c = tid; c < waves * C; c += 1024) hist[c] = 0;
    __syncthreads();
    if (wave < waves)
        for (long long n = lo + lane; n < hi; n += 64) atomicAdd(&hist[wave * C + class_of(index[n], L)], 1);
    __syncthreads();
    long long carry = 0;                              // rows in the low half, tiles in the high half
    for (int c0 = 0; c0 < C; c0 += 1024) {
        const int c = c0 + tid;
        int rows = 0;
        if (c < C)
            for (int w = 0; w < waves; ++w) rows += hist[w * C + c];
        long long v = (long long)((rows + TM - 1) / TM) << 32 | rows;
        const long long mine = v;
        for (int d = 1; d < 64; d <<= 1) {
            const long long o = __shfl_up(v, d, 64);
            if (lane >= d) v += o;
        }
        if (lane == 63) scan[wave] = v;
        __syncthreads();
        long long before = carry + v - mine, all = 0;
        for (int w = 0; w < 16; ++w) {
            if (w < wave) before += scan[w];
            all += scan[w];
        }
        carry += all;
        if (c < C) {
            int place = (int)(before & 0xffffffff);
            int t = (int)(before >> 32);
            offs[c] = place;
            for (int at = 0; at < rows; at += TM) tiles[t++] = make_int4(c, place + at, rows - at < TM ? rows - at : TM, 0);
            for (int w = 0; w < waves; ++w) {
                const int k = hist[w * C + c];
                hist[w * C + c] = place;
                place += k;
            }
        }
        __syncthreads();
    }
    if (tid == 0) *ntiles = (int)(carry >> 32);
    if (wave < waves) {
        volatile int *mine = hist + wave * C;
        for (long long n0 = lo; n0 < hi; n0 += 64) {
            const long long n = n0 + lane;
            const int cls = n < hi ? class_of(index[n], L) : -1;
            unsigned long long same = __ballot(n < hi);
            for (int b = 0; b < bits; ++b) {
                const unsigned long long set = __ballot(cls >> b & 1);
                same &= cls >> b & 1 ? set : ~set;
            }
            if (n < hi) {
                const int rank = __popcll(same & ((1ull << lane) - 1));
                const int place = mine[cls];
                if (rank == 0) mine[cls] = place + __popcll(same);
                perm[place + rank] = (int)n;
            }
        }
    }
}

// ------------------------------------------------------------------------------------------------------------- contract
// part[s][n][r] = sum over K slice s of x[n][k] m[i][r][k], for the rows of one tile against their adapter: a GEMM tile of
// TM rows x R ranks, K long.  Bound by reading x and m once (both stream from memory, nothing is read twice by a tile), so the
// operands go straight from memory into the registers of the matrix instruction: lane (j, q) of a 16-row fragment holds 16
// consecutive bytes of row j at q * 16 bytes - four float32 steps of v_mfma_f32_16x16x4_f32 with k in another order, the same
// on both sides, or one bf16 step of v_mfma_f32_16x16x32_bf16.  The four waves take a quarter of the slice each and join in
// LDS; the next fragments are in flight while the present ones multiply.
template <class TX, class TM>
struct Frag;
template <>
struct Frag<float, float> {
    typedef f32x4 VX;
    typedef f32x4 VM;
    static constexpr int E = 4;                        // elements of a lane
    static __device__ VX load(const float *p) { return *(const f32x4_m *)p; }
    static __device__ f32x4 mma(const VX &a, const VM &b, f32x4 c) {
#pragma unroll
        for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], c, 0, 0, 0);
        return c;
    }
};
template <>
struct Frag<bf16, bf16> {
    typedef bf16x8 VX;
    typedef bf16x8 VM;
    static constexpr int E = 8;
    static __device__ VX load(const bf16 *p) { return *(const bf16x8_m *)p; }
    static __device__ f32x4 mma(const VX &a, const VM &b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};
template <>
struct Frag<float, bf16> {                             // float32 gradients against bf16 weights: widened, exact
    typedef f32x4 VX;
    typedef bf16x4 VM;
    static constexpr int E = 4;
    static __device__ VX load(const float *p) { return *(const f32x4_m *)p; }
    static __device__ VM load(const bf16 *p) { return *(const bf16x4_m *)p; }
    static __device__ f32x4 mma(const VX &a, const VM &b, f32x4 c) {
#pragma unroll
        for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], (float)b[e], c, 0, 0, 0);
        return c;
    }
};
template <class V, class T>
__device__ inline V load_tail(const T *p, int n, int left) {       // what there is of n elements, zeros behind
    V v;
    for (int e = 0; e < n; ++e) v[e] = e < left ? p[e] : (T)0.f;
    return v;
}

template <class TX, class TM>
struct ContractArgs {
    const TX *x;               // (N,K) stride ldx
    const TM *m;               // (L,R,K) strides sm, ldm
    float *part;               // (slices, N, R)
    long long ldx, ldm, sm;
    int K, R, slices;
};

template <class TX, class TW, int NT, int RT>
__global__ __launch_bounds__(256) void contract_kernel(const ContractArgs<TX, TW> a, const Plan p) {
    typedef Frag<TX, TW> F;
    typedef typename F::VX VX;
    typedef typename F::VM VM;
    constexpr int TM = 16 * NT, R16 = 16 * RT, E = F::E, KC = 4 * E;
    constexpr int UN = 16 / (NT + RT) < 2 ? 2 : 16 / (NT + RT) > 8 ? 8 : 16 / (NT + RT);      // fragments in flight per operand row
    __shared__ TileLds tl;
    __shared__ float red[4][TM * R16];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), j = lane & 15, q = lane >> 4;
    const int t = blockIdx.x / a.slices, s = blockIdx.x - t * a.slices;
    int adapter;
    const int count = find_tile<TM>(p, t, tl, adapter);
    if (count == 0 || adapter >= p.L) return;

    const TX *xp[NT];
    const TW *mp[RT];
#pragma unroll
    for (int b = 0; b < NT; ++b) xp[b] = a.x + tl.rows[16 * b + j < count ? 16 * b + j : count - 1] * a.ldx + q * E;
#pragma unroll
    for (int b = 0; b < RT; ++b) mp[b] = a.m + adapter * a.sm + (16 * b + j < a.R ? 16 * b + j : a.R - 1) * a.ldm + q * E;
    f32x4 acc[NT][RT];
#pragma unroll
    for (int b = 0; b < NT; ++b)
#pragma unroll
        for (int c = 0; c < RT; ++c) acc[b][c] = f32x4{0.f, 0.f, 0.f, 0.f};

    // this wave's whole fragments [c0, c1) of KC elements; the wave with the last ones also takes what is left of K
    const int chunks = a.K / KC;
    const int share = 4 * s + wave, shares = 4 * a.slices;
    const int c0 = (int)((long long)chunks * share / shares), c1 = (int)((long long)chunks * (share + 1) / shares);
    VX xa[UN][NT], xb[UN][NT];
    VM ma[UN][RT], mb[UN][RT];
    auto load = [&](VX(&xv)[UN][NT], VM(&mv)[UN][RT], int c) {
        const long long k = (long long)c * KC;
#pragma unroll
        for (int u = 0; u < UN; ++u) {
#pragma unroll
            for (int b = 0; b < NT; ++b) xv[u][b] = F::load(xp[b] + k + u * KC);
#pragma unroll
            for (int b = 0; b < RT; ++b) mv[u][b] = F::load(mp[b] + k + u * KC);
        }
    };
    auto multiply = [&](const VX(&xv)[UN][NT], const VM(&mv)[UN][RT]) {
#pragma unroll
        for (int u = 0; u < UN; ++u)
#pragma unroll
            for (int b = 0; b < NT; ++b)
#pragma unroll
                for (int r = 0; r < RT; ++r) acc[b][r] = F::mma(xv[u][b], mv[u][r], acc[b][r]);
    };
    int c = c0;
    if (c + UN <= c1) {
        load(xa, ma, c);
        c += UN;
        for (;;) {
            if (c + UN > c1) {
                multiply(xa, ma);
                break;
            }
            load(xb, mb, c);
            c += UN;
            multiply(xa, ma);
            if (c + UN > c1) {
                multiply(xb, mb);
                break;
            }
            load(xa, ma, c);
            c += UN;
            multiply(xb, mb);
        }
    }
    for (; c < c1; ++c) {
        const long long k = (long long)c * KC;
        VX xv[NT];
        VM mv[RT];
#pragma unroll
        for (int b = 0; b < NT; ++b) xv[b] = F::load(xp[b] + k);
#pragma unroll
        for (int b = 0; b < RT; ++b) mv[b] = F::load(mp[b] + k);
#pragma unroll
        for (int b = 0; b < NT; ++b)
#pragma unroll
            for (int r = 0; r < RT; ++r) acc[b][r] = F::mma(xv[b], mv[r], acc[b][r]);
    }
    if (share == shares - 1 && chunks * KC < a.K) {     // zeros on both sides behind the end: nothing there takes part
        const int k = chunks * KC, left = a.K - k - q * E;
        VX xv[NT];
        VM mv[RT];
#pragma unroll
        for (int b = 0; b < NT; ++b) xv[b] = load_tail<VX>(xp[b] + k, E, left);
#pragma unroll
        for (int b = 0; b < RT; ++b) mv[b] = load_tail<VM>(mp[b] + k, E, left);
#pragma unroll
        for (int b = 0; b < NT; ++b)
#pragma unroll
            for (int r = 0; r < RT; ++r) acc[b][r] = F::mma(xv[b], mv[r], acc[b][r]);
    }
#pragma unroll
    for (int b = 0; b < NT; ++b)
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
            for (int v = 0; v < 4; ++v) red[wave][(16 * b + 4 * q + v) * R16 + 16 * r + j] = acc[b][r][v];
    __syncthreads();
    float *part = a.part + (long long)s * p.N * a.R;
    for (int e = tid; e < count * R16; e += 256) {
        const int row = e / R16, r = e % R16;
        if (r < a.R) part[(long long)tl.rows[row] * a.R + r] = red[0][e] + red[1][e] + red[2][e] + red[3][e];
    }
}

// --------------------------------------------------------------------------------------------------------------- expand
// out[n][u] (+)= sum_r h[n][r] m[i][r][u] with h = scale[i] sum_s part[s]: one wave per 64 columns, lane (j, q) holding four
// consecutive ones, so that loads of m and stores of out are 256 bytes a row.  Bound by reading m and writing out.  h is
// joined from the K slices on the way (and stored, without the scale, where the caller keeps it).  float32 matrix instruction
// for both types: bf16 weights are widened, h is not rounded.
__device__ inline f32x4 load4(const float *p) { return *(const f32x4_m *)p; }
__device__ inline f32x4 load4(const bf16 *p) {
    const bf16x4_m v = *(const bf16x4_m *)p;
    return f32x4{(float)v[0], (float)v[1], (float)v[2], (float)v[3]};
}
template <class T>
__device__ inline f32x4 load4(const T *p, int left) {
    if (left >= 4) return load4(p);
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    for (int e = 0; e < 4; ++e)
        if (e < left) v[e] = (float)p[e];
    return v;
}

// dst[row][r] (row stride ld) = f * sum_s part[s][rows[row]][r], zero for r in [R, R16); also stored to keep, without f
template <int R16, int LD>
__device__ inline void join(float *dst, float *lds, const float *__restrict__ part, int slices, long long slab, const int *rows, int count,
                            int batch, int R, float f, float *keep) {
    const int tid = threadIdx.x;
    if (batch * R16 <= 128 && slices > 4) {           // a small batch: several threads to a value, as many for every tile
        const int n = batch * R16, groups = 256 / n;
        const int e = tid % n, g = tid / n, row = e / R16, r = e % R16;
        float v = 0.f;
        if (g < groups && row < count && r < R)
            for (int s = g; s < slices; s += groups) v += part[s * slab + (long long)rows[row] * R + r];
        lds[tid] = v;
        __syncthreads();
        if (row < count && tid < n) {
            float sum = 0.f;
            for (int k = 0; k < groups; ++k) sum += lds[k * n + tid];
            dst[row * LD + r] = f * sum;
            if (keep && r < R) keep[(long long)rows[row] * R + r] = sum;
        }
    } else {
        for (int e = tid; e < count * R16; e += 256) {
            const int row = e / R16, r = e % R16;
            float v = 0.f;
            if (r < R)
                for (int s = 0; s < slices; ++s) v += part[s * slab + (long long)rows[row] * R + r];
            dst[row * LD + r] = f * v;
            if (keep && r < R) keep[(long long)rows[row] * R + r] = v;
        }
    }
    __syncthreads();
}

template <class T>
struct ExpandArgs {
    const float *part;         // (slices, N, R)
    const T *m;                // (L, R, U) strides sm, ldm
    const float *scale;        // (L)
    float *out, *keep;         // (N, U) stride ldo; (N, R) or null
    long long ldm, sm, ldo;
    int U, R, slices, blocks, accumulate;
};

template <class T, int NT, int RT>
__global__ __launch_bounds__(256) void expand_kernel(const ExpandArgs<T> a, const Plan p) {
    constexpr int TM = 16 * NT, R16 = 16 * RT, LD = R16 + 4, STEPS = R16 / 4;
    __shared__ TileLds tl;
    __shared__ __attribute__((aligned(16))) float h[TM * LD];
    __shared__ float sums[256];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), j = lane & 15, q = lane >> 4;
    const int t = blockIdx.x / a.blocks, block = blockIdx.x - t * a.blocks;
    int adapter;
    const int count = find_tile<TM>(p, t, tl, adapter);
    if (count == 0) return;
    float *keep = block == 0 ? a.keep : nullptr;
    const int u = block * 256 + wave * 64 + 4 * j, left = a.U - u;
    if (adapter >= p.L) {                              // no adapter: zeros (or out as it is); an index behind the bank: NaN
        for (int row = 0; row < count; ++row) {
            const int n = tl.rows[row];
            const bool bad = p.index[n] >= 0;
            const float v = bad ? __builtin_nanf("") : 0.f;
            const int c = block * 256 + tid;
            if (c < a.U && (bad || !a.accumulate)) a.out[n * a.ldo + c] = v;
            if (keep && tid < a.R) keep[(long long)n * a.R + tid] = v;
        }
        return;
    }
    f32x4 m[STEPS];                                    // step k of lane (j, q): rank q * STEPS + k, the same order as h's
    const T *mp = a.m + adapter * a.sm + u;
#pragma unroll
    for (int k = 0; k < STEPS; ++k) {
        const int r = q * STEPS + k;
        m[k] = r < a.R && left > 0 ? load4(mp + r * a.ldm, left) : f32x4{0.f, 0.f, 0.f, 0.f};
    }
    for (int e = tid; e < (TM - count) * LD; e += 256) h[count * LD + e] = 0.f;
    join<R16, LD>(h, sums, a.part, a.slices, (long long)p.N * a.R, tl.rows, count, p.N, a.R, a.scale[adapter], keep);
    if (block * 256 + wave * 64 >= a.U) return;
#pragma unroll
    for (int b = 0; b < NT; ++b) {
        if (16 * b >= count) break;
        f32x4 acc[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) acc[c] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < STEPS; k += 4) {
            const f32x4 hv = *(const f32x4 *)(h + (16 * b + j) * LD + q * STEPS + k);
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int c = 0; c < 4; ++c) acc[c] = __builtin_amdgcn_mfma_f32_16x16x4f32(hv[e], m[k + e][c], acc[c], 0, 0, 0);
        }
#pragma unroll
        for (int v = 0; v < 4; ++v) {
            const int row = 16 * b + 4 * q + v;
            if (row >= count || left <= 0) continue;
            float *o = a.out + tl.rows[row] * a.ldo + u;
            f32x4 val = {acc[0][v], acc[1][v], acc[2][v], acc[3][v]};
            if (left >= 4) {
                if (a.accumulate) val += load4(o);
                *(f32x4_m *)o = val;
            } else {
                for (int e = 0; e < left; ++e) o[e] = a.accumulate ? o[e] + val[e] : val[e];
            }
        }
    }
}

// ----------------------------------------------------------------------------------------------------------------- rows
// out[i][r][k] = f sum over the rows n of adapter i of g[n][r] x[n][k], g = sum_s part[s]: one wave per 64 columns, lane (j, q)
// holding four consecutive ones of row 4 step + q, so that loads of x and stores of out are 256 bytes a row.  Bound by reading
// x and writing out once.  Two such products (A's gradient and B's) share a launch.  SPLIT: the four waves share the columns
// and take a quarter of the rows each (few adapters: four times the workgroups).
template <class T>
struct RowsArgs {
    const float *part;         // (slices, N, R)
    const T *x;                // (N, K) stride ldx
    float *out;                // (L, R, K) strides so, ldo
    long long ldx, ldo, so;
    int K, slices, blocks;
};

struct RowsLds {
    int rows[64];
    int wave_rows[4];
};

template <class T, int RT, bool SPLIT>
__device__ inline void rows_tile(const RowsArgs<T> &a, const Plan &p, const float *scale, int R, int block, float *g, float *red, RowsLds &tl) {
    constexpr int R16 = 16 * RT, LD = RT == 1 ? 16 : R16 + 16;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), j = lane & 15, q = lane >> 4;
    const int i = block / a.blocks, cb = block - i * a.blocks;
    const int k0 = SPLIT ? cb * 64 : cb * 256 + wave * 64, k = k0 + 4 * j, left = a.K - k;
    f32x4 acc[RT][4];
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
        for (int c = 0; c < 4; ++c) acc[t][c] = f32x4{0.f, 0.f, 0.f, 0.f};
    int first = 0, total;
    bool mine = false;
    int place = 0;
    if (p.perm) {
        first = p.offs[i];
        total = p.offs[i + 1] - first;
    } else {
        mine = tid < p.N && p.index[tid] == i;
        const unsigned long long vote = __ballot(mine);
        if (lane == 0) tl.wave_rows[wave] = __popcll(vote);
        __syncthreads();
        place = __popcll(vote & ((1ull << lane) - 1));
        total = 0;
        for (int w = 0; w < 4; ++w) {
            if (w < wave) place += tl.wave_rows[w];
            total += tl.wave_rows[w];
        }
    }
    const float f = total ? scale[i] : 0.f;
    for (int r0 = 0; r0 < total; r0 += 64) {
        const int count = total - r0 < 64 ? total - r0 : 64, padded = (count + 15) & ~15;
        __syncthreads();
        if (p.perm) {
            if (tid < count) tl.rows[tid] = p.perm[first + r0 + tid];
        } else if (mine && place >= r0 && place < r0 + 64) {
            tl.rows[place - r0] = tid;
        }
        __syncthreads();
        for (int e = tid; e < (padded - count) * LD; e += 256) g[count * LD + e] = 0.f;
        join<R16, LD>(g, red, a.part, a.slices, (long long)p.N * R, tl.rows, count, p.N, R, f, nullptr);
        for (int s0 = SPLIT ? 16 * wave : 0; s0 < count; s0 += SPLIT ? 64 : 16) {
            f32x4 x[4];
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                const int row = s0 + 4 * s + q;
                x[s] = row < count && left > 0 ? load4(a.x + tl.rows[row] * a.ldx + k, left) : f32x4{0.f, 0.f, 0.f, 0.f};
            }
#pragma unroll
            for (int s = 0; s < 4; ++s)
#pragma unroll
                for (int t = 0; t < RT; ++t) {
                    const float gv = g[(s0 + 4 * s + q) * LD + 16 * t + j];
#pragma unroll
                    for (int c = 0; c < 4; ++c) acc[t][c] = __builtin_amdgcn_mfma_f32_16x16x4f32(gv, x[s][c], acc[t][c], 0, 0, 0);
                }
        }
    }
    float *out = a.out + i * a.so;
    if (SPLIT) {
#pragma unroll
        for (int t = 0; t < RT; ++t) {
            __syncthreads();
#pragma unroll
            for (int v = 0; v < 4; ++v) *(f32x4 *)(red + wave * 1024 + (4 * q + v) * 64 + 4 * j) = f32x4{acc[t][0][v], acc[t][1][v], acc[t][2][v], acc[t][3][v]};
            __syncthreads();
            const int r = 16 * t + (tid >> 4), c = cb * 64 + 4 * (tid & 15);
            const f32x4 *e = (const f32x4 *)red + tid;
            const f32x4 val = e[0] + e[256] + e[512] + e[768];
            if (r < R && c < a.K) {
                float *o = out + r * a.ldo + c;
                if (a.K - c >= 4) *(f32x4_m *)o = val;
                else
                    for (int y = 0; y < a.K - c; ++y) o[y] = val[y];
            }
        }
    } else {
#pragma unroll
        for (int t = 0; t < RT; ++t)
#pragma unroll
            for (int v = 0; v < 4; ++v) {
                const int r = 16 * t + 4 * q + v;
                if (r >= R || left <= 0) continue;
                float *o = out + r * a.ldo + k;
                const f32x4 val = {acc[t][0][v], acc[t][1][v], acc[t][2][v], acc[t][3][v]};
                if (left >= 4) *(f32x4_m *)o = val;
                else
                    for (int y = 0; y < left; ++y) o[y] = val[y];
            }
    }
}

template <class T, int RT, bool SPLIT>
__global__ __launch_bounds__(256) void rows_kernel(const RowsArgs<T> a, const RowsArgs<float> b, const Plan p, const float *__restrict__ scale,
                                                   int R, int a_blocks) {
    constexpr int R16 = 16 * RT, LD = RT == 1 ? 16 : R16 + 16;
    __shared__ RowsLds tl;
    __shared__ __attribute__((aligned(16))) float g[64 * LD];
    __shared__ __attribute__((aligned(16))) float red[SPLIT ? 4096 : 256];
    if ((int)blockIdx.x < a_blocks) rows_tile<T, RT, SPLIT>(a, p, scale, R, blockIdx.x, g, red, tl);
    else rows_tile<float, RT, SPLIT>(b, p, scale, R, blockIdx.x - a_blocks, g, red, tl);
}

// ------------------------------------------------------------------------------------------------------------- the host
int check_sizes(const char *what, int N, int K, int U, int L, int R) {
    TY1_REQUIRE(N >= 0 && K > 0 && U > 0, "%s: bad dimensions N=%d K=%d U=%d", what, N, K, U);
    TY1_REQUIRE(L >= 1 && L <= kMaxAdapters, "%s: %d adapters, 1 to %d are supported", what, L, kMaxAdapters);
    TY1_REQUIRE(R >= 1 && R <= kMaxRank, "%s: rank %d, 1 to %d are supported", what, R, kMaxRank);
    return 0;
}

// Everything that follows from the sizes alone: tile height, number of tiles at the most, and the scratch memory's layout.
struct Layout {
    int rt, nt;                // ranks and rows of a tile, in 16s
    int max_tiles;
    bool sorted;               // plan_kernel's list, not each workgroup's own
    size_t perm, offs, tiles, ntiles, part, part2, bytes;
    int slices, slices2;       // K slices of the first contraction and, backward only, of the one that computes h again
};

int slices_for(int tiles, int K) {
    // enough workgroups for every CU to hold four, but at least 512 elements of K for a workgroup (128 a wave: below that the
    // join of the slices costs more than their reading)
    const int want = (4 * 256 + tiles - 1) / tiles, most = (K + 511) / 512;
    const int s = want < most ? want : most;
    return s < 1 ? 1 : s > 64 ? 64 : s;
}

Layout layout(int N, int K, int U, int L, int R, bool back) {
    Layout y;
    y.rt = R <= 16 ? 1 : R <= 32 ? 2 : R <= 64 ? 4 : 8;
    const int classes = L < N ? L : N;
    y.nt = N >= 48ll * classes ? (y.rt == 8 ? 2 : 4) : 1;
    const long long tiles = (long long)N / (16 * y.nt) + (L + 1 < N ? L + 1 : N);
    y.max_tiles = (int)(tiles < N ? tiles : N > 1 ? N : 1);
    y.sorted = N > kSelfPlan;
    y.slices = back ? slices_for(y.max_tiles, U) : slices_for(y.max_tiles, K);
    y.slices2 = back ? slices_for(y.max_tiles, K) : 0;
    size_t at = 0;
    auto take = [&](size_t n) {
        const size_t here = at;
        at += (n + 255) & ~(size_t)255;
        return here;
    };
    y.perm = take(y.sorted ? 4 * (size_t)N : 0);
    y.offs = take(y.sorted ? 4 * ((size_t)L + 1) : 0);
    y.tiles = take(y.sorted ? 16 * (size_t)y.max_tiles : 0);
    y.ntiles = take(y.sorted ? 4 : 0);
    y.part = take(4 * (size_t)y.slices * N * R);
    y.part2 = take(4 * (size_t)y.slices2 * N * R);
    y.bytes = at < 256 ? 256 : at;
    return y;
}

Plan make_plan(const Layout &y, char *ws, const int32_t *index, int N, int L, hipStream_t s) {
    Plan p = {index, N, L, nullptr, nullptr, nullptr, nullptr};
    if (!y.sorted) return p;
    int waves = 15360 / (L + 1), bits = 1;             // 60 KB of counters
    waves = waves > 16 ? 16 : waves;
    while (1 << bits < L + 1) ++bits;
    int *perm = (int *)(ws + y.perm), *offs = (int *)(ws + y.offs), *ntiles = (int *)(ws + y.ntiles);
    int4 *tiles = (int4 *)(ws + y.tiles);
    plan_kernel<<<dim3(1), dim3(1024), (size_t)waves * (L + 1) * 4, s>>>(index, N, L, waves, bits, 16 * y.nt, perm, offs, tiles, ntiles);
    p.perm = perm;
    p.offs = offs;
    p.tiles = tiles;
    p.ntiles = ntiles;
    return p;
}

#define TY1_BY_TILE(y, CALL)                                                      \
    do {                                                                          \
        if (y.nt == 1) {                                                          \
            if (y.rt == 1) CALL(1, 1); else if (y.rt == 2) CALL(1, 2);            \
            else if (y.rt == 4) CALL(1, 4); else CALL(1, 8);                      \
        } else {                                                                  \
            if (y.rt == 1) CALL(4, 1); else if (y.rt == 2) CALL(4, 2);            \
            else if (y.rt == 4) CALL(4, 4); else CALL(2, 8);                      \
        }                                                                         \
    } while (0)

template <class TX, class TM>
void contract(const Layout &y, const Plan &p, const TX *x, long long ldx, const TM *m, long long ldm, long long sm, float *part, int K, int R,
              int slices, hipStream_t s) {
    const ContractArgs<TX, TM> a = {x, m, part, ldx, ldm, sm, K, R, slices};
    const dim3 grid((unsigned)(y.max_tiles * slices));
#define CALL(NT, RT) contract_kernel<TX, TM, NT, RT><<<grid, dim3(256), 0, s>>>(a, p)
    TY1_BY_TILE(y, CALL);
#undef CALL
}

template <class T>
void expand(const Layout &y, const Plan &p, const float *part, int slices, const T *m, long long ldm, long long sm, const float *scale, float *out,
            long long ldo, float *keep, int U, int R, int accumulate, hipStream_t s) {
    const int blocks = (U + 255) / 256;
    const ExpandArgs<T> a = {part, m, scale, out, keep, ldm, sm, ldo, U, R, slices, blocks, accumulate};
    const dim3 grid((unsigned)(y.max_tiles * blocks));
#define CALL(NT, RT) expand_kernel<T, NT, RT><<<grid, dim3(256), 0, s>>>(a, p)
    TY1_BY_TILE(y, CALL);
#undef CALL
}

// a tensor that is written: its rows must not overlap
bool apart(int64_t ld, int rows, int64_t stride, int slabs, int cols) {
    if (rows > 1 && ld < cols) return false;
    return slabs <= 1 || stride >= (rows > 1 ? ld * (rows - 1) : 0) + cols;
}

// workgroups of one launch: below 2^31, and below 2^32 threads
int check_grid(const char *what, const Layout &y, long long per_tile) {
    TY1_REQUIRE(y.max_tiles * per_tile < (1ll << 24), "%s: %d tiles of %lld workgroups are more than one launch holds", what, y.max_tiles, per_tile);
    return 0;
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
    const Layout y = layout(N, K, U, L, R, false);
    TY1_REQUIRE(ws && ((uintptr_t)ws & 15) == 0 && ws_bytes >= y.bytes, "%s: workspace null, not 16-byte aligned, or %zu bytes where %zu are needed", what,
                ws_bytes, y.bytes);
    if (check_grid(what, y, y.slices) || check_grid(what, y, (U + 255ll) / 256)) return 1;
    hipStream_t s = (hipStream_t)stream;
    ty1::ProfScope prof("adapter_forward", s, 2.0 * N * R * ((double)K + U), sizeof(T) * ((double)N * K + (double)(L < N ? L : N) * R * ((double)K + U)) + 4.0 * N * U);
    const Plan p = make_plan(y, (char *)ws, index, N, L, s);
    float *part = (float *)((char *)ws + y.part);
    contract(y, p, x, ldx, a, lda, sa, part, K, R, y.slices, s);
    expand<T>(y, p, part, y.slices, b, ldb, sb, scale, out, ldo, h, U, R, accumulate, s);
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
    const Layout y = layout(N, K, U, L, R, true);
    TY1_REQUIRE(ws && ((uintptr_t)ws & 15) == 0 && ws_bytes >= y.bytes, "%s: workspace null, not 16-byte aligned, or %zu bytes where %zu are needed", what,
                ws_bytes, y.bytes);
    // few adapters: 64 columns a workgroup and the rows split over its waves; enough of them: 256 columns, whole waves
    const bool split = (long long)L * ((K + 255) / 256 + (U + 255) / 256) < 1024;
    const long long ka = split ? (K + 63ll) / 64 : (K + 255ll) / 256, ub = split ? (U + 63ll) / 64 : (U + 255ll) / 256;
    TY1_REQUIRE(L * (ka + ub) < (1ll << 24), "%s: %d adapters of %d x %d are more than one launch holds", what, L, K, U);
    if (check_grid(what, y, y.slices) || check_grid(what, y, y.slices2) || (dx && check_grid(what, y, (K + 255ll) / 256))) return 1;
    hipStream_t s = (hipStream_t)stream;
    ty1::ProfScope prof("adapter_backward", s, 2.0 * N * R * (K * (dx ? 2.0 : 1.0) + 2.0 * U),
                        sizeof(T) * (double)N * K + 4.0 * N * U + 4.0 * L * R * ((double)K + U) + (dx ? 4.0 * N * K : 0.0));
    Plan p = {index, N, L, nullptr, nullptr, nullptr, nullptr};
    float *part = (float *)((char *)ws + y.part), *part2 = (float *)((char *)ws + y.part2);
    if (N > 0) {
        p = make_plan(y, (char *)ws, index, N, L, s);
        contract(y, p, dz, lddz, b, ldb, sb, part, U, R, y.slices, s);
        if (!h) contract(y, p, x, ldx, a, lda, sa, part2, K, R, y.slices2, s);
    }
    const RowsArgs<T> ra = {part, x, da, ldx, ldda, sda, K, y.slices, (int)ka};
    const RowsArgs<float> rb = {h ? h : part2, dz, db, lddz, lddb, sdb, U, h ? 1 : y.slices2, (int)ub};
    const dim3 grid((unsigned)(L * (ka + ub)));
#define CALL(RT)                                                                                                                    \
    do {                                                                                                                            \
        if (split) rows_kernel<T, RT, true><<<grid, dim3(256), 0, s>>>(ra, rb, p, scale, R, (int)(L * ka));                          \
        else rows_kernel<T, RT, false><<<grid, dim3(256), 0, s>>>(ra, rb, p, scale, R, (int)(L * ka));                               \
    } while (0)
    if (y.rt == 1) CALL(1); else if (y.rt == 2) CALL(2); else if (y.rt == 4) CALL(4); else CALL(8);
#undef CALL
    if (dx && N > 0) expand<T>(y, p, part, y.slices, a, lda, sa, scale, dx, lddx, nullptr, K, R, 0, s);
    return ty1::check_launch(what);
}

}  // namespace

extern "C" int ty1_adapter_workspace_bytes(int N, int K, int U, int L, int R, int backward, size_t *bytes) {
    TY1_REQUIRE(bytes, "ty1_adapter_workspace_bytes: null result pointer");
    if (check_sizes("ty1_adapter_workspace_bytes", N, K, U, L, R)) return 1;
    *bytes = layout(N, K, U, L, R, backward != 0).bytes;
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
