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
// float32 on the matrix cores and nothing between x and out is rounded to less: bf16 operands multiply as they are (their products
// are exact in float32) or are widened against float32 ones.  No atomics: every order of summation follows from the sizes and from
// which rows an adapter has, and a row's own results (out, h, dx) do not depend on the rows beside it in a batch of that size.
#include "common.h"
#include <type_traits>

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
constexpr int kSelfPlan = 256;            // rows up to which every workgroup finds its tile by itself
constexpr int kPiece = 256;               // rows of an adapter that one workgroup sums for its gradient in a long batch

// ---------------------------------------------------------------------------------------------------------------- tiles
// The rows of a batch come in any order of adapters; a tile is up to TM rows of ONE adapter, so that the adapter's weights are
// read once for all of them.  Rows without an adapter (index < 0 or >= L) form a class of their own, L, whose tiles are only
// filled in.  Up to kSelfPlan rows every workgroup works its tile out from the index itself; above, one workgroup sorts the
// rows once (plan_kernel, 5 to 10 us and a launch) and the others read the list.
struct Plan {
    const int *index;          // (N)
    int N, L;
    const int *perm;           // (N) rows, stably sorted by class        | null: N <= kSelfPlan
    const int *offs;           // (L + 1) first place of each class in perm
    const int4 *tiles;         // {class, first place, rows, -}, the unused ones without rows
    const int4 *pieces;        // backward of long batches: {adapter or -1, first place, up to kPiece rows, slot or -1}  | null
};

__device__ inline int class_of(int i, int L) { return i < 0 || i >= L ? L : i; }

struct TileLds {
    int rows[64];
};

// Up to 64 W rows, W to a lane: every wave finds the tile for itself by ballots over the bits of the class, without a barrier
// (a version that compares rows through LDS took 2 to 3 us more).  A row leads a tile when the rows of its class before it are
// a multiple of TM; tile t belongs to the t-th leader.
template <int W>
__device__ inline int tile_by_ballots(const Plan &p, int t, int TM, TileLds &lds, int &adapter) {
    const int lane = threadIdx.x & 63;
    int cls[W], before[W];
    unsigned long long same[W][W];                     // lanes of word v with the class of this lane's row in word w >= v
#pragma unroll
    for (int w = 0; w < W; ++w) {
        const int n = 64 * w + lane;
        cls[w] = n < p.N ? class_of(p.index[n], p.L) : p.L + 1;
#pragma unroll
        for (int v = 0; v <= w; ++v) same[w][v] = ~0ull;
    }
    for (int b = 0; (p.L + 1) >> b; ++b) {
        unsigned long long set[W];
#pragma unroll
        for (int w = 0; w < W; ++w) set[w] = __ballot(cls[w] >> b & 1);
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const unsigned long long all = -(unsigned long long)(cls[w] >> b & 1);
#pragma unroll
            for (int v = 0; v <= w; ++v) same[w][v] &= ~(set[v] ^ all);
        }
    }
    const unsigned long long below = (1ull << lane) - 1;
    int passed = 0, first = 0;
    adapter = -1;
#pragma unroll
    for (int w = 0; w < W; ++w) {
        before[w] = __popcll(same[w][w] & below);
#pragma unroll
        for (int v = 0; v < w; ++v) before[w] += __popcll(same[w][v]);
        const bool leads = 64 * w + lane < p.N && (before[w] & (TM - 1)) == 0;
        const unsigned long long leaders = __ballot(leads);
        const unsigned long long mine = __ballot(leads && passed + __popcll(leaders & below) == t);
        if (mine) {
            const int lead = __builtin_ctzll(mine);
            adapter = __builtin_amdgcn_readlane(cls[w], lead);
            first = __builtin_amdgcn_readlane(before[w], lead);
        }
        passed += __popcll(leaders);
    }
    if (adapter < 0) return 0;
    int count = 0;
#pragma unroll
    for (int w = 0; w < W; ++w) {
        const int slot = before[w] - first;
        const bool in = cls[w] == adapter && slot >= 0 && slot < TM;
        if (in) lds.rows[slot] = 64 * w + lane;        // all waves write the same: each reads what it wrote itself
        count += __popcll(__ballot(in));
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    return count;
}

// tile t of up to TM rows -> its class and number of rows (0: there is no tile t); lds.rows holds them.  All 256 threads call it.
__device__ inline int find_tile(const Plan &p, int t, int TM, TileLds &lds, int &adapter) {
    const int tid = threadIdx.x;
    if (p.perm) {
        const int4 tile = p.tiles[t];                  // (no rows: behind the last tile)
        if (tid < tile.z) lds.rows[tid] = p.perm[tile.y + tid];
        adapter = tile.x;
        __syncthreads();
        return tile.z;
    }
    if (p.N <= 64) return tile_by_ballots<1>(p, t, TM, lds, adapter);
    if (p.N <= 128) return tile_by_ballots<2>(p, t, TM, lds, adapter);
    return tile_by_ballots<4>(p, t, TM, lds, adapter);
}

// One workgroup sorts the rows by class (a stable counting sort, so that an adapter's rows stay in ascending order) and cuts
// the classes into tiles and, where pieces are asked for, the adapters into pieces of up to kPiece rows: an adapter with more than
// one piece gets a slot for each (what its pieces sum waits there to be joined).  Each wave owns a contiguous segment of the rows: counts them by class in LDS, the counts turn into
// first places (class by class, segment by segment), and each wave puts its rows down in order, equal classes within 64 rows
// ranked by ballots over the bits of the class.
template <bool PIECES>
__global__ __launch_bounds__(1024) void plan_kernel(const int *__restrict__ index, int N, int L, int waves, int bits, int TM,
                                                    int *__restrict__ perm, int *__restrict__ offs, int4 *__restrict__ tiles,
                                                    int max_tiles, int4 *__restrict__ pieces, int max_pieces, int2 *__restrict__ slots,
                                                    int max_slots) {
    extern __shared__ int hist[];                     // [waves][L + 1]
    __shared__ long long scan[16];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, C = L + 1;
    const int per = ((N + waves - 1) / waves + 63) & ~63;
    const long long lo = (long long)wave * per, hi = lo + per < N ? lo + per : N;
    constexpr int KEEP = 8;                           // the first rows' classes stay in registers between the two passes
    int kept[KEEP];
#pragma unroll
    for (int k = 0; k < KEEP; ++k) {
        const long long n = lo + 64 * k + lane;
        kept[k] = wave < waves && n < hi ? class_of(index[n], L) : -1;
    }
    for (int c = tid; c < waves * C; c += 1024) hist[c] = 0;
    __syncthreads();
    if (wave < waves) {
#pragma unroll
        for (int k = 0; k < KEEP; ++k)
            if (kept[k] >= 0) atomicAdd(&hist[wave * C + kept[k]], 1);
        for (long long n = lo + 64 * KEEP + lane; n < hi; n += 64) atomicAdd(&hist[wave * C + class_of(index[n], L)], 1);
    }
    __syncthreads();
    // what comes before this thread's two counts (low and high half), over all threads and the classes before them
    auto before_me = [&](long long v, long long &carry) {
        const long long mine = v;
        for (int d = 1; d < 64; d <<= 1) {
            const long long o = __shfl_up(v, d, 64);
            if (lane >= d) v += o;
        }
        __syncthreads();
        if (lane == 63) scan[wave] = v;
        __syncthreads();
        long long before = carry + v - mine;
#pragma unroll 4
        for (int w = 0; w < 16; ++w) {
            if (w < wave) before += scan[w];
            carry += scan[w];
        }
        return before;
    };
    long long carry = 0, carry2 = 0;                  // tiles and rows; slots and pieces
    for (int c0 = 0; c0 < C; c0 += 1024) {
        const int c = c0 + tid;
        int rows = 0;
        if (c < C)
            for (int w = 0; w < waves; ++w) rows += hist[w * C + c];
        const long long before = before_me((long long)((rows + TM - 1) / TM) << 32 | rows, carry);
        const int first = (int)(before & 0xffffffff);
        if (PIECES) {
            const int n = c >= L ? 0 : rows > kPiece ? (rows + kPiece - 1) / kPiece : 1, kept_apart = n > 1 ? n : 0;
            const long long b2 = before_me((long long)kept_apart << 32 | n, carry2);
            const int at = (int)(b2 & 0xffffffff), slot = (int)(b2 >> 32);
#pragma unroll 1
            for (int i = 0; i < n; ++i) pieces[at + i] = make_int4(c, first + i * kPiece, rows - i * kPiece < kPiece ? rows - i * kPiece : kPiece, n > 1 ? slot + i : -1);
#pragma unroll 1
            for (int i = 0; i < kept_apart; ++i) slots[slot + i] = make_int2(c, i == 0 ? n : 0);
        }
        if (c < C) {
            int place = first, t = (int)(before >> 32);
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
    if (PIECES) {
        for (int t = (int)(carry2 & 0xffffffff) + tid; t < max_pieces; t += 1024) pieces[t] = make_int4(-1, 0, 0, -1);
        for (int t = (int)(carry2 >> 32) + tid; t < max_slots; t += 1024) slots[t] = make_int2(0, 0);
    }
    for (int t = (int)(carry >> 32) + tid; t < max_tiles; t += 1024) tiles[t] = make_int4(0, 0, 0, 0);
    if (wave < waves) {
        volatile int *mine = hist + wave * C;
        auto put = [&](int cls, long long n) {
            unsigned long long same = __ballot(cls >= 0);
#pragma unroll 1
            for (int b = 0; b < bits; ++b) {
                const unsigned long long set = __ballot(cls >> b & 1);
                same &= cls >> b & 1 ? set : ~set;
            }
            if (cls >= 0) {
                const int rank = __popcll(same & ((1ull << lane) - 1));
                const int place = mine[cls];
                if (rank == 0) mine[cls] = place + __popcll(same);
                perm[place + rank] = (int)n;
            }
        };
#pragma unroll
        for (int k = 0; k < KEEP; ++k)
            if (lo + 64 * k < hi) put(kept[k], lo + 64 * k + lane);
        for (long long n0 = lo + 64 * KEEP; n0 < hi; n0 += 64) {
            const long long n = n0 + lane;
            put(n < hi ? class_of(index[n], L) : -1, n);
        }
    }
}

// ------------------------------------------------------------------------------------------------------------- contract
// part[s][n][r] = sum over K slice s of x[n][k] m[i][r][k], for the rows of one tile against their adapter: a GEMM tile of
// TM rows x R ranks, K long.  Bound by reading x and m once.  Every wave takes a quarter of the slice, the four sums join in LDS.
// Two forms:
//   direct   Fragments come from memory straight into the registers of the matrix instruction: lane (j, q) of a 16-row fragment
//            holds 16 consecutive bytes of row j at q * 16 bytes - four steps of v_mfma_f32_16x16x4_f32 with k in another
//            order, the same on both sides, or one of v_mfma_f32_16x16x32_bf16.  No barrier before the end: the shortest way
//            for one slice (one row x 12544 of rank 8: 4.5 us, most of it launch and three dependent loads; 64 rows of 16
//            adapters of rank 16, 16 MB: 7.1 to 8.2 us).
//   staged   A fragment load is 64 cache accesses an instruction (its neighbouring lanes are different rows), which is what
//            bounds the direct form in the long run.  Here 256 consecutive bytes of every row go through registers into
//            LDS, 16 accesses an instruction, and the fragments are read from there.  A row's 16-byte pieces are permuted by
//            its number: the 16 rows of a fragment read lie in 16 different bank groups.  The loads of the next stage are in
//            flight while the present one multiplies (a second LDS buffer and 512-byte stages measured slower).  4096 rows
//            x 12544 of 64 adapters of rank 64 in float32: 105 to 109 us, 436 MB read = 4.1 TB/s, matrix pipe 44 % busy
//            (counters: profiles/adapters_clip_kernels.csv).
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
struct __attribute__((packed, aligned(2))) Piece_m {               // 16 bytes from wherever a row's elements lie
    u32x4 v;
};

template <class T>
__device__ inline u32x4 load_piece(const T *p, int left) {          // the first `left` of a piece's elements, zeros behind them
    constexpr int E = 16 / sizeof(T);
    if (left >= E) return ((const Piece_m *)p)->v;
    T e[E];
#pragma unroll
    for (int k = 0; k < E; ++k) e[k] = k < left ? p[k] : (T)0.f;
    return __builtin_bit_cast(u32x4, e);
}

template <class TX, class TW>
struct ContractArgs {
    const TX *x;               // (N,K) stride ldx
    const TW *m;               // (L,R,K) strides sm, ldm
    float *part;               // (slices, N, R16): R rounded up to the tile's 16s, so that a row is whole 16-byte pieces
    long long ldx, ldm, sm;
    int K, R, slices;
};

// elements of K in a stage: 256 bytes a row of m (and so 512 of x where x is float32 and m bf16)
constexpr int stage_elements(int sw) { return 256 / sw; }

// The waves' sums of a tile, (0 + 2) + (1 + 3): into red[0 .. TM R16) + red[TM R16 ..).
template <int NB, int NT, int RT>
__device__ inline void join_waves(const f32x4 (&acc)[NB][RT], float *red) {
    constexpr int TM = 16 * NT, R16 = 16 * RT;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, j = lane & 15, q = lane >> 4;
    float *mine = red + (wave & 1) * TM * R16 + 4 * q * R16 + j;
    if (wave >= 2) {
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int r = 0; r < RT; ++r)
#pragma unroll
                for (int v = 0; v < 4; ++v) mine[(16 * b + v) * R16 + 16 * r] = acc[b][r][v];
    }
    __syncthreads();
    if (wave < 2) {
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int r = 0; r < RT; ++r)
#pragma unroll
                for (int v = 0; v < 4; ++v) mine[(16 * b + v) * R16 + 16 * r] += acc[b][r][v];
    }
    __syncthreads();
}

// The direct form: the fragments of a lane.
template <class TX, class TW>
struct Frag;
template <>
struct Frag<float, float> {
    typedef f32x4 VX;
    typedef f32x4 VM;
    static constexpr int E = 4, STEPS = 4;             // elements of a lane, matrix instructions of a fragment
    static __device__ f32x4 mma(const VX &a, const VM &b, int e, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], c, 0, 0, 0); }
};
template <>
struct Frag<bf16, bf16> {
    typedef bf16x8 VX;
    typedef bf16x8 VM;
    static constexpr int E = 8, STEPS = 1;
    static __device__ f32x4 mma(const VX &a, const VM &b, int, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};
template <>
struct Frag<float, bf16> {                             // float32 gradients against bf16 weights: widened, exact
    typedef f32x4 VX;
    typedef bf16x4 VM;
    static constexpr int E = 4, STEPS = 4;
    static __device__ f32x4 mma(const VX &a, const VM &b, int e, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], (float)b[e], c, 0, 0, 0); }
};
template <class V, class T>
__device__ inline V load_lane(const T *p, int left) {               // the first `left` of a lane's elements, zeros behind them
    struct __attribute__((packed, aligned(2))) M {
        V v;
    };
    constexpr int E = sizeof(V) / sizeof(T);
    if (left >= E) return ((const M *)p)->v;
    V v;
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = e < left ? p[e] : (T)0.f;
    return v;
}

// The waves take neighbouring groups of UN fragments in turn, so that the workgroup reads 256 consecutive bytes of a row or
// more at a time.  UN is the same for full and partial tiles: a row's sum does not depend on the tile it is in.
template <class TX, class TW, int NB, int NT, int RT>
__device__ inline void contract_direct(const ContractArgs<TX, TW> &a, const int *rows, int count, int adapter, int s, float *red) {
    typedef Frag<TX, TW> F;
    typedef typename F::VX VX;
    typedef typename F::VM VM;
    constexpr int E = F::E, KC = 4 * E;
    constexpr int UN = NT + RT >= 6 ? 2 : 16 / (NT + RT) > 4 ? 4 : 16 / (NT + RT);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), j = lane & 15, q = lane >> 4;
    const int chunks = a.K / KC;                       // whole fragments; the last slice also takes what is left of K
    const int c0 = (int)((long long)chunks * s / a.slices), c1 = (int)((long long)chunks * (s + 1) / a.slices);
    const TX *xp[NB];
    const TW *mp[RT];
#pragma unroll
    for (int b = 0; b < NB; ++b) xp[b] = a.x + rows[16 * b + j < count ? 16 * b + j : count - 1] * a.ldx + q * E + (long long)(c0 + wave * UN) * KC;
#pragma unroll
    for (int b = 0; b < RT; ++b) mp[b] = a.m + adapter * a.sm + (16 * b + j < a.R ? 16 * b + j : a.R - 1) * a.ldm + q * E + (long long)(c0 + wave * UN) * KC;
    f32x4 acc[NB][RT];
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int c = 0; c < RT; ++c) acc[b][c] = f32x4{0.f, 0.f, 0.f, 0.f};
    VX xa[UN][NB], xb[UN][NB];
    VM ma[UN][RT], mb[UN][RT];
    auto walk = [&](int n) {                           // the pointers walk along: no address arithmetic but their steps
#pragma unroll
        for (int b = 0; b < NB; ++b) xp[b] += n * KC;
#pragma unroll
        for (int b = 0; b < RT; ++b) mp[b] += n * KC;
    };
    auto load = [&](VX(&xv)[UN][NB], VM(&mv)[UN][RT]) {
#pragma unroll
        for (int u = 0; u < UN; ++u) {
#pragma unroll
            for (int b = 0; b < NB; ++b) xv[u][b] = load_lane<VX>(xp[b] + u * KC, E);
#pragma unroll
            for (int b = 0; b < RT; ++b) mv[u][b] = load_lane<VM>(mp[b] + u * KC, E);
        }
        walk(4 * UN);
    };
    auto multiply1 = [&](const VX(&xv)[NB], const VM(&mv)[RT]) {     // neighbouring instructions on different accumulators
#pragma unroll
        for (int e = 0; e < F::STEPS; ++e)
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int r = 0; r < RT; ++r) acc[b][r] = F::mma(xv[b], mv[r], e, acc[b][r]);
    };
    auto multiply = [&](const VX(&xv)[UN][NB], const VM(&mv)[UN][RT]) {
#pragma unroll
        for (int u = 0; u < UN; ++u) multiply1(xv[u], mv[u]);
    };
    const int groups = (c1 - c0) / (4 * UN);
    if (groups > 0) {
        load(xa, ma);
        for (int g = 1;; g += 2) {
            if (g < groups) load(xb, mb);
            multiply(xa, ma);
            if (g >= groups) break;
            if (g + 1 < groups) load(xa, ma);
            multiply(xb, mb);
            if (g + 1 >= groups) break;
        }
    }
    // single fragments behind the last whole group in turn, then what is left of K: zeros on both sides behind the end
    const int rest = c0 + groups * 4 * UN, end = c1 + (s == a.slices - 1 && chunks * KC < a.K ? 1 : 0);
    walk(wave - wave * UN);
    for (int c = rest + wave; c < end; c += 4) {
        const int left = c < c1 ? E : a.K - c * KC - q * E;
        VX xv[NB];
        VM mv[RT];
#pragma unroll
        for (int b = 0; b < NB; ++b) xv[b] = load_lane<VX>(xp[b], left);
#pragma unroll
        for (int b = 0; b < RT; ++b) mv[b] = load_lane<VM>(mp[b], left);
        multiply1(xv, mv);
        walk(4);
    }
    join_waves<NB, NT, RT>(acc, red);
}

// The staged form.  One operand's rows of a stage: which pieces this thread carries, and where they go.
template <class T, int ROWS, int KS>
struct Carrier {
    static constexpr int E = 16 / sizeof(T), PPR = KS / E, LOADS = ROWS * PPR / 256, STEP = 256 / PPR;
    static_assert(ROWS * PPR % 256 == 0 && PPR >= 16 && 256 % PPR == 0, "a stage is whole loads");
    const T *src[LOADS];
    u32x4 reg[LOADS];
    // row(i) -> pointer to the row's first element of this slice
    template <class F>
    __device__ void start(const F &row) {
        const int piece = threadIdx.x % PPR, first = threadIdx.x / PPR;
#pragma unroll
        for (int i = 0; i < LOADS; ++i) src[i] = row(first + i * STEP) + piece * E;
    }
    __device__ void load(int left) {                                   // left: elements of the slice from the stage on
        const int mine = left - (int)(threadIdx.x % PPR) * E;
        if (left >= KS) {
#pragma unroll
            for (int i = 0; i < LOADS; ++i) reg[i] = ((const Piece_m *)src[i])->v;
        } else {
#pragma unroll
            for (int i = 0; i < LOADS; ++i) reg[i] = load_piece(src[i], mine);
        }
#pragma unroll
        for (int i = 0; i < LOADS; ++i) src[i] += KS;
    }
    __device__ void store(u32x4 *lds) const {
        const int piece = threadIdx.x % PPR, first = threadIdx.x / PPR;
#pragma unroll
        for (int i = 0; i < LOADS; ++i) lds[(first + i * STEP) * PPR + (piece ^ ((first + i * STEP) & 15))] = reg[i];
    }
};

template <class T, int KS>
__device__ inline u32x4 fragment(const u32x4 *lds, int row, int piece) {
    constexpr int PPR = KS * sizeof(T) / 16;
    return lds[row * PPR + (piece ^ (row & 15))];
}

template <class TX, class TW, int NB, int NT, int RT>
__device__ inline void contract_staged(const ContractArgs<TX, TW> &a, const int *rows, int count, int adapter, int s, u32x4 *lds) {
    constexpr int R16 = 16 * RT, KS = stage_elements(sizeof(TW)), E = 16 / sizeof(TX), KC = 4 * E;
    constexpr int FRAGMENTS = KS / KC / 4;             // of a stage, for each wave
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), j = lane & 15, q = lane >> 4;
    const int chunks = (a.K + KC - 1) / KC;            // slices are cut between fragments
    const int k0 = (int)((long long)chunks * s / a.slices) * KC, k9 = (int)((long long)chunks * (s + 1) / a.slices) * KC, k1 = k9 < a.K ? k9 : a.K;
    u32x4 *lx = lds, *lm = lds + 16 * NB * (KS * sizeof(TX) / 16);
    Carrier<TX, 16 * NB, KS> cx;
    Carrier<TW, R16, KS> cm;
    cx.start([&](int i) { return a.x + rows[i < count ? i : count - 1] * a.ldx + k0; });
    cm.start([&](int i) { return a.m + adapter * a.sm + (i < a.R ? i : a.R - 1) * a.ldm + k0; });
    f32x4 acc[NB][RT];
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int c = 0; c < RT; ++c) acc[b][c] = f32x4{0.f, 0.f, 0.f, 0.f};
    int k = k0;
    cx.load(k1 - k);
    cm.load(k1 - k);
    for (;;) {
        cx.store(lx);
        cm.store(lm);
        __syncthreads();
        k += KS;
        if (k < k1) {
            cx.load(k1 - k);
            cm.load(k1 - k);
        }
#pragma unroll
        for (int f = 0; f < FRAGMENTS; ++f) {
            const int g = f * 4 + wave;
            if constexpr (sizeof(TX) == 2) {
                bf16x8 xv[NB], mv[RT];
#pragma unroll
                for (int b = 0; b < NB; ++b) xv[b] = __builtin_bit_cast(bf16x8, fragment<TX, KS>(lx, 16 * b + j, 4 * g + q));
#pragma unroll
                for (int r = 0; r < RT; ++r) mv[r] = __builtin_bit_cast(bf16x8, fragment<TW, KS>(lm, 16 * r + j, 4 * g + q));
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int r = 0; r < RT; ++r) acc[b][r] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(xv[b], mv[r], acc[b][r], 0, 0, 0);
            } else {                                   // lane (j, q) has k = 4 q .. 4 q + 3: four steps with k in another order
                f32x4 xv[NB], mv[RT];
#pragma unroll
                for (int b = 0; b < NB; ++b) xv[b] = __builtin_bit_cast(f32x4, fragment<TX, KS>(lx, 16 * b + j, 4 * g + q));
#pragma unroll
                for (int r = 0; r < RT; ++r) {
                    if constexpr (sizeof(TW) == 4) {
                        mv[r] = __builtin_bit_cast(f32x4, fragment<TW, KS>(lm, 16 * r + j, 4 * g + q));
                    } else {                           // float32 gradients against bf16 weights: widened, exact
                        const bf16x8 w = __builtin_bit_cast(bf16x8, fragment<TW, KS>(lm, 16 * r + j, 2 * g + (q >> 1)));
#pragma unroll
                        for (int e = 0; e < 4; ++e) mv[r][e] = (float)(q & 1 ? w[4 + e] : w[e]);
                    }
                }
#pragma unroll
                for (int e = 0; e < 4; ++e)
#pragma unroll
                    for (int b = 0; b < NB; ++b)
#pragma unroll
                        for (int r = 0; r < RT; ++r) acc[b][r] = __builtin_amdgcn_mfma_f32_16x16x4f32(xv[b][e], mv[r][e], acc[b][r], 0, 0, 0);
            }
        }
        __syncthreads();
        if (k >= k1) break;
    }
    join_waves<NB, NT, RT>(acc, (float *)lds);
}

template <class TX, class TW, int NT, int RT, bool STAGED>
__global__ __launch_bounds__(256, 2) void contract_kernel(const ContractArgs<TX, TW> a, const Plan p) {
    constexpr int TM = 16 * NT, R16 = 16 * RT, KS = stage_elements(sizeof(TW));
    constexpr int STAGE = STAGED ? (TM * sizeof(TX) + R16 * sizeof(TW)) * KS : 0, SUMS = 2 * TM * R16 * 4, BYTES = STAGE > SUMS ? STAGE : SUMS;
    __shared__ TileLds tl;
    __shared__ u32x4 lds[BYTES / 16];
    float *red = (float *)lds;
    const int tid = threadIdx.x;
    const int t = blockIdx.x / a.slices, s = blockIdx.x - t * a.slices;
    int adapter;
    const int count = __builtin_amdgcn_readfirstlane(find_tile(p, t, TM, tl, adapter));
    if (count == 0 || adapter >= p.L) return;
    auto tile = [&](auto nb) {
        constexpr int NB = decltype(nb)::value;
        if constexpr (STAGED) contract_staged<TX, TW, NB, NT, RT>(a, tl.rows, count, adapter, s, lds);
        else contract_direct<TX, TW, NB, NT, RT>(a, tl.rows, count, adapter, s, red);
    };
    if (NT == 1 || count <= 16) tile(std::integral_constant<int, 1>());
    else if (NT == 2 || count <= 32) tile(std::integral_constant<int, 2>());
    else if (count <= 48) tile(std::integral_constant<int, NT == 4 ? 3 : 2>());
    else tile(std::integral_constant<int, NT>());
    float *part = a.part + (long long)s * p.N * R16;
    for (int e = 4 * tid; e < count * R16; e += 1024)
        *(f32x4 *)(part + (long long)tl.rows[e / R16] * R16 + e % R16) = *(const f32x4 *)(red + e) + *(const f32x4 *)(red + TM * R16 + e);
}

// --------------------------------------------------------------------------------------------------------------- expand
// out[n][u] (+)= sum_r h[n][r] m[i][r][u] with h = scale[i] sum_s part[s]: one wave per 64 columns, lane (j, q) holding four
// consecutive ones, so that loads of m and stores of out are 256 bytes a row.  Bound by reading m and writing out.  h is
// joined from the K slices on the way (and stored, without the scale, where the caller keeps it).  float32 matrix instruction
// for both types: bf16 weights are widened, h is not rounded.  One row x 1470: 5.3 us; 4096 rows x 539 of rank 64: 20.5 us, 49 MB
// moved, the K slices read again by every column block among them; the gradient of x of 2048 rows x 12544 of rank 32: 39 us, 131 MB
// moved = 3.3 TB/s (counters: profiles/adapters_clip_kernels.csv).
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

// dst[row][r] (row stride LD) = f * sum_s part[s][rows[row]][r], zero for r in [R, R16); also stored to keep (N, R), without f
__device__ inline void put4(float *dst, f32x4 v, float f, float *keep, long long n, int r, int R) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const bool live = r + e < R;
        dst[e] = live ? f * v[e] : 0.f;
        if (keep && live) keep[n * R + r + e] = v[e];
    }
}
template <int R16, int LD>
__device__ inline void join(float *dst, f32x4 *lds, const float *__restrict__ part, int slices, int N, const int *rows, int count, int R,
                            float f, float *keep) {
    constexpr int R4 = R16 / 4;
    const int tid = threadIdx.x;
    const long long slab = (long long)N * R16;
    if (slices > 4 && N <= 64 / R4) {           // a batch of few values: 4 to 8 threads to a value, as many for every tile
        const int n = N * R4, most = 256 / n, groups = most < 8 ? most : 8, e = tid % n, g = tid / n, row = e / R4, r = 4 * (e % R4);
        f32x4 v = {0.f, 0.f, 0.f, 0.f};
        if (g < groups && row < count) {
            const float *src = part + (long long)rows[row] * R16 + r;
#pragma unroll 8
            for (int s = g; s < slices; s += groups) v += *(const f32x4 *)(src + s * slab);
        }
        lds[tid] = v;
        __syncthreads();
        if (tid < n && row < count) {
            f32x4 sum = v;
            for (int k = 1; k < groups; ++k) sum += lds[k * n + tid];
            put4(dst + row * LD + r, sum, f, keep, rows[row], r, R);
        }
    } else {
        for (int e = tid; e < count * R4; e += 256) {
            const int row = e / R4, r = 4 * (e % R4);
            const float *src = part + (long long)rows[row] * R16 + r;
            f32x4 v = *(const f32x4 *)src;
#pragma unroll 8
            for (int s = 1; s < slices; ++s) v += *(const f32x4 *)(src + s * slab);
            put4(dst + row * LD + r, v, f, keep, rows[row], r, R);
        }
    }
    __syncthreads();
}

template <class T>
struct ExpandArgs {
    const float *part;         // (slices, N, R16)
    const T *m;                // (L, R, U) strides sm, ldm
    const float *scale;        // (L)
    float *out, *keep;         // (N, U) stride ldo; (N, R) or null
    long long ldm, sm, ldo;
    int U, R, slices, blocks, accumulate;          // `blocks` of 256 columns, one to a workgroup
    int TM, subs, max_tiles;   // rows of a tile; a workgroup takes 16 NT of them, `subs` workgroups cover the tile
};

template <class T, int NT, int RT>
__global__ __launch_bounds__(256, NT == 1 ? 4 : RT <= 2 ? 3 : 1) void expand_kernel(const ExpandArgs<T> a, const Plan p) {
    constexpr int TM = 16 * NT, R16 = 16 * RT, LD = R16 + 4;
    __shared__ TileLds tl;
    __shared__ __attribute__((aligned(16))) float h[TM * LD];
    __shared__ f32x4 sums[256];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), j = lane & 15, q = lane >> 4;
    // Workgroups that read the same part of m belong on one XCD (blockIdx % 8), whose L2 then fetches it once: the tiles of an
    // adapter on the same columns where there are 8 column blocks or more, the row blocks of a tile below that (gradient of x
    // at 2048 rows x 12544: 39 -> 38 us; 4096 rows x 539 of rank 64: 24 -> 22.5, before the ranks came 16 at a time).
    int t, sub, block;
    if (a.blocks >= 8) {
        const int b8 = (a.blocks + 7) & ~7, ts = blockIdx.x / b8;
        block = blockIdx.x - ts * b8;
        t = ts / a.subs;
        sub = ts - t * a.subs;
    } else {
        const int g = blockIdx.x >> 3, gs = g / a.subs, pair = gs * 8 + (blockIdx.x & 7);
        sub = g - gs * a.subs;
        t = pair / a.blocks;
        block = pair - t * a.blocks;
    }
    if (t >= a.max_tiles || block >= a.blocks) return;
    int adapter;
    const int all = find_tile(p, t, a.TM, tl, adapter) - sub * TM, count = __builtin_amdgcn_readfirstlane(all < TM ? all : TM);
    if (count <= 0) return;
    const int *rows = tl.rows + sub * TM;
    float *keep = block == 0 ? a.keep : nullptr;
    if (adapter >= p.L) {                              // no adapter: zeros (or out as it is); an index behind the bank: NaN
        const int c = block * 256 + tid;
        for (int row = 0; row < count; ++row) {
            const int n = rows[row];
            const bool bad = p.index[n] >= 0;
            const float v = bad ? __builtin_nanf("") : 0.f;
            if ((bad || !a.accumulate) && c < a.U) a.out[n * a.ldo + c] = v;
            if (keep && tid < a.R) keep[(long long)n * a.R + tid] = v;
        }
        return;
    }
    const int u = block * 256 + wave * 64 + 4 * j, left = a.U - u;
    const T *mp = a.m + adapter * a.sm + u;
    auto load = [&](f32x4 (&v)[4], int r0) {           // ranks r0 + 4 q .. r0 + 4 q + 3 of this lane's columns
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int r = r0 + 4 * q + e;
            const T *at = mp + (r < a.R ? r : 0) * a.ldm;
            if (u - 4 * j + 64 <= a.U) v[e] = load4(at);             // (uniform) all of the wave's columns are there
            else v[e] = left > 0 ? load4(at, left) : f32x4{0.f, 0.f, 0.f, 0.f};
        }
        if (r0 + 16 > a.R)                             // ranks that are not there: zeros on both sides
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (r0 + 4 * q + e >= a.R) v[e] = f32x4{0.f, 0.f, 0.f, 0.f};
    };
    // One row block: 16 ranks at a time, the next ones on their way (few registers, many workgroups to a CU).  Several: all ranks
    // stay in registers for them.
    constexpr int HELD = NT == 1 && RT > 1 ? 2 : RT;
    f32x4 m[HELD][4];
#pragma unroll
    for (int k = 0; k < (NT == 1 ? 1 : RT); ++k) load(m[k], 16 * k);
    for (int e = tid; e < (TM - count) * LD; e += 256) h[count * LD + e] = 0.f;
    join<R16, LD>(h, sums, a.part, a.slices, p.N, rows, count, a.R, a.scale[adapter], keep);
#pragma unroll
    for (int b = 0; b < NT; ++b) {
        if (16 * b >= count) break;
        f32x4 acc[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) acc[c] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < RT; ++k) {
            if (NT == 1 && k + 1 < RT) load(m[(k + 1) % HELD], 16 * (k + 1));
            const f32x4 hv = *(const f32x4 *)(h + (16 * b + j) * LD + 16 * k + 4 * q);
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int c = 0; c < 4; ++c) acc[c] = __builtin_amdgcn_mfma_f32_16x16x4f32(hv[e], m[k % HELD][e][c], acc[c], 0, 0, 0);
        }
#pragma unroll
        for (int v = 0; v < 4; ++v) {
            const int row = 16 * b + 4 * q + v;
            if (row >= count || left <= 0) continue;
            float *o = a.out + rows[row] * a.ldo + u;
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
// out[i][r][k] = scale[i] sum over the rows n of adapter i of g[n][r] x[n][k], g = sum_s part[s]: lane (j, q) of a wave holds
// four consecutive columns of row 4 step + q, so that loads of x and stores of out are 256 bytes a row.  Bound by reading x
// and writing out once.  A wave runs through the adapter's rows by itself, 16 at a time, reading g from L2: a version that put
// g into LDS for the workgroup stood still at its barriers (2048 rows x 12544 of 16 adapters of rank 32: 81 us, now 44 to 56: 154 MB moved).
// Two such products (A's gradient and B's) share a launch.  Loading the next 16 rows ahead costs more registers than it hides
// latency (74 us): occupancy carries it.
//   few rows to an adapter: a wave has 64 columns and all rows of the adapter or piece, a workgroup 256 columns;
//   many (SPLIT): the four waves have the same 64 columns and a quarter of the rows each, joined in LDS (128 or 256 columns to
//   a wave read g less often and measured slower, 54 against 61 and 99 us: the adapter with the most rows has too few waves).
template <class T>
struct RowsArgs {
    const float *part;         // (slices, N, ldp)
    const T *x;                // (N, K) stride ldx
    float *out;                // (L, R, K) strides so, ldo
    long long ldx, ldo, so;
    int K, slices, ldp, blocks, ranks;     // `blocks` workgroups to an adapter (or piece) and 64 ranks, `ranks` times 64 ranks
    float *apart;              // (slots, R, lda) sums of the pieces of adapters with several
    long long lda;             // K rounded up to 16 bytes
};

// the rows of adapter i in ascending order, up to kSelfPlan of them: every wave writes and reads the same list
template <int W>
__device__ inline int rows_by_ballots(const Plan &p, int i, int *rows) {
    const int lane = threadIdx.x & 63;
    int total = 0;
#pragma unroll
    for (int w = 0; w < W; ++w) {
        const int n = 64 * w + lane;
        const bool mine = n < p.N && p.index[n] == i;
        const unsigned long long vote = __ballot(mine);
        if (mine) rows[total + __popcll(vote & ((1ull << lane) - 1))] = n;
        total += __popcll(vote);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    return total;
}

template <class T, int RT, bool SPLIT>
__device__ inline void rows_tile(const RowsArgs<T> &a, const Plan &p, const float *scale, int R, int block, float *red, int *own) {
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), j = lane & 15, q = lane >> 4;
    const int ir = block / a.blocks, cb = block - ir * a.blocks, item = ir / a.ranks, r0 = 64 * (ir - item * a.ranks);
    const int k0 = SPLIT ? cb * 64 : cb * 256 + wave * 64, k = k0 + 4 * j;
    int total, i = item, slot = -1;
    const int *rows = own;                             // (LDS) or the sorted list's
    if (p.pieces) {
        const int4 piece = p.pieces[item];
        i = piece.x;
        rows = p.perm + piece.y;
        total = piece.z;
        slot = piece.w;
        if (i < 0) return;
    } else if (p.perm) {
        const int first = p.offs[i];
        total = p.offs[i + 1] - first;
        rows = p.perm + first;
    } else {
        total = p.N <= 64 ? rows_by_ballots<1>(p, i, own) : rows_by_ballots<4>(p, i, own);
    }
    total = __builtin_amdgcn_readfirstlane(total);
    const float f = slot >= 0 ? 1.f : total ? scale[i] : 0.f;
    f32x4 acc[RT][4];
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
        for (int c = 0; c < 4; ++c) acc[t][c] = f32x4{0.f, 0.f, 0.f, 0.f};
    const long long slab = (long long)p.N * a.ldp;
    const bool whole = k0 + 64 <= a.K;                 // no lane's columns reach behind the end
    const bool inside = r0 + 16 * RT <= a.ldp;         // no rank behind a row of part
    const int stride = SPLIT ? 4 : 1, groups = (total + 15) >> 4;
    int n[4];                                          // this lane's rows of the next group
    auto find = [&](int group) {
        if (group < groups)
#pragma unroll
            for (int s = 0; s < 4; ++s) n[s] = rows[16 * group + 4 * s + q < total ? 16 * group + 4 * s + q : 0];
    };
    auto load = [&](f32x4(&x)[4], float(&g)[4][RT], int group) {
        if (group >= groups) return;
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const T *xp = a.x + n[s] * a.ldx + k;
            if (whole) x[s] = load4(xp);
            else x[s] = k < a.K ? load4(xp, a.K - k) : f32x4{0.f, 0.f, 0.f, 0.f};
        }
        if (inside) {
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                const float *gp = a.part + (long long)n[s] * a.ldp + r0 + j;
#pragma unroll
                for (int t = 0; t < RT; ++t) g[s][t] = gp[16 * t];
            }
        } else {                                       // the caller's h: no ranks behind R to read
#pragma unroll 1
            for (int t = 0; t < RT; ++t) {
                const int r = r0 + 16 * t + j < R ? r0 + 16 * t + j : 0;
#pragma unroll
                for (int s = 0; s < 4; ++s) {
                    const float v = a.part[(long long)n[s] * a.ldp + r];
#pragma unroll
                    for (int k = 0; k < RT; ++k) g[s][k] = k == t ? v : g[s][k];
                }
            }
        }
#pragma unroll 1
        for (int sl = 1; sl < a.slices; ++sl)          // (only kernels' partial sums come in slices)
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                const float *gp = a.part + sl * slab + (long long)n[s] * a.ldp + r0 + j;
#pragma unroll
                for (int t = 0; t < RT; ++t) g[s][t] += gp[16 * t];
            }
    };
    auto multiply = [&](f32x4(&x)[4], float(&g)[4][RT], int group) {
        if (16 * group + 16 > total)                   // (uniform) behind the last row: another row's values, zeros on both sides
#pragma unroll
            for (int s = 0; s < 4; ++s)
                if (16 * group + 4 * s + q >= total) {
                    x[s] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int t = 0; t < RT; ++t) g[s][t] = 0.f;
                }
#pragma unroll
        for (int s = 0; s < 4; ++s)
#pragma unroll
            for (int t = 0; t < RT; ++t)
#pragma unroll
                for (int c = 0; c < 4; ++c) acc[t][c] = __builtin_amdgcn_mfma_f32_16x16x4f32(g[s][t], x[s][c], acc[t][c], 0, 0, 0);
    };
    int group = SPLIT ? wave : 0;
    find(group);
    for (; group < groups; group += stride) {
        f32x4 x[4];
        float g[4][RT];
        load(x, g, group);
        find(group + stride);
        multiply(x, g, group);
    }
    float *out = slot >= 0 ? a.apart + slot * (R * a.lda) : a.out + i * a.so;
    const long long ldo = slot >= 0 ? a.lda : a.ldo;
    auto put = [&](int r, int c, f32x4 val) {
        if (r >= R || c >= a.K) return;
        float *o = out + r * ldo + c;
        if (a.K - c >= 4) *(f32x4_m *)o = f * val;
        else
            for (int y = 0; y < a.K - c; ++y) o[y] = f * val[y];
    };
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        if (SPLIT) {
            __syncthreads();
#pragma unroll
            for (int v = 0; v < 4; ++v)
                *(f32x4 *)(red + wave * 1024 + (4 * q + v) * 64 + 4 * j) = f32x4{acc[t][0][v], acc[t][1][v], acc[t][2][v], acc[t][3][v]};
            __syncthreads();
            const f32x4 *e = (const f32x4 *)red + tid;
            put(r0 + 16 * t + (tid >> 4), k0 + 4 * (tid & 15), (e[0] + e[256]) + (e[512] + e[768]));
        } else {
#pragma unroll
            for (int v = 0; v < 4; ++v) put(r0 + 16 * t + 4 * q + v, k, f32x4{acc[t][0][v], acc[t][1][v], acc[t][2][v], acc[t][3][v]});
        }
    }
}

template <class T, int RT, bool SPLIT>
__global__ __launch_bounds__(256) void rows_kernel(const RowsArgs<T> a, const RowsArgs<float> b, const Plan p, const float *__restrict__ scale,
                                                   int R, int b_blocks) {
    __shared__ int own[kSelfPlan];
    __shared__ __attribute__((aligned(16))) float red[SPLIT ? 4096 : 4];
    if ((int)blockIdx.x >= b_blocks) rows_tile<T, RT, SPLIT>(a, p, scale, R, blockIdx.x - b_blocks, red, own);
    else rows_tile<float, RT, SPLIT>(b, p, scale, R, blockIdx.x, red, own);          // (fewer: a long one last would be waited for)
}

// out[i] = scale[i] times the sum of the pieces of an adapter that has several, in order
template <class T>
__device__ inline void join_pieces(const RowsArgs<T> &a, int i, int slot, int n, float f, int R, long long first, long long step) {
    const long long row4 = a.lda / 4;
    for (long long e = first; e < R * row4; e += step) {
        const int r = (int)(e / row4), c = 4 * (int)(e - r * row4);
        const float *src = a.apart + (slot * (long long)R + r) * a.lda + c;
        f32x4 v = *(const f32x4 *)src;
#pragma unroll 4
        for (int k = 1; k < n; ++k) v += *(const f32x4 *)(src + k * (R * a.lda));
        float *o = a.out + i * a.so + r * a.ldo + c;
        if (a.K - c >= 4) *(f32x4_m *)o = f * v;
        else
            for (int y = 0; y < a.K - c; ++y) o[y] = f * v[y];
    }
}
template <class T>
__global__ __launch_bounds__(256) void join_pieces_kernel(const RowsArgs<T> a, const RowsArgs<float> b, const int2 *__restrict__ slots,
                                                          const float *__restrict__ scale, int R, int blocks) {
    const int slot = blockIdx.x / blocks, k = blockIdx.x - slot * blocks;
    const int2 s = slots[slot];                        // {adapter, its pieces: at the first of its slots alone}
    if (s.y == 0) return;
    const float f = scale[s.x];
    join_pieces(a, s.x, slot, s.y, f, R, k * 256ll + threadIdx.x, blocks * 256ll);
    join_pieces(b, s.x, slot, s.y, f, R, k * 256ll + threadIdx.x, blocks * 256ll);
}

// part[0] = sum_s part[s], in order: where so many slices were needed that every reader joining them would cost more
__global__ __launch_bounds__(256) void join_kernel(float *part, long long n4, int slices) {
    f32x4 *p = (f32x4 *)part;
    for (long long e = blockIdx.x * 256ll + threadIdx.x; e < n4; e += gridDim.x * 256ll) {
        f32x4 v = p[e];
#pragma unroll 8
        for (int s = 1; s < slices; ++s) v += p[s * n4 + e];
        p[e] = v;
    }
}

// ------------------------------------------------------------------------------------------------------------- the host
int check_sizes(const char *what, int N, int K, int U, int L, int R) {
    constexpr int kMost = 1 << 30;
    TY1_REQUIRE(N >= 0 && K > 0 && U > 0 && N <= kMost && K <= kMost && U <= kMost, "%s: bad dimensions N=%d K=%d U=%d", what, N, K, U);
    TY1_REQUIRE(L >= 1 && L <= kMaxAdapters, "%s: %d adapters, 1 to %d are supported", what, L, kMaxAdapters);
    TY1_REQUIRE(R >= 1 && R <= kMaxRank, "%s: rank %d, 1 to %d are supported", what, R, kMaxRank);
    return 0;
}

// Everything that follows from the sizes alone: tile height, number of tiles at the most, and the scratch memory's layout.
struct Layout {
    int rt, nt;                // ranks and rows of a tile, in 16s
    int max_tiles;
    bool sorted;               // plan_kernel's list, not each workgroup's own
    bool pieced;               // backward of a long batch: adapters in pieces of kPiece rows
    int max_pieces, max_slots;
    size_t perm, offs, tiles, pieces, slots, apart_a, apart_b, part, part2, bytes;
    int slices, slices2;       // K slices of the first contraction and, backward only, of the one that computes h again
};

int slices_for(int tiles, int K, int least) {
    // enough workgroups for every CU to hold four, but at least `least` elements of K for a workgroup
    const int want = (4 * 256 + tiles - 1) / tiles, most = (K + least - 1) / least;
    const int s = want < most ? want : most;
    return s < 1 ? 1 : s > 64 ? 64 : s;
}

Layout layout(int N, int K, int U, int L, int R, bool back) {
    Layout y;
    y.rt = R <= 16 ? 1 : R <= 32 ? 2 : R <= 64 ? 4 : 8;
    const int classes = L < N ? L : N;
    // 64 rows to a tile (32 at ranks above 64) from 48 rows an adapter on, from 20 where the tiles and slices of 512 elements
    // still make two workgroups a CU, and 16 rows below.  Forward, x 12544: 1024 rows of 32 adapters of rank 32 38 us tall, 50
    // low; 4096 of 64 of rank 64 146 and 222; 1024 of 128 adapters of rank 16 45 tall, 42 low; 333 rows x 4999 of 7 adapters of
    // rank 11 19 tall, 17 low.
    const auto tiles = [&](int nt) { return (long long)N / (16 * nt) + (L + 1 < N ? L + 1 : N); };
    const int tall = y.rt == 8 ? 2 : 4, axis = back ? U : K;
    y.nt = N >= 48ll * classes || (N >= 20ll * classes && tiles(tall) * ((axis + 511) / 512) >= 512) ? tall : 1;
    const long long most = tiles(y.nt);
    y.max_tiles = (int)(most < N ? most : N > 1 ? N : 1);
    y.sorted = N > kSelfPlan;
    // Slices that every reader joins by itself: 512 elements (256 make one frame's contraction 0.7 us faster and what reads it
    // 1 us slower).  Joined by a launch of their own: 256 (2048 rows x 1470 of rank 32: 12.5 -> 10.2 us).
    y.slices = slices_for(y.max_tiles, back ? U : K, back && y.sorted ? 256 : 512);
    y.slices2 = back ? slices_for(y.max_tiles, K, 256) : 0;
    size_t at = 0;
    auto take = [&](size_t n) {
        const size_t here = at;
        at += (n + 255) & ~(size_t)255;
        return here;
    };
    y.perm = take(y.sorted ? 4 * (size_t)N : 0);
    y.offs = take(y.sorted ? 4 * ((size_t)L + 1) : 0);
    y.tiles = take(y.sorted ? 16 * (size_t)y.max_tiles : 0);
    // Pieces where one adapter's rows would hold up the rest: from 700 rows an adapter on, and from 4096 rows whatever the mean (a
    // batch can lean on one adapter).  Backward x 12544: one adapter, 2048 rows of rank 32 64 us in pieces, 91 whole; 1024 of rank
    // 16 39 and 48; 2048 rows of 8 adapters 66 and 57; 4096 rows of 64 adapters of rank 64 210 and 206, with a fourth of them on
    // one adapter 163 and 305 (539 units).  At most one piece an adapter and one for every kPiece rows; slots only for adapters
    // with more rows than that, so at most one for every kPiece / 2 rows (memory is reserved for all of them).  The host does not see
    // the index: of 64 adapters of rank 64, a fourth of the rows on one, h kept and no dx, 4095 rows take 250 us whole and 4096 take 158
    // in pieces, where rows spread evenly take 154 and 156.
    y.pieced = back && y.sorted && (N >= 700ll * classes || N >= 4096);
    y.max_pieces = y.pieced ? L + N / kPiece : 0;
    y.max_slots = y.pieced ? N / (kPiece / 2) : 0;
    y.pieces = take(16 * (size_t)y.max_pieces);
    y.slots = take(8 * (size_t)y.max_slots);
    y.apart_a = take(16 * (size_t)y.max_slots * R * ((K + 3ll) / 4));
    y.apart_b = take(16 * (size_t)y.max_slots * R * ((U + 3ll) / 4));
    y.part = take(64 * (size_t)y.slices * N * y.rt);
    y.part2 = take(64 * (size_t)y.slices2 * N * y.rt);
    y.bytes = at < 256 ? 256 : at;
    return y;
}

Plan make_plan(const Layout &y, char *ws, const int32_t *index, int N, int L, hipStream_t s) {
    Plan p = {index, N, L, nullptr, nullptr, nullptr, nullptr};
    if (!y.sorted) return p;
    int waves = 15360 / (L + 1), bits = 1;             // 60 KB of counters
    waves = waves > 16 ? 16 : waves;
    while (1 << bits < L + 1) ++bits;
    int *perm = (int *)(ws + y.perm), *offs = (int *)(ws + y.offs);
    int4 *tiles = (int4 *)(ws + y.tiles), *pieces = y.pieced ? (int4 *)(ws + y.pieces) : nullptr;
    const size_t lds = (size_t)waves * (L + 1) * 4;
#define CALL(PIECES) plan_kernel<PIECES><<<dim3(1), dim3(1024), lds, s>>>(index, N, L, waves, bits, 16 * y.nt, perm, offs, tiles, y.max_tiles, pieces, y.max_pieces, (int2 *)(ws + y.slots), y.max_slots)
    if (y.pieced) CALL(true); else CALL(false);
#undef CALL
    p.perm = perm;
    p.offs = offs;
    p.tiles = tiles;
    p.pieces = pieces;
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
    // staged where tall tiles fill the chip with long slices: 4096 rows x 12544 of rank 64 take 104 us against 115 to 130 direct;
    // direct where latency counts: one row 4.7 us against 5.5, 2048 rows x 1470 of rank 32 in three slices 13.0 against 15.9
    const bool staged = y.nt > 1 && y.max_tiles * slices >= 512 && K / slices * (int)sizeof(TX) >= 2048;
#define CALL(NT, RT)                                                                                 \
    do {                                                                                             \
        if (NT > 1 && staged) contract_kernel<TX, TM, NT, RT, (NT > 1)><<<grid, dim3(256), 0, s>>>(a, p); \
        else contract_kernel<TX, TM, NT, RT, false><<<grid, dim3(256), 0, s>>>(a, p);                \
    } while (0)
    TY1_BY_TILE(y, CALL);
#undef CALL
}

template <class T>
void expand(const Layout &y, const Plan &p, const float *part, int slices, const T *m, long long ldm, long long sm, const float *scale, float *out,
            long long ldo, float *keep, int U, int R, int accumulate, hipStream_t s) {
    // few workgroups: 16 rows each instead of the tile's height
    const int blocks = (U + 255) / 256, nt = (long long)y.max_tiles * blocks < 1024 ? 1 : y.nt, subs = y.nt / nt;
    const ExpandArgs<T> a = {part, m, scale, out, keep, ldm, sm, ldo, U, R, slices, blocks, accumulate, 16 * y.nt, subs, y.max_tiles};
    const dim3 grid((unsigned)(blocks >= 8 ? y.max_tiles * subs * ((blocks + 7) & ~7) : (y.max_tiles * blocks + 7) / 8 * 8 * subs));
    Layout z = y;
    z.nt = nt;
#define CALL(NT, RT) expand_kernel<T, NT, RT><<<grid, dim3(256), 0, s>>>(a, p)
    TY1_BY_TILE(z, CALL);
#undef CALL
}

void join_slices(const Layout &y, float *part, int &slices, int N, hipStream_t s) {
    if (slices == 1) return;
    const long long n4 = 4ll * N * y.rt, blocks = (n4 + 255) / 256;
    join_kernel<<<dim3((unsigned)(blocks < 1024 ? blocks : 1024)), dim3(256), 0, s>>>(part, n4, slices);
    slices = 1;
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
    if (check_grid(what, y, y.slices) || check_grid(what, y, 8 * ((U + 255ll) / 256))) return 1;
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
    Layout y = layout(N, K, U, L, R, true);
    TY1_REQUIRE(ws && ((uintptr_t)ws & 15) == 0 && ws_bytes >= y.bytes, "%s: workspace null, not 16-byte aligned, or %zu bytes where %zu are needed", what,
                ws_bytes, y.bytes);
    // Many rows to an adapter are split over the waves of a workgroup (rows_tile), unless the adapters fill the chip without it:
    // 500 rows of 8 adapters at rank 16 12 us split, 31 not; 2048 of 16 at rank 32 54 and 142; 4096 of 64 at rank 64 (the whole
    // call) 224 split, 174 not; 600 rows of 20 adapters, fewer than 32 each, 37 split, 33 not (measured without pieces).
    const int items = y.pieced ? y.max_pieces : L;
    const bool split = N > 32ll * (L < N ? L : N) && items * ((K + 255ll) / 256 + (U + 255ll) / 256) < 2048;
    const int wide = split ? 64 : 256;
    const long long ka = (K + wide - 1ll) / wide, ub = (U + wide - 1ll) / wide;
    TY1_REQUIRE(2 * items * (ka + ub) < (1ll << 24), "%s: %d adapters of %d x %d are more than one launch holds", what, L, K, U);
    const int each = y.pieced ? 8192 / y.max_slots : 0, blocks = each < 16 ? 16 : each > 256 ? 256 : each;      // to a slot, in the joining launch
    TY1_REQUIRE((long long)y.max_slots * blocks < (1ll << 24), "%s: %d rows are more than one launch holds", what, N);
    if (check_grid(what, y, y.slices) || check_grid(what, y, y.slices2) || (dx && check_grid(what, y, 8 * ((K + 255ll) / 256)))) return 1;
    hipStream_t s = (hipStream_t)stream;
    ty1::ProfScope prof("adapter_backward", s, 2.0 * N * R * (K * (dx ? 2.0 : 1.0) + 2.0 * U),
                        sizeof(T) * (double)N * K + 4.0 * N * U + 4.0 * L * R * ((double)K + U) + (dx ? 4.0 * N * K : 0.0));
    Plan p = {index, N, L, nullptr, nullptr, nullptr, nullptr};
    float *part = (float *)((char *)ws + y.part), *part2 = (float *)((char *)ws + y.part2);
    if (N > 0) {
        p = make_plan(y, (char *)ws, index, N, L, s);
        contract(y, p, dz, lddz, b, ldb, sb, part, U, R, y.slices, s);
        if (y.sorted) join_slices(y, part, y.slices, N, s);       // read by a workgroup for every 64 columns: once is worth a launch
        if (!h) {
            contract(y, p, x, ldx, a, lda, sa, part2, K, R, y.slices2, s);
            join_slices(y, part2, y.slices2, N, s);
        }
    }
    const int ranks = y.rt == 8 ? 2 : 1;               // (128 ranks of accumulators would leave one wave a SIMD)
    const RowsArgs<T> ra = {part, x, da, ldx, ldda, sda, K, y.slices, 16 * y.rt, (int)ka, ranks, (float *)((char *)ws + y.apart_a), (K + 3ll) & ~3ll};
    const RowsArgs<float> rb = {h ? h : part2, dz, db, lddz, lddb, sdb, U, 1, h ? R : 16 * y.rt, (int)ub, ranks, (float *)((char *)ws + y.apart_b), (U + 3ll) & ~3ll};
    const dim3 grid((unsigned)(items * ranks * (ka + ub)));
#define CALL(RT)                                                                                                                    \
    do {                                                                                                                            \
        if (split) rows_kernel<T, RT, true><<<grid, dim3(256), 0, s>>>(ra, rb, p, scale, R, (int)(items * ranks * ub));                          \
        else rows_kernel<T, RT, false><<<grid, dim3(256), 0, s>>>(ra, rb, p, scale, R, (int)(items * ranks * ub));                               \
    } while (0)
    if (y.rt == 1) CALL(1); else if (y.rt == 2) CALL(2); else CALL(4);
#undef CALL
    if (y.pieced) {
        join_pieces_kernel<T><<<dim3((unsigned)(y.max_slots * blocks)), dim3(256), 0, s>>>(ra, rb, (const int2 *)((char *)ws + y.slots), scale, R, blocks);
    }
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
