// Orthogonalised updates (Newton-Schulz products) and the optimiser step built on them.
//
// X_0 = G / (|G|_F + eps);  X_{k+1} = a X_k + (b A_k + c A_k^2) X_k,  A_k = X_k X_k^T:  an odd polynomial applied to
// the singular values of G, which the usual coefficients bring near one in five steps.  G is m x n with m <= n
// (a tall matrix is worked on as its transpose).
//
// Gram form.  With Q_k = a I + b A_k + c A_k^2 the steps are X_{k+1} = Q_k X_k and A_{k+1} = Q_k A_k Q_k; all Q_k and
// A_k are polynomials of A_0, symmetric, and commute.  So L steps are one product A = X X^T, L steps of m x m
// products that carry P = Q_{L-1} ... Q_0 along, and one product P X: 3 m^2 n + (4 L - 3) m^3 operations (half of a
// symmetric product's tiles are computed, the others mirrored) against L (3 m^2 n + m^3) step by step.
//
// Precision.  The first steps amplify small singular values by up to a each, and with them every rounding made
// before: iterates rounded to 16 bits lose 4 % (fp16) to 30 % (bf16) of an update that is a few strong directions
// over a noise floor.  Here every operand is a pair of fp16 values hi + lo (22 bits; a power-of-two scale per
// buffer, from a bound on its norm, keeps both in fp16's range) and a product is hi hi + hi lo + lo hi with fp32
// sums on the matrix units: the accuracy of fp32 products at three fp16 passes instead of the sixteen that the
// fp32 matrix instructions take.  Forming A squares the singular values, so a segment of L Gram steps loses the
// directions whose share of A is below its rounding, amplified a^(2L)-fold.  Measured against 64 bits on a few strong
// directions over a noise floor (rank 4 and noise of 0.3 to 0.001, 128 x 128 to 2048 x 8192): five steps at once cost
// 1e-4 to 2e-4 of the result (rank 1: up to 5e-4 from 129 rows on, 1.4e-3 for 17), a part of a bf16 result's rounding
// (1.7e-3) but more than an fp16 result's (2.1e-4).  So bf16 results of more than 128 rows take all five at once, smaller
// ones and fp16 two and three (2e-6 to 4e-5, what fp32 products are off by there; 8e-5 at 2048 x 8192, where those are off
// by 1.3e-4).  For fp32 results the segments are of two and three steps too, or of one for
// matrices that are nearly square (n < 2 m, where the smallest singular values sit near zero) and for those of up to 64
// rows (where the squares saved are cheap): 0.3 to 1.9 times the error of fp32 products on the same inputs (512 x 4608
// without structure 1.4e-6 against 4.3e-6, 128 x 300 of rank 4 and noise of 0.1 3.8e-6 against 2.6e-6); 64 x 288 2.5e-8
// (1.5e-6), worked on in 64 bits.
#include "fc3d_common.h"

#include <cmath>

namespace fc3d {
namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));

typedef float float4v __attribute__((ext_vector_type(4)));
typedef uint32_t uint4v __attribute__((ext_vector_type(4)));
typedef float float16v __attribute__((ext_vector_type(16)));

constexpr int kSlice = 64;            // depth of one staged slice of a product, and the unit that sizes are padded to
constexpr int kMaxItems = 48;         // matrices of one group (their descriptions travel as kernel arguments once)
constexpr int kChunk = 16384;         // elements of one workgroup of the norm pass

// A matrix's buffers, each a plane of hi values and one of lo values: X in two orders (the transpose twice: a segment
// reads one and writes the other), then the m x m matrices of the Gram form.
enum Buffer : uint8_t { BUF_X, BUF_XT0, BUF_XT1, BUF_A, BUF_Q, BUF_R, BUF_P0, BUF_P1, BUF_COUNT };

__host__ __device__ inline int64_t plane_of(int id, int64_t mp, int64_t np) {     // values of one plane of a buffer
    return id < BUF_A ? mp * np : mp * mp;
}
__host__ __device__ inline int64_t before(int id, int64_t mp, int64_t np) {       // values in front of it
    return id < BUF_A ? 2 * id * mp * np : 2 * BUF_A * mp * np + 2 * (id - BUF_A) * mp * mp;
}

struct Matrix {
    const void* g;
    float* mom;                       // NULL: g itself is orthogonalised
    void* out;
    int64_t base;                     // halves from the start of the workspace's planes to its buffers
    int m, n, mp, np;                 // m <= n, and both padded
    float lr;                         // learning rate times the shape's factor
    int part0;                        // its first partial sum of squares
    int split, sums0;                 // workgroups that share the depth of a Gram tile, its first tile of their sums
    int tall, plan;                   // the tensor is n x m; which sequence of products it goes through

    __device__ __forceinline__ void from_lane(int w) {        // this lane's entry becomes lane w's, in all lanes
        static_assert(sizeof(Matrix) % 4 == 0, "copied as words");
        int words[sizeof(Matrix) / 4];
        __builtin_memcpy(words, this, sizeof(Matrix));
#pragma unroll
        for (unsigned i = 0; i < sizeof(Matrix) / 4; ++i) words[i] = __builtin_amdgcn_readlane(words[i], w);
        __builtin_memcpy(this, words, sizeof(Matrix));
    }
};
struct Table {
    int count;
    Matrix e[kMaxItems];
};

// Element types are template arguments or dispatched outside the loops: a branch around every load would make each
// wait for the one before.
template <typename T>
__device__ __forceinline__ float ld(const void* p, size_t i) {
    return (float)static_cast<const T*>(p)[i];
}
template <typename F>
__device__ __forceinline__ void with_type(int type, F&& f) {
    if (type == FC3D_F32) f(float{});
    else if (type == FC3D_BF16) f(__bf16{});
    else f(_Float16{});
}
// four values, at the element's own alignment
typedef float float4a __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t word2a __attribute__((ext_vector_type(2), aligned(2)));
template <typename T>
__device__ __forceinline__ void ld4(const void* p, size_t i, float (&v)[4]) {
    if constexpr (sizeof(T) == 4) {
        const float4a w = *reinterpret_cast<const float4a*>(static_cast<const float*>(p) + i);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = w[j];
    } else {
        const word2a w = *reinterpret_cast<const word2a*>(static_cast<const T*>(p) + i);
        T h[4];
        __builtin_memcpy(h, &w, 8);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = (float)h[j];
    }
}

// Which matrix this workgroup works on: lane l counts the workgroups of matrix l, a scan over the wavefront numbers
// them.  Returns the matrix, and the workgroup's number within it in `block` (the same in all lanes).
__device__ __forceinline__ int find_matrix(int mine, int& block) {
    int sum = mine;
    sum += __builtin_amdgcn_update_dpp(0, sum, 0x111, 0xf, 0xf, true);       // the lane 1, 2, 4, 8 below, in rows of 16
    sum += __builtin_amdgcn_update_dpp(0, sum, 0x112, 0xf, 0xf, true);
    sum += __builtin_amdgcn_update_dpp(0, sum, 0x114, 0xf, 0xf, true);
    sum += __builtin_amdgcn_update_dpp(0, sum, 0x118, 0xf, 0xf, true);
    sum += __builtin_amdgcn_update_dpp(0, sum, 0x142, 0xa, 0xf, false);      // the last lane of the row, of the half below
    sum += __builtin_amdgcn_update_dpp(0, sum, 0x143, 0xc, 0xf, false);
    const int w = __builtin_ctzll(ballot64(sum > block) | (1ull << 63));
    block -= __builtin_amdgcn_readlane(sum - mine, w);
    return w;
}

struct Blend {                        // m' = beta m + (1 - beta) g;  u = (1 - beta) g + beta m' (nesterov) or m'
    float beta, rest;
    int nesterov;
};
__device__ __forceinline__ float blend(const Blend& k, float g, float mom_new) {
    return k.nesterov ? fmaf(k.beta, mom_new, k.rest * g) : mom_new;
}

__device__ __forceinline__ int parts_of(const Matrix& e) { return (int)(((size_t)e.m * e.n + kChunk - 1) / kChunk); }

// Sums of squares of the update per workgroup (64 bits: any fp32 input stays in range), and the momentum's update.
// The first workgroup leaves the table in device memory for the launches that follow: kernel arguments may lie in host
// memory, where a search through them costs microseconds.
template <typename T>
__global__ __launch_bounds__(256) void ns_norm_kernel(Table t, Blend k, double* __restrict__ parts,
                                                      Matrix* __restrict__ table) {
    __shared__ double red[4];
    const int lane = threadIdx.x & 63;
    if (blockIdx.x == 0) {
        const int words = t.count * (int)(sizeof(Matrix) / 4);
        const uint32_t* from = reinterpret_cast<const uint32_t*>(&t.e[0]);
        for (int q = threadIdx.x; q < words; q += 256) reinterpret_cast<uint32_t*>(table)[q] = from[q];
    }
    int block = blockIdx.x;
    const int w = find_matrix(lane < t.count ? parts_of(t.e[lane < t.count ? lane : 0]) : 0, block);
    const Matrix& e = t.e[w];
    const size_t count = (size_t)e.m * e.n;
    const size_t lo = (size_t)block * kChunk;
    const size_t hi = lo + kChunk < count ? lo + kChunk : count;
    double s = 0.0;
    const auto one = [&](size_t j) {
        float u = ld<T>(e.g, j);
        if (e.mom) {
            const float mn = fmaf(k.beta, e.mom[j], k.rest * u);
            e.mom[j] = mn;
            u = blend(k, u, mn);
        }
        s = fma((double)u, (double)u, s);
    };
    const size_t whole = lo + (hi - lo) / 4 * 4;
#pragma unroll 4
    for (size_t j = lo + 4 * threadIdx.x; j < whole; j += 1024) {
        float u[4];
        ld4<T>(e.g, j, u);
        if (e.mom) {
            float m[4];
            ld4<float>(e.mom, j, m);
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                m[q] = fmaf(k.beta, m[q], k.rest * u[q]);
                u[q] = blend(k, u[q], m[q]);
            }
            float4a v;
            __builtin_memcpy(&v, m, 16);
            *reinterpret_cast<float4a*>(e.mom + j) = v;
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) s = fma((double)u[q], (double)u[q], s);
    }
    if (whole + threadIdx.x < hi) one(whole + threadIdx.x);
#pragma unroll
    for (int q = 32; q > 0; q >>= 1) s += __shfl_xor(s, q, 64);
    if (lane == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) parts[e.part0 + block] = (red[0] + red[1]) + (red[2] + red[3]);
}

__device__ __forceinline__ void split8(_Float16* p, size_t plane, const float (&v)[8]) {
    half8 h, l;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        h[j] = (_Float16)v[j];
        l[j] = (_Float16)(v[j] - (float)h[j]);
    }
    *reinterpret_cast<half8*>(p) = h;
    *reinterpret_cast<half8*>(p + plane) = l;
}

// What the products need to know of a matrix's norm.
struct Norm {
    float rest;                       // see ns_prepare_kernel
    int low;                          // the norm of X_0 is at most 2^-low
};
// Where eps is far above the norm, X starts small and its pairs would fall below fp16's range: after `steps` steps, each of
// which multiplies it by 2^gain at most, X is kept times 2^lift.  (Up to 2^96, whose inverse leaves fp32 its precision.)
__device__ __forceinline__ int lift(int low, float gain, int steps) {
    const int e = (int)floorf((float)low - gain * (float)steps);
    return e < 0 ? 0 : e > 96 ? 96 : e;
}

// X and its transpose, scaled by sx 2^lift / (norm + eps), zero beyond the matrix, one 64 x 64 tile per workgroup.
// `exact` (16-bit input taken as it is): one plane that holds the input times a power of two, without rounding; the
// remaining factor in [1, 2) goes to Norm::rest and into the products that read X.
template <typename T>
__global__ __launch_bounds__(256) void ns_prepare_kernel(const Matrix* __restrict__ t, int matrices, Blend k,
                                                         const double* __restrict__ parts, double eps, float sx, int exact,
                                                         _Float16* __restrict__ planes, Norm* __restrict__ norms) {
    __shared__ float tile[64][65];
    __shared__ double red[4];
    const int lane = threadIdx.x & 63;
    int block = blockIdx.x;
    const int w = find_matrix(lane < matrices ? (t[lane].mp / 64) * (t[lane].np / 64) : 0, block);
    const Matrix& e = t[w];
    const int tn = e.np / 64;
    const int i0 = block / tn * 64, j0 = block % tn * 64;
    const int ty = threadIdx.x >> 6;
    float v[16];
    {
        size_t at[16];
        bool in[16];
#pragma unroll
        for (int q = 0; q < 16; ++q) {
            const int fast = lane, slow = q * 4 + ty;        // fast: along the tensor's rows
            const int i = i0 + (e.tall ? fast : slow), j = j0 + (e.tall ? slow : fast);
            in[q] = i < e.m && j < e.n;
            at[q] = !in[q] ? 0 : e.tall ? (size_t)j * e.m + i : (size_t)i * e.n + j;
        }
#pragma unroll
        for (int q = 0; q < 16; ++q) v[q] = ld<T>(e.g, at[q]);
        if (e.mom)
#pragma unroll
            for (int q = 0; q < 16; ++q) v[q] = blend(k, v[q], e.mom[at[q]]);
#pragma unroll
        for (int q = 0; q < 16; ++q)
            if (!in[q]) v[q] = 0.0f;
    }
    const int count = parts_of(e);
    double s = 0.0;
#pragma unroll 4
    for (int q = threadIdx.x; q < count; q += 256) s += parts[e.part0 + q];
#pragma unroll
    for (int q = 32; q > 0; q >>= 1) s += __shfl_xor(s, q, 64);
    if (lane == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    const double norm = sqrt((red[0] + red[1]) + (red[2] + red[3]));
    int above = 0, below = 0;                                // norm + eps and norm, below 2^ these and not below half of it
    frexp(norm + eps, &above);
    frexp(norm, &below);
    const int low = norm > 0.0 && norm < 1e300 && above - 1 > below ? above - 1 - below : 0;
    const double factor = ldexp((double)sx / (norm + eps), lift(low, 0.0f, 0));
    int shift = 0;
    float rest = 1.0f;
    if (exact) {
        rest = 2.0f * (float)frexp(factor, &shift);          // factor = rest * 2^(shift - 1), rest in [1, 2)
        shift -= 1;
        if (!(factor < 1e300) || factor == 0.0) {            // a zero matrix with eps 0, an infinity or a NaN: 0 * inf below
            shift = 0;
            rest = (float)factor;
        }
    }
    if (block == 0 && threadIdx.x == 0) norms[w] = Norm{rest, low};
#pragma unroll
    for (int q = 0; q < 16; ++q) {
        const int fast = lane, slow = q * 4 + ty, r = e.tall ? fast : slow, c = e.tall ? slow : fast;
        const bool in = i0 + r < e.m && j0 + c < e.n;
        tile[r][c] = !in ? 0.0f : exact ? ldexpf(v[q], shift) : (float)((double)v[q] * factor);
    }
    __syncthreads();
    const size_t plane = plane_of(BUF_X, e.mp, e.np);
    _Float16* x = planes + e.base;
    _Float16* xt = x + before(BUF_XT0, e.mp, e.np);
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        const int id = threadIdx.x + 256 * q, r = id >> 3, c = (id & 7) * 8;
        float u[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) u[j] = tile[r][c + j];
        split8(x + (size_t)(i0 + r) * e.np + j0 + c, plane, u);
#pragma unroll
        for (int j = 0; j < 8; ++j) u[j] = tile[c + j][r];
        split8(xt + (size_t)(j0 + r) * e.mp + i0 + c, plane, u);
    }
}

__device__ __forceinline__ uint32_t pair_word(float v) {
    const _Float16 hi = (_Float16)v, lo = (_Float16)(v - (float)hi);
    return (uint32_t)__builtin_bit_cast(uint16_t, hi) | (uint32_t)__builtin_bit_cast(uint16_t, lo) << 16;
}

// ---- products -----------------------------------------------------------------------------------------------
// D[i][j] = sum_k S1[i][k] S2[j][k]: both operands run along the depth in memory (a symmetric matrix is its own
// transpose, and X is kept in both orders), so one kernel serves every product:
//   GRAM   A = X X^T           POLY  Q = a I + b A + c A A        MUL  R = A Q, A = R Q, P = P Q  (symmetric: the upper
//   APPLY  X = P X                                                     triangle's tiles, mirrored)
// A launch does the next product of every matrix, whatever its kind: matrices of different shapes go through
// different sequences (plans) side by side.
enum Kind : uint8_t { NONE, GRAM, POLY, MUL, APPLY };
struct Op {
    uint8_t kind, src1, src2, dst;
    float alpha;                      // sum -> stored value (scales of the operands and of the result)
    uint8_t exact, last;              // the first segment of an input taken as it is; APPLY: to the tensors
    uint8_t from, to;                 // GRAM, APPLY: steps that X has behind it, and that the result has
};
constexpr int kPlans = 2;
struct Launch {
    Op op[kPlans][2];                 // up to two products of a matrix that do not need each other
    float a, b;                       // POLY: Q = a I + b A + c A A, in units of the stored result
    float gain;                       // log2 of the most that a step multiplies X by
    int out_type, step;               // step: weights := decay * weights - lr * result
    float decay;
    int matrices;
    const Matrix* table;
    _Float16* planes;
    const Norm* norms;
    float* sums;                      // Gram tiles of shared depth: [tile][share][TILE * TILE]
};

// The factor of a product's sums that depends on its matrix: X is kept lifted, and may lack Norm::rest
__device__ __forceinline__ float alpha_of(const Op& o, const Norm& n, float gain) {
    if (o.kind != GRAM && o.kind != APPLY) return o.alpha;
    const float rest = o.exact ? n.rest : 1.0f;
    const int up = lift(n.low, gain, o.from);
    if (o.kind == GRAM) return ldexpf(o.alpha * (rest * rest), -2 * up);
    return ldexpf(o.alpha * rest, (o.last ? 0 : lift(n.low, gain, o.to)) - up);
}

__device__ __forceinline__ _Float16* buffer(const Matrix& e, _Float16* planes, int id, int& ld, size_t& plane) {
    ld = id == BUF_X ? e.np : e.mp;
    plane = (size_t)plane_of(id, e.mp, e.np);
    return planes + e.base + before(id, e.mp, e.np);
}

__host__ __device__ inline int tiles_of(int kind, int mp, int np, int split, int tile) {
    const int tm = (mp + tile - 1) / tile, tn = (np + tile - 1) / tile;
    return kind == NONE ? 0 : kind == APPLY ? tm * tn : tm * (tm + 1) / 2 * (kind == GRAM ? split : 1);
}

// Workgroups next to each other, which run at the same time behind one L2, take tiles in strips of kStrip: 4 x 8 tiles
// read 12 different operand slices where a row of 32 reads 33.
constexpr int kStrip = 8;

__device__ __forceinline__ int column_of(int block) {         // the column of a triangle numbered column by column
    int tj = (int)((sqrtf(8.0f * (float)block + 1.0f) - 1.0f) * 0.5f);
    while ((long)tj * (tj + 1) / 2 > block) --tj;
    while ((long)(tj + 1) * (tj + 2) / 2 <= block) ++tj;
    return tj;
}
// The upper triangle of t x t tiles: strips of kStrip columns, each by rows, its own triangle last
__device__ __forceinline__ void upper_tile(int block, int t, int& ti, int& tj) {
    const int left = column_of(block) / kStrip * kStrip, wide = t - left < kStrip ? t - left : kStrip;
    int l = block - (int)((long)left * (left + 1) / 2);
    if (l < left * wide) {
        ti = l / wide;
        tj = left + l % wide;
    } else {
        l -= left * wide;
        const int c = column_of(l);
        ti = left + l - c * (c + 1) / 2;
        tj = left + c;
    }
}

template <int T>
struct Turn {
    static constexpr int value = T;
};

// A workgroup computes a TILE x TILE tile.  A wavefront holds BLK x BLK of the 32 x 32 matrix instruction's sums, so that
// an operand read from LDS feeds 3 BLK of them: TILE 64 and 96: every wavefront the whole tile, its part of the depth;
// TILE 128: two wavefronts per quadrant.  Their sums meet at the end.  Stages are fetched ahead into registers (what
// another compute unit has just written comes from behind the L2: most of a microsecond) and go through two LDS
// buffers, one barrier per stage.  P1, P2: planes of the operands that count (1: the lo plane is zero).
// 2048 rows and depth, one symmetric product, 37 us: about 5 us pass outside the workgroups, 1.6 until the first stage,
// 25.7 in the stages, 4.5 for the result.  The stages alone take 15.7 us with nothing but the matrix instructions,
// 16.6 with their reads from LDS, and the way from memory into LDS 20.6 us (400 MB, 19 TB/s out of the L2s): that path
// bounds it, and the two overlap for the larger part.
template <int TILE, int WAVES, int P1, int P2>
__global__ __launch_bounds__(WAVES * 64, TILE == 64 && WAVES == 4 ? 2 : 1) void ns_product_kernel(Launch a) {
    constexpr bool QUADS = TILE == 128;
    constexpr int THREADS = WAVES * 64, BLK = QUADS ? 2 : TILE / 32;
    constexpr int NP = P1 + P2;
    constexpr int DEPTH = kSlice, ROW = DEPTH / 8;           // of a stage, in values and in 16-byte pieces
    constexpr int AHEAD = QUADS ? (NP == 4 ? 1 : 2) : NP == 2 ? 3 : 2;      // stages in flight in registers
    static_assert(QUADS || WAVES * 16 == DEPTH, "every wavefront has 16 values of a stage's depth");
    constexpr int PIECES = TILE * ROW / THREADS;             // pieces of a stage per lane and plane
    constexpr int ROWS = THREADS / ROW;                      // rows that the workgroup's lanes cover at once
    constexpr int SHARES = QUADS ? 2 : WAVES, LD = TILE + 8, LD2 = TILE + 4;
    constexpr int STAGE = NP * TILE * ROW;                   // pieces of one stage
    constexpr int SWAP = TILE * TILE * 4 * (SHARES - 1), RESULT = TILE * (LD + LD2) * 4;    // bytes
    constexpr int MOST = SWAP > RESULT ? SWAP : RESULT, BYTES = 2 * STAGE * 16 > MOST ? 2 * STAGE * 16 : MOST;
    __shared__ __attribute__((aligned(16))) char shared[BYTES];
    half8* lds = reinterpret_cast<half8*>(shared);
    float* out = reinterpret_cast<float*>(shared);

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    int block = (int)block_x();
    // every lane reads one matrix of the table: what the workgroup needs of its own comes from that lane's registers
    Matrix e = a.table[lane < a.matrices ? lane : 0];
    const Op o00 = a.op[0][0], o01 = a.op[0][1], o10 = a.op[1][0], o11 = a.op[1][1];
    const int k0 = e.plan ? o10.kind : o00.kind, k1 = e.plan ? o11.kind : o01.kind;
    int n0 = tiles_of(k0, e.mp, e.np, e.split, TILE);
    const int w = find_matrix(lane < a.matrices ? n0 + tiles_of(k1, e.mp, e.np, e.split, TILE) : 0, block);
    e.from_lane(w);
    const Norm norm = a.norms[w];                             // (on its way while the stages run)
    n0 = __builtin_amdgcn_readlane(n0, w);
    Op o = e.plan ? o10 : o00;
    if (block >= n0) {
        block -= n0;
        o = e.plan ? o11 : o01;
    }
    int share = 0;
    if (o.kind == GRAM && e.split > 1) {
        const int tiles = tiles_of(MUL, e.mp, 0, 1, TILE);
        share = block / tiles;
        block -= share * tiles;
    }
    int ti, tj;
    if (o.kind == APPLY) {
        const int tm = (e.mp + TILE - 1) / TILE, tn = (e.np + TILE - 1) / TILE, strip = block / (kStrip * tn);
        const int wide = tm - strip * kStrip < kStrip ? tm - strip * kStrip : kStrip;
        const int l = block - strip * kStrip * tn;
        ti = strip * kStrip + l % wide;
        tj = l / wide;
    } else {
        upper_tile(block, (e.mp + TILE - 1) / TILE, ti, tj);
    }
    int ld1, ld2;
    size_t pl1, pl2;
    const _Float16* s1 = buffer(e, a.planes, o.src1, ld1, pl1) + (size_t)ti * TILE * ld1;
    const _Float16* s2 = buffer(e, a.planes, o.src2, ld2, pl2) + (size_t)tj * TILE * ld2;
    const int rows1 = e.mp - ti * TILE, rows2 = (o.kind == APPLY ? e.np : e.mp) - tj * TILE;       // from this tile on
    int slices = (o.kind == GRAM ? e.np : e.mp) / kSlice;
    if (o.kind == GRAM && e.split > 1) {
        const int each = (slices + e.split - 1) / e.split, from = share * each;
        slices = from + each < slices ? each : slices - from;
        s1 += (size_t)from * kSlice;
        s2 += (size_t)from * kSlice;
    }

    // A row's pieces are stored in an order of its own (piece ^ key), so that 16 rows read at one depth, 256 bytes, lie in
    // different banks (a row is 128 bytes long).
    const auto key = [](int row) { return (row >> 1) & 7; };
    const int row0 = tid / ROW, piece0 = tid % ROW;
    const int stages = slices;
    unsigned at1[PIECES], at2[PIECES];                        // bytes from the tile's first row; rows behind the matrix: its last
#pragma unroll
    for (int q = 0; q < PIECES; ++q) {
        const int row = row0 + ROWS * q;
        at1[q] = ((unsigned)(row < rows1 ? row : rows1 - 1) * (unsigned)ld1 + piece0 * 8) * 2u;
        at2[q] = ((unsigned)(row < rows2 ? row : rows2 - 1) * (unsigned)ld2 + piece0 * 8) * 2u;
    }
    half8 next[AHEAD][NP * PIECES];
    const auto fetch = [&](int s, half8 (&to)[NP * PIECES]) {
#pragma unroll
        for (int p = 0; p < NP; ++p) {
            const char* src = reinterpret_cast<const char*>((p < P1 ? s1 + p * pl1 : s2 + (p - P1) * pl2) + (size_t)s * DEPTH);
#pragma unroll
            for (int q = 0; q < PIECES; ++q)
                to[p * PIECES + q] = *reinterpret_cast<const half8*>(src + (p < P1 ? at1[q] : at2[q]));
        }
    };
    const auto stage = [&](int s, const half8 (&from)[NP * PIECES]) {
#pragma unroll
        for (int p = 0; p < NP; ++p)
#pragma unroll
            for (int q = 0; q < PIECES; ++q) {
                const int row = row0 + ROWS * q;
                lds[(s & 1) * STAGE + (p * TILE + row) * ROW + (piece0 ^ key(row))] = from[p * PIECES + q];
            }
    };
    const int quad = wave >> 1;
    const int bi = QUADS ? (quad >> 1) * 64 : 0, bj = QUADS ? (quad & 1) * 64 : 0;
    const int own = QUADS ? (wave & 1) * 2 : wave;            // this wavefront's first 16 values of a stage's depth, in 16s
    // The matrix units' sums lose up to a unit of the running sum's last place per instruction: that the wavefronts
    // share the depth keeps the chains short (a depth of 4608: 216 instructions, fewer where workgroups share it
    // too; one wavefront's 864 would double the error of the result).
    float16v acc[BLK][BLK] = {};
    struct Part {                                             // both operands at 16 values of the depth
        half8 f1[BLK][P1], f2[BLK][P2];
    };
    const auto load = [&](int s, int kk, Part& f) {
        const int piece = kk * 2 + (lane >> 5);
#pragma unroll
        for (int h = 0; h < BLK; ++h) {
            const int r1 = bi + h * 32 + (lane & 31), r2 = bj + h * 32 + (lane & 31);
#pragma unroll
            for (int p = 0; p < P1; ++p) f.f1[h][p] = lds[(s & 1) * STAGE + (p * TILE + r1) * ROW + (piece ^ key(r1))];
#pragma unroll
            for (int p = 0; p < P2; ++p) f.f2[h][p] = lds[(s & 1) * STAGE + ((P1 + p) * TILE + r2) * ROW + (piece ^ key(r2))];
        }
    };
    const auto multiply = [&](const Part& f) {
#pragma unroll
        for (int pass = 0; pass < 3; ++pass) {                // lo hi, hi lo, hi hi
            const int p1 = pass == 0 ? 1 : 0, p2 = pass == 1 ? 1 : 0;
            if (p1 >= P1 || p2 >= P2) continue;
#pragma unroll
            for (int q = 0; q < BLK * BLK; ++q)
                acc[q / BLK][q % BLK] =
                    __builtin_amdgcn_mfma_f32_32x32x16_f16(f.f1[q / BLK][p1], f.f2[q % BLK][p2], acc[q / BLK][q % BLK], 0, 0, 0);
        }
    };
    // Stage s: behind the barrier that makes it visible, its operands are read while the matrix units still work on what
    // was read before; stage s + 1 goes from registers to the other LDS buffer, s + 1 + AHEAD into the registers.
    // `whole`: no branch around the loads, so that the compiler knows how many are in flight and waits for the oldest
    // alone.
    const auto step = [&](int s, half8 (&regs)[NP * PIECES], Part& x, Part& y, bool first, bool whole) {
        __syncthreads();
        load(s, own, x);
        if (!first) multiply(y);
        if constexpr (QUADS) load(s, own + 1, y);
        if (whole || s + 1 < stages) stage(s + 1, regs);
        if (whole || s + 1 + AHEAD < stages) fetch(s + 1 + AHEAD, regs);
        if constexpr (QUADS) multiply(x);
        // LDS and memory instructions one by one between the matrix instructions: issued in a row they would fill the LDS
        // queue, and the matrix units would wait for it
        if (whole && P1 == 2 && P2 == 2) {
            constexpr int READS = 4 * BLK, LOADS = NP * PIECES, EACH = QUADS || BLK == 3 ? 1 : 2;
#pragma unroll
            for (int half = 0; half < (QUADS ? 2 : 1); ++half) {
#pragma unroll
                for (int q = 0; q < READS; ++q) {
                    __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);        // LDS read
                    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);        // matrix
                }
#pragma unroll
                for (int q = 0; q < LOADS / EACH / (QUADS ? 2 : 1); ++q) {
                    __builtin_amdgcn_sched_group_barrier(0x200, EACH, 0);     // LDS write
                    __builtin_amdgcn_sched_group_barrier(0x020, EACH, 0);     // load
                    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                }
            }
        }
        __builtin_amdgcn_sched_barrier(0);
    };
    // Even and odd stages' operands, or, in quadrants, those of a stage's two halves.  Registers, LDS buffers and operands
    // come round every GROUP stages; the last ones, which fetch no more, are written out behind the loop.
    Part part[2];
    constexpr int GROUP = AHEAD == 3 ? 6 : 2;
    const auto turn = [&](int s, auto t, bool first, bool whole) {       // stage s, the t-th of a group behind the first stage
        constexpr int T = decltype(t)::value;
        step(s, next[(T + 1) % AHEAD], part[QUADS ? 0 : T & 1], part[QUADS ? 1 : (T + 1) & 1], first, whole);
    };
#pragma unroll
    for (int q = 0; q < AHEAD; ++q) fetch(q < stages ? q : stages - 1, next[q]);
    stage(0, next[0]);
    fetch(AHEAD < stages ? AHEAD : stages - 1, next[0]);
    int s = 1;
    if (s + GROUP + AHEAD < stages) {                         // the loop is entered with all loads in flight, on no other path
        turn(0, Turn<0>{}, true, true);
        for (; s + GROUP + AHEAD < stages; s += GROUP) {
            turn(s, Turn<1>{}, false, true);
            turn(s + 1, Turn<2>{}, false, true);
            if constexpr (GROUP == 6) {
                turn(s + 2, Turn<3>{}, false, true);
                turn(s + 3, Turn<4>{}, false, true);
                turn(s + 4, Turn<5>{}, false, true);
                turn(s + 5, Turn<6>{}, false, true);
            }
        }
    } else {
        turn(0, Turn<0>{}, true, false);
    }
    const int rest = stages - s;                              // at most GROUP + AHEAD
    const auto tail = [&](auto t) {
        constexpr int T = decltype(t)::value;
        if (T <= GROUP + AHEAD && T <= rest) turn(s + T - 1, t, false, false);
    };
    tail(Turn<1>{});
    tail(Turn<2>{});
    tail(Turn<3>{});
    tail(Turn<4>{});
    if constexpr (GROUP == 6) {
        tail(Turn<5>{});
        tail(Turn<6>{});
        tail(Turn<7>{});
        tail(Turn<8>{});
        tail(Turn<9>{});
    }
    // A lane holds column (lane & 31) of a 32 x 32 block, rows 8 (r / 4) + 4 (lane / 32) + r % 4
    constexpr int OWN = 4 / SHARES;                           // of a block's quads of rows
    const int half = QUADS ? wave & 1 : wave;
    const int i0 = ti * TILE, j0 = tj * TILE;
    const auto row_of = [&](int q, int k) { return bi + q / BLK * 32 + 8 * (half * OWN + k) + 4 * (lane >> 5); };
    const auto col_of = [&](int q) { return bj + q % BLK * 32 + (lane & 31); };
    constexpr int G = TILE / 8, MOVES = (TILE * G + THREADS - 1) / THREADS;       // a tile in pieces of eight values
    half8 hi[MOVES], lo[MOVES];                               // POLY: A at the tile, on its way while the last products run
    if (o.kind == POLY) {
        int lda;
        size_t pa;
        const _Float16* A = buffer(e, a.planes, o.src1, lda, pa);
#pragma unroll
        for (int q = 0; q < MOVES; ++q) {
            const int id = tid + THREADS * q, r = id / G, c = id % G * 8;
            const size_t at = r < rows1 && c < rows2 ? (size_t)(i0 + r) * lda + j0 + c : 0;
            hi[q] = *reinterpret_cast<const half8*>(A + at);
            lo[q] = *reinterpret_cast<const half8*>(A + pa + at);
        }
    }
    if (QUADS || (rest & 1)) multiply(part[1]);
    else multiply(part[0]);

    // ---- the result.  The wavefronts that share a block's depth exchange their sums as they hold them, 16 bytes at a
    // time, and each is left with the whole sum of its rows.
    const float alpha = alpha_of(o, norm, a.gain);
    float4v sum[BLK * BLK][OWN];
    float4v* swap = reinterpret_cast<float4v*>(shared);
    const auto slot = [&](int to, int from, int q, int k) {   // of the share `from` (without the receiver's own) for wavefront `to`
        return ((to * (SHARES - 1) + from) * (BLK * BLK * OWN) + q * OWN + k) * 64 + lane;
    };
    __syncthreads();
#pragma unroll
    for (int d = 0; d < SHARES; ++d)
#pragma unroll
        for (int q = 0; q < BLK * BLK; ++q)
#pragma unroll
            for (int k = 0; k < OWN; ++k) {
                const int r = 4 * (d * OWN + k);
                const float16v& c = acc[q / BLK][q % BLK];
                const float4v v = {c[r], c[r + 1], c[r + 2], c[r + 3]};
                if (d == half) sum[q][k] = v;
                else swap[slot(QUADS ? (wave & ~1) + d : d, half < d ? half : half - 1, q, k)] = v;
            }
    __syncthreads();
#pragma unroll
    for (int f = 0; f < SHARES - 1; ++f)
#pragma unroll
        for (int q = 0; q < BLK * BLK; ++q)
#pragma unroll
            for (int k = 0; k < OWN; ++k) sum[q][k] += swap[slot(wave, f, q, k)];
    if (o.kind == GRAM && e.split > 1) {
        float* to = a.sums + ((size_t)e.sums0 + (size_t)block * e.split + share) * TILE * TILE;
#pragma unroll
        for (int q = 0; q < BLK * BLK; ++q)
#pragma unroll
            for (int k = 0; k < OWN; ++k)
#pragma unroll
                for (int r = 0; r < 4; ++r) to[(row_of(q, k) + r) * TILE + col_of(q)] = sum[q][k][r];
        return;
    }
#pragma unroll
    for (int q = 0; q < BLK * BLK; ++q)
#pragma unroll
        for (int k = 0; k < OWN; ++k) sum[q][k] *= alpha;
    if (o.kind == APPLY && o.last) {
        with_type(a.out_type, [&](auto zero) {
            typedef decltype(zero) T;
            T* to = static_cast<T*>(e.out);
            // A step reads the weights: all of a lane's first, without a branch of their own (behind the matrix its last
            // row and column), which would wait for each.
            if (!e.tall) {                                    // along the tensor's rows as the lanes hold them
                T old[BLK * BLK][OWN][4];
                if (a.step)
#pragma unroll
                    for (int q = 0; q < BLK * BLK; ++q)
#pragma unroll
                        for (int k = 0; k < OWN; ++k)
#pragma unroll
                            for (int r = 0; r < 4; ++r) {
                                const int i = i0 + row_of(q, k) + r, j = j0 + col_of(q);
                                old[q][k][r] = to[(size_t)(i < e.m ? i : e.m - 1) * e.n + (j < e.n ? j : e.n - 1)];
                            }
#pragma unroll
                for (int q = 0; q < BLK * BLK; ++q)
#pragma unroll
                    for (int k = 0; k < OWN; ++k)
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const int i = i0 + row_of(q, k) + r, j = j0 + col_of(q);
                            float v = sum[q][k][r];
                            if (a.step) v = fmaf(a.decay, (float)old[q][k][r], -e.lr * v);
                            if (i < e.m && j < e.n) to[(size_t)i * e.n + j] = (T)v;
                        }
                return;
            }
            __syncthreads();
#pragma unroll
            for (int q = 0; q < BLK * BLK; ++q)
#pragma unroll
                for (int k = 0; k < OWN; ++k) *reinterpret_cast<float4v*>(out + col_of(q) * LD2 + row_of(q, k)) = sum[q][k];
            __syncthreads();
            constexpr int CHUNK = BLK == 3 ? 9 : 8;            // values of a lane in flight
            for (int from = tid; from < TILE * TILE; from += CHUNK * THREADS) {
                T old[CHUNK];
                if (a.step)
#pragma unroll
                    for (int c = 0; c < CHUNK; ++c) {
                        const int id = from + c * THREADS, i = i0 + id % TILE, j = j0 + id / TILE;
                        old[c] = to[(size_t)(j < e.n ? j : e.n - 1) * e.m + (i < e.m ? i : e.m - 1)];
                    }
#pragma unroll
                for (int c = 0; c < CHUNK; ++c) {
                    const int id = from + c * THREADS, i = i0 + id % TILE, j = j0 + id / TILE;
                    float v = out[(id / TILE) * LD2 + id % TILE];
                    if (a.step) v = fmaf(a.decay, (float)old[c], -e.lr * v);
                    if (i < e.m && j < e.n) to[(size_t)j * e.m + i] = (T)v;
                }
            }
        });
        return;
    }
    // To the buffers: the tile, and its mirror image (or, of X, the transpose), from LDS in whole rows, eight values at a
    // time.  A tile on the diagonal holds every pair twice, its cross terms summed in two orders: the upper one counts.
    const bool diagonal = o.kind != APPLY && ti == tj;
    uint32_t* pairs = reinterpret_cast<uint32_t*>(shared);    // hi and lo in one word
    uint32_t* mirror = pairs + TILE * LD;
    __syncthreads();
    if (o.kind == POLY) {                                     // A through LDS, into the lanes that hold the sums
        float* A = reinterpret_cast<float*>(shared);
#pragma unroll
        for (int q = 0; q < MOVES; ++q) {
            const int id = tid + THREADS * q, r = id / G, c = id % G * 8;
            if (r >= TILE) break;
            float4v x, y;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                x[j] = (float)hi[q][j] + (float)lo[q][j];
                y[j] = (float)hi[q][4 + j] + (float)lo[q][4 + j];
            }
            *reinterpret_cast<float4v*>(A + r * LD + c) = x;
            *reinterpret_cast<float4v*>(A + r * LD + c + 4) = y;
        }
        __syncthreads();
#pragma unroll
        for (int q = 0; q < BLK * BLK; ++q)
#pragma unroll
            for (int k = 0; k < OWN; ++k)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int i = row_of(q, k) + r, j = col_of(q);
                    sum[q][k][r] = fmaf(a.b, A[i * LD + j], sum[q][k][r]);
                    if (i0 + i == j0 + j && i0 + i < e.m) sum[q][k][r] += a.a;
                }
        __syncthreads();
    }
    const auto words_of = [&](int q, int k) {
        return uint4v{pair_word(sum[q][k][0]), pair_word(sum[q][k][1]), pair_word(sum[q][k][2]), pair_word(sum[q][k][3])};
    };
    if (!diagonal) {
#pragma unroll
        for (int q = 0; q < BLK * BLK; ++q)
#pragma unroll
            for (int k = 0; k < OWN; ++k) {
                const uint4v word = words_of(q, k);
                *reinterpret_cast<uint4v*>(mirror + col_of(q) * LD2 + row_of(q, k)) = word;
#pragma unroll
                for (int r = 0; r < 4; ++r) pairs[(row_of(q, k) + r) * LD + col_of(q)] = word[r];
            }
    } else {
#pragma unroll
        for (int q = 0; q < BLK * BLK; ++q)
#pragma unroll
            for (int k = 0; k < OWN; ++k) {
                const uint4v word = words_of(q, k);
                const int i = row_of(q, k), j = col_of(q);
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (i + r <= j) {
                        pairs[(i + r) * LD + j] = word[r];
                        pairs[j * LD + i + r] = word[r];
                    }
            }
    }
    __syncthreads();
    for (int side = 0; side < (diagonal ? 1 : 2); ++side) {
        int ld;
        size_t plane;
        _Float16* d = buffer(e, a.planes, o.kind == APPLY && side == 0 ? (int)BUF_X : o.dst, ld, plane);
        d += (size_t)(side ? j0 : i0) * ld + (side ? i0 : j0);
        const uint32_t* from = side ? mirror : pairs;
        const int rows = side ? rows2 : rows1, cols = side ? rows1 : rows2;
#pragma unroll
        for (int q = 0; q < MOVES; ++q) {
            const int id = tid + THREADS * q, r = id / G, c = id % G * 8;
            if (r >= TILE || r >= rows || c >= cols) continue;
            const uint32_t* at = from + r * (side ? LD2 : LD) + c;
            const uint4v x = *reinterpret_cast<const uint4v*>(at), y = *reinterpret_cast<const uint4v*>(at + 4);
            uint4v h, l;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                h[j] = __builtin_amdgcn_perm(x[2 * j + 1], x[2 * j], 0x05040100u);
                h[2 + j] = __builtin_amdgcn_perm(y[2 * j + 1], y[2 * j], 0x05040100u);
                l[j] = __builtin_amdgcn_perm(x[2 * j + 1], x[2 * j], 0x07060302u);
                l[2 + j] = __builtin_amdgcn_perm(y[2 * j + 1], y[2 * j], 0x07060302u);
            }
            _Float16* to = d + (size_t)r * ld + c;
            *reinterpret_cast<uint4v*>(to) = h;
            *reinterpret_cast<uint4v*>(to + plane) = l;
        }
    }
}

// The shares of the Gram tiles' depth, added in order, to A (one TILE x TILE tile per workgroup, upper triangle)
template <int TILE>
__global__ __launch_bounds__(256) void ns_gram_sum_kernel(Launch a) {
    constexpr int LD = TILE + 1;
    __shared__ float out[TILE * LD];
    const int tid = threadIdx.x, lane = tid & 63;
    int block = blockIdx.x;
    int mine = 0;
    if (lane < a.matrices && a.op[a.table[lane].plan][0].kind == GRAM && a.table[lane].split > 1)
        mine = tiles_of(MUL, a.table[lane].mp, 0, 1, TILE);
    const int w = find_matrix(mine, block);
    const Matrix& e = a.table[w];
    const Op& o = a.op[e.plan][0];
    int ti, tj;
    upper_tile(block, (e.mp + TILE - 1) / TILE, ti, tj);
    const float4* from = reinterpret_cast<const float4*>(a.sums + ((size_t)e.sums0 + (size_t)block * e.split) * TILE * TILE);
    const float alpha = alpha_of(o, a.norms[w], a.gain);
    constexpr int QUARTS = TILE * TILE / 4, EACH = QUARTS / 256 % 4 == 0 ? 4 : 3;
    static_assert(QUARTS % (256 * EACH) == 0, "loads in flight per lane");
    for (int g = 0; g < QUARTS / 256; g += EACH) {
        float4 v[EACH];
#pragma unroll
        for (int q = 0; q < EACH; ++q) v[q] = from[tid + 256 * (g + q)];
#pragma unroll 4
        for (int h = 1; h < e.split; ++h)
#pragma unroll
            for (int q = 0; q < EACH; ++q) {
                const float4 u = from[(size_t)h * QUARTS + tid + 256 * (g + q)];
                v[q].x += u.x;
                v[q].y += u.y;
                v[q].z += u.z;
                v[q].w += u.w;
            }
#pragma unroll
        for (int q = 0; q < EACH; ++q) {
            const int id = 4 * (tid + 256 * (g + q)), at = id / TILE * LD + id % TILE;
            out[at] = v[q].x * alpha;
            out[at + 1] = v[q].y * alpha;
            out[at + 2] = v[q].z * alpha;
            out[at + 3] = v[q].w * alpha;
        }
    }
    __syncthreads();
    int ld;
    size_t plane;
    _Float16* d = buffer(e, a.planes, o.dst, ld, plane);
#pragma unroll
    for (int side = 0; side < 2; ++side) {
        if (side == 1 && ti == tj) break;
        const int i0 = (side ? tj : ti) * TILE, j0 = (side ? ti : tj) * TILE;
#pragma unroll 2
        for (int id = tid; id < TILE * TILE / 8; id += 256) {
            const int r = id / (TILE / 8), c = id % (TILE / 8) * 8;
            if (i0 + r >= e.mp || j0 + c >= e.mp) continue;
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const bool other = side || (ti == tj && r > c + j);
                v[j] = other ? out[(c + j) * LD + r] : out[r * LD + c + j];
            }
            split8(d + (size_t)(i0 + r) * ld + j0 + c, plane, v);
        }
    }
}

// ---- matrices of up to 64 rows, in three launches -----------------------------------------------------------
// A list of small matrices is bound by launches, not by products.  There the Gram form runs in 64 bits, all steps in one
// segment (its rounding is 1e-16), one workgroup per matrix with everything in LDS.  The norm is the trace of A; X is only
// read as the tensor holds it, by the first launch and the last.  64 x 288: 7 + 49 + 8 us, 64 us per call, against 109 us
// for the general path's 17 launches.  The chain of 17 products on one compute unit is the rest: 768 fp64 matrix
// instructions of 64 cycles on the busiest SIMD, 20 us, and the operands' way through LDS, which they wait for at the start
// of each; more units per matrix would pay a launch or a wait for each other after every product.
typedef double double4v __attribute__((ext_vector_type(4)));

constexpr int kSmall = 64;            // rows
constexpr int kSmallLd = 68;          // doubles from row to row in LDS
constexpr int kPairs = 10;            // 16 x 16 tiles on and above the diagonal of 64 x 64
constexpr int kGramValues = kPairs * 256;

// lane l of the fp64 instruction: operands row l % 16, depth l / 16; results column l % 16, rows 4 r + l / 16
__device__ __forceinline__ void pair_of(int p, int& ti, int& tj) {         // column by column
    tj = p < 1 ? 0 : p < 3 ? 1 : p < 6 ? 2 : 3;
    ti = p - tj * (tj + 1) / 2;
}

// N values of the update, at rows i(q) and columns j(q) of X (0 beyond it); `store`: the momentum moves on, which each
// value does once.
template <typename T, int N, typename I, typename J>
__device__ __forceinline__ void small_values(const Matrix& e, const Blend& k, bool store, I&& row, J&& col, double (&x)[N]) {
    float g[N], m[N];
    size_t at[N];
    bool in[N];
#pragma unroll
    for (int q = 0; q < N; ++q) {
        const int i = row(q), j = col(q);
        in[q] = i < e.m && j < e.n;
        at[q] = !in[q] ? 0 : e.tall ? (size_t)j * e.m + i : (size_t)i * e.n + j;
    }
#pragma unroll
    for (int q = 0; q < N; ++q) g[q] = ld<T>(e.g, at[q]);
    if (e.mom) {
#pragma unroll
        for (int q = 0; q < N; ++q) m[q] = e.mom[at[q]];
#pragma unroll
        for (int q = 0; q < N; ++q) {
            if (store) {
                m[q] = fmaf(k.beta, m[q], k.rest * g[q]);
                if (in[q]) e.mom[at[q]] = m[q];
            }
            g[q] = blend(k, g[q], m[q]);
        }
    }
#pragma unroll
    for (int q = 0; q < N; ++q) x[q] = in[q] ? (double)g[q] : 0.0;
}

// Sums of the Gram matrix over a chunk of columns (Matrix::np of them) per workgroup, in the instruction's own order
template <typename T>
__global__ __launch_bounds__(256) void ns_small_gram_kernel(Table t, Blend k, Matrix* __restrict__ table,
                                                            double* __restrict__ gram) {
    __shared__ double red[3][kGramValues];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    if (blockIdx.x == 0) {
        const int words = t.count * (int)(sizeof(Matrix) / 4);
        const uint32_t* from = reinterpret_cast<const uint32_t*>(&t.e[0]);
        for (int q = tid; q < words; q += 256) reinterpret_cast<uint32_t*>(table)[q] = from[q];
    }
    int block = blockIdx.x;
    const int w = find_matrix(lane < t.count ? t.e[lane < t.count ? lane : 0].split : 0, block);
    const Matrix& e = t.e[w];
    const int tiles = (e.m + 15) / 16;
    const int lo = block * e.np, hi = lo + e.np < e.n ? lo + e.np : e.n;
    double4v acc[kPairs] = {};
    // sixteen columns at a time per wavefront: a lane holds four neighbouring ones of its row, the instruction takes
    // them in any order as long as both operands keep it
    for (int c = lo + wave * 16; c < hi; c += 64) {
        double x[16];                                         // [tile][column]
        small_values<T>(e, k, true, [&](int q) { return 16 * (q >> 2) + (lane & 15); },
                        [&](int q) { return c + 4 * (lane >> 4) + (q & 3); }, x);
#pragma unroll
        for (int p = 0; p < kPairs; ++p) {
            int ti, tj;
            pair_of(p, ti, tj);
            if (tj >= tiles) break;
#pragma unroll
            for (int q = 0; q < 4; ++q) acc[p] = __builtin_amdgcn_mfma_f64_16x16x4f64(x[ti * 4 + q], x[tj * 4 + q], acc[p], 0, 0, 0);
        }
    }
    if (wave > 0)
#pragma unroll
        for (int p = 0; p < kPairs; ++p)
#pragma unroll
            for (int r = 0; r < 4; ++r) red[wave - 1][p * 256 + r * 64 + lane] = acc[p][r];
    __syncthreads();
    if (wave == 0) {
        double* to = gram + ((size_t)e.sums0 + block) * kGramValues;
#pragma unroll
        for (int p = 0; p < kPairs; ++p)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int at = p * 256 + r * 64 + lane;
                to[at] = ((acc[p][r] + red[0][at]) + red[1][at]) + red[2][at];
            }
    }
}

// One workgroup per matrix: A / (norm + eps)^2, the steps, and P / (norm + eps) to the front of the matrix's sums. A
// product's tiles on and above the diagonal are dealt out to 16 wavefronts, four to a SIMD: one waits for its operands or
// writes its tile while another's instructions run.
struct SmallLds {
    double A[kSmall * kSmallLd], Q[kSmall * kSmallLd], R[kSmall * kSmallLd], P[kSmall * kSmallLd], trace[16];
};
template <int tiles>
__device__ __forceinline__ void small_chain(const Matrix& e, double* __restrict__ sums, int steps, double a, double b, double c,
                                            double eps, SmallLds& lds) {
    double *A = lds.A, *Q = lds.Q, *R = lds.R, *P = lds.P, *trace = lds.trace;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    constexpr int pairs = tiles * (tiles + 1) / 2;
    const int row = lane >> 4, col = lane & 15;               // of a tile's result: row + 4 r, col
    // a tile on the diagonal holds its pairs twice: the upper one counts
    const auto put = [&](double* to, int ti, int tj, const double4v& v) {
        double* over = to + (16 * ti + row) * kSmallLd + 16 * tj + col;
        double* under = to + (16 * tj + col) * kSmallLd + 16 * ti + row;
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (ti < tj || row + 4 * r <= col) {
                over[4 * r * kSmallLd] = v[r];
                under[4 * r] = v[r];
            }
    };
    // S1 S2 at one tile; both symmetric and commuting
    const auto product = [&](const double* S1, const double* S2, int ti, int tj) {
        const double *p1 = S1 + (16 * ti + col) * kSmallLd + row, *p2 = S2 + (16 * tj + col) * kSmallLd + row;
        double x[4 * tiles], y[4 * tiles];
#pragma unroll
        for (int q = 0; q < 4 * tiles; ++q) {
            x[q] = p1[4 * q];
            y[q] = p2[4 * q];
        }
        double4v acc[2] = {};
#pragma unroll
        for (int q = 0; q < 4 * tiles; ++q) acc[q & 1] = __builtin_amdgcn_mfma_f64_16x16x4f64(x[q], y[q], acc[q & 1], 0, 0, 0);
        return acc[0] + acc[1];
    };
    int ti = 0, tj = 0;                                       // this wavefront's tile, and that of its second job below
    if (wave < pairs) pair_of(wave, ti, tj);
    double4v v = {};
    double tr = 0.0;
    if (wave < pairs) {
        const double* from = sums + wave * 256 + lane;
#pragma unroll 4
        for (int s = 0; s < e.split; ++s)
#pragma unroll
            for (int r = 0; r < 4; ++r) v[r] += from[(size_t)s * kGramValues + r * 64];
        if (ti == tj)
#pragma unroll
            for (int r = 0; r < 4; ++r) tr += row + 4 * r == col ? v[r] : 0.0;
    }
#pragma unroll
    for (int q = 32; q > 0; q >>= 1) tr += __shfl_xor(tr, q, 64);
    if (lane == 0) trace[wave] = tr;
    __syncthreads();
    tr = 0.0;
#pragma unroll
    for (int q = 0; q < pairs; ++q) tr += trace[q];
    const double inv = 1.0 / (sqrt(tr) + eps);
    if (wave < pairs) put(A, ti, tj, v * inv * inv);
    __syncthreads();
    for (int step = 0; step < steps; ++step) {
        const bool first = step == 0, last = step + 1 == steps;
        if (wave < pairs) {                                   // Q = a I + b A + c A A
            double4v q = product(A, A, ti, tj);
            const double* from = A + (16 * ti + row) * kSmallLd + 16 * tj + col;
#pragma unroll
            for (int r = 0; r < 4; ++r)
                q[r] = fma(b, from[4 * r * kSmallLd], c * q[r]) +
                       (ti == tj && row + 4 * r == col && 16 * ti + col < e.m ? a : 0.0);
            put(Q, ti, tj, q);
            if (first) put(P, ti, tj, q);
        }
        __syncthreads();
        // R = A Q, and P Q, which is held back until all have read P: the jobs behind R's fall to the wavefronts that have none
        double4v next[2] = {};
        if (!last && wave < pairs) put(R, ti, tj, product(A, Q, ti, tj));
        if (!first)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int job = wave + 16 * h - (last ? 0 : pairs);
                if (job < 0 || job >= pairs) continue;
                int pi, pj;
                pair_of(job, pi, pj);
                next[h] = product(P, Q, pi, pj);
            }
        __syncthreads();
        if (!first)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int job = wave + 16 * h - (last ? 0 : pairs);
                if (job < 0 || job >= pairs) continue;
                int pi, pj;
                pair_of(job, pi, pj);
                put(P, pi, pj, next[h]);
            }
        if (!last && wave < pairs) put(A, ti, tj, product(R, Q, ti, tj));
        __syncthreads();
    }
    for (int q = tid; q < kSmall * kSmall; q += 1024) {
        const int i = q / kSmall, j = q % kSmall;
        sums[q] = i < 16 * tiles && j < 16 * tiles ? P[i * kSmallLd + j] * inv : 0.0;
    }
}

__global__ __launch_bounds__(1024) void ns_small_chain_kernel(const Matrix* __restrict__ table, double* __restrict__ gram, int steps,
                                                              double a, double b, double c, double eps) {
    __shared__ SmallLds lds;
    const Matrix e = table[blockIdx.x];
    double* sums = gram + (size_t)e.sums0 * kGramValues;
    switch ((e.m + 15) / 16) {
        case 1: return small_chain<1>(e, sums, steps, a, b, c, eps, lds);
        case 2: return small_chain<2>(e, sums, steps, a, b, c, eps, lds);
        case 3: return small_chain<3>(e, sums, steps, a, b, c, eps, lds);
        default: return small_chain<4>(e, sums, steps, a, b, c, eps, lds);
    }
}

// result = P X, 64 columns per workgroup, 16 per wavefront
template <typename T>
__global__ __launch_bounds__(256) void ns_small_apply_kernel(const Matrix* __restrict__ table, int matrices, Blend k,
                                                             const double* __restrict__ gram, int out_type, int step, float decay) {
    __shared__ double P[kSmall * kSmallLd];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int block = blockIdx.x;
    const int w = find_matrix(lane < matrices ? (table[lane].n + 63) / 64 : 0, block);
    const Matrix& e = table[w];
    const int tiles = (e.m + 15) / 16, col = block * 64 + wave * 16 + (lane & 15);
    double x[16];
    small_values<T>(e, k, false, [&](int q) { return 4 * q + (lane >> 4); }, [&](int) { return col; }, x);
    const double* from = gram + (size_t)e.sums0 * kGramValues;
#pragma unroll
    for (int q = 0; q < kSmall * kSmall / 256; ++q) P[(q * 256 + tid) / kSmall * kSmallLd + tid % kSmall] = from[q * 256 + tid];
    __syncthreads();
    double4v acc[4] = {};
#pragma unroll
    for (int ti = 0; ti < 4; ++ti) {
        if (ti >= tiles) break;
        const int r1 = (16 * ti + (lane & 15)) * kSmallLd + (lane >> 4);
#pragma unroll
        for (int q = 0; q < 16; ++q)
            if (q < 4 * tiles) acc[ti] = __builtin_amdgcn_mfma_f64_16x16x4f64(P[r1 + 4 * q], x[q], acc[ti], 0, 0, 0);
    }
    with_type(out_type, [&](auto zero) {
        typedef decltype(zero) U;
        U* to = static_cast<U*>(e.out);
#pragma unroll
        for (int ti = 0; ti < 4; ++ti)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int i = 16 * ti + 4 * r + (lane >> 4);
                if (i < e.m && col < e.n) {
                    const size_t at = e.tall ? (size_t)col * e.m + i : (size_t)i * e.n + col;
                    float v = (float)acc[ti][r];
                    if (step) v = fmaf(decay, (float)to[at], -e.lr * v);
                    to[at] = (U)v;
                }
            }
    });
}

// ---- the sequence of launches ---------------------------------------------------------------------------------
struct Call {
    hipStream_t s;
    int count;
    const void* const* g;
    float* const* mom;                // NULL: orthogonalise g itself
    void* const* out;
    const int64_t *rows, *cols;
    const float* lr;                  // NULL without a step
    int g_type, out_type, steps;
    double a, b, c, eps;
    Blend blend;
    float decay;
    char* ws;
};

bool is_exact(const Call& k) { return k.g_type != FC3D_F32 && !k.mom; }     // the operands of the first products: one plane

struct Shape {
    int64_t m, n, mp, np;
    int64_t parts() const { return (m * n + kChunk - 1) / kChunk; }
    int64_t halves() const { return before(BUF_COUNT, mp, np); }
};
bool shape_of(int64_t rows, int64_t cols, Shape& s) {
    const int64_t most = 1 << 23;
    if (rows < 0 || cols < 0 || rows >= most || cols >= most) return false;
    s.m = rows < cols ? rows : cols;
    s.n = rows < cols ? cols : rows;
    s.mp = (s.m + kSlice - 1) / kSlice * kSlice;
    s.np = (s.n + kSlice - 1) / kSlice * kSlice;
    return (s.m / 64 + 2) * (s.n / 64 + 2) < (1 << 22);       // workgroups of a launch
}

float pow2_below(double bound) { return (float)std::exp2(14.0 - std::ceil(std::log2(bound))); }     // bound * it <= 2^14

// How many steps the Gram form takes at once.  A segment of L amplifies what it rounded gain^(2L)-fold: bf16 results bear
// five of the usual steps (gain 3.4), fp16 and fp32 ones three; steps that amplify more go two by two and, of fp32 results,
// one by one.  So do more than five steps: near one the usual polynomial spreads neighbouring values (its slope is -1.4 at
// 0.75), and every further step amplifies what a segment rounded (ten steps of a bf16 result five by five left it off by
// 1.1e-3 in front of its rounding, 1.7e-3).
constexpr double kGain = 4.0;
int segment_of(const Call& k, double gain) {                  // the longest one: the running products' scale follows from it
    const int apart = k.out_type == FC3D_F32 ? 1 : 2;
    const int most = gain > kGain || k.steps > 5 ? apart : k.out_type == FC3D_BF16 ? 5 : 3;
    return k.steps < most ? k.steps : most;
}
// Whether small matrices take all steps at once in 64 bits: what is rounded (1e-16) stays under 1e-5 when amplified, which
// ten of the usual steps do.
bool small_of(const Call& k, double gain) { return 2.0 * k.steps * std::log2(gain) <= 36.0; }

struct Scales {
    float x, a, r, q;                 // X, A, R = A Q, and Q with the running product
    double gain;                      // the most that a step multiplies a singular value by
    int segment;                      // steps of one segment
};
// Bounds on the spectra: singular values start in [0, 1] and stay below the polynomial's maximum over what they can be.
// false: the coefficients let them grow past what the fp16 pairs resolve.
bool scales_of(const Call& k, Scales& s) {
    double top = 1.0, all = 1.0;
    for (int i = 0; i < k.steps; ++i) {
        double next = 0.0;
        for (int j = 0; j <= 512; ++j) {
            const double x = top * j / 512.0, p = std::fabs(x * (k.a + x * x * (k.b + x * x * k.c)));
            if (!(p <= next)) next = p;
        }
        top = next * 1.01;
        if (!(top <= 16.0)) return false;
        if (top > all) all = top;
    }
    const double lam = all * all * 1.05;
    double q = 0.0, r = 0.0;
    for (int j = 0; j <= 512; ++j) {
        const double x = lam * j / 512.0, v = std::fabs(k.a + x * (k.b + x * k.c));
        if (v > q) q = v;
        if (v * x > r) r = v * x;
    }
    s.gain = q > 1.0 ? q : 1.0;
    s.segment = segment_of(k, s.gain);
    const double p = std::pow(s.gain, s.segment);
    if (!(p <= 65536.0)) return false;
    s.x = pow2_below(all * 1.05);
    s.a = pow2_below(lam);
    s.r = pow2_below(r > 1e-3 ? r * 1.05 : 1e-3);
    s.q = pow2_below(p * 1.05);
    return true;
}

// Plan 0 goes through segments of `segment` steps, plan 1 through one of two steps and one of three: fp16, large matrices in
// fp32, and matrices of up to kFew rows in bf16, whose results five steps at once would leave further off than their rounding
// allows (rank 1 and noise of 0.001, in front of a rounding of 1.7e-3: 17 rows 1.4e-3, 64 6.5e-4, 128 5.1e-4, 256 3.9e-4).
constexpr int kFew = 128;
int plan_of(const Call& k, double gain, const Shape& s) {
    if (gain > kGain || k.steps > 5) return 0;
    if (k.out_type == FC3D_BF16) return s.m <= kFew;
    return k.out_type == FC3D_F16 || (s.n >= 2 * s.m && s.m > 64);
}
bool starts(int segment, int plan, int step) {
    return plan == 0 ? step % segment == 0 : step == 0 || step == 2;
}

constexpr int kMaxOps = 5 * 64;
struct PlanOps {
    int count;
    Op op[kMaxOps][2];
};
// Every launch's products of one plan
void ops_of(const Call& k, int plan, const Scales& s, bool exact, PlanOps& to) {
    to.count = 0;
    uint8_t xt = BUF_XT0, p = BUF_P0, at = 0;                 // at: steps in front of the segment
    const auto put = [&](Op first, Op second) {
        to.op[to.count][0] = first;
        to.op[to.count++][1] = second;
    };
    const Op none = {};
    bool first_segment = true;
    const int segment = k.out_type == FC3D_F32 ? 1 : s.segment;     // plan 0 of an fp32 result: one by one
    for (int step = 0; step < k.steps; ++step) {
        const bool begin = starts(segment, plan, step), end = step + 1 == k.steps || starts(segment, plan, step + 1);
        const uint8_t whole = exact && first_segment, done = (uint8_t)step;
        if (begin) {
            at = done;
            put(Op{GRAM, BUF_X, BUF_X, BUF_A, s.a / (s.x * s.x), whole, 0, at, at}, none);
        }
        const uint8_t q = begin ? BUF_P0 : BUF_Q;              // the first of a segment is its running product too
        if (begin) p = BUF_P0;
        put(Op{POLY, BUF_A, BUF_A, q, (float)k.c * s.q / (s.a * s.a), 0, 0, 0, 0}, none);
        Op running = none;
        if (!begin) {
            const uint8_t np = p == BUF_P0 ? BUF_P1 : BUF_P0;
            running = Op{MUL, p, q, np, 1.0f / s.q, 0, 0, 0, 0};
            p = np;
        }
        if (!end) {
            put(Op{MUL, BUF_A, q, BUF_R, s.r / (s.a * s.q), 0, 0, 0, 0}, running);
            put(Op{MUL, BUF_R, q, BUF_A, s.a / (s.r * s.q), 0, 0, 0, 0}, none);
        } else {
            if (running.kind != NONE) put(running, none);
            const uint8_t last = step + 1 == k.steps, nxt = xt == BUF_XT0 ? BUF_XT1 : BUF_XT0;
            put(Op{APPLY, p, xt, nxt, (last ? 1.0f : s.x) / (s.q * s.x), whole, last, at, (uint8_t)(done + 1)}, none);
            xt = nxt;
            first_segment = false;
        }
    }
}

// What a group of matrices is worked on with, from its sizes alone: the workspace's size and its layout follow from it.
struct Layout {
    int64_t parts, halves, sum_tiles;
    int gram;                         // the Gram products' kernel
    int order[kMaxItems];             // the group's matrices as they are worked on: deep ones first, they take longest (numbers in the call)
    Shape shape[kMaxItems];           // in that order, like split
    int split[kMaxItems];
    int64_t head() const { return (parts * 8 + kMaxItems * (int64_t)(sizeof(Norm) + sizeof(Matrix)) + 255) / 256 * 256; }
    int64_t sums_at() const { return head() + (halves * 2 + 255) / 256 * 256; }
    bool small;                       // all of up to kSmall rows: sum_tiles is the number of partial Gram matrices
    int64_t bytes() const;
};

// The kernels a launch can take.  `beside`: workgroups that a compute unit holds.  A round of workgroups on all units
// takes `fixed` microseconds (starting, finding the tile, the first operands, the result's way out) and slice[] for every
// 64 of the depth, by the operands' planes (2 x 2, 2 x 1, 1 x 1); fitted to launches of 100 to 4000 tiles at depths of
// 512 to 8192.  Two small workgroups per unit hide each other's waits best; 96 x 96 tiles fill one round where the small
// ones need a second (2048 rows: 253 tiles, 37 us, against 46 us for 528); 128 x 128 tiles read least, for launches of many
// rounds of deep products (2048 x 8192, P X: 145 us against 191) and symmetric products of 1024 rows (32 us against 38);
// small ones hide a step's last product, which reads and writes the weights (1024 rows: 112 us against 129).
struct Kernel {
    int tile, waves, beside;
    double fixed, slice[3];
};
constexpr Kernel kKernels[] = {
    {64, 4, 2, 7.4, {0.68, 0.51, 0.32}}, {96, 4, 1, 9.8, {0.85, 0.73, 0.43}}, {128, 8, 1, 13.0, {1.33, 0.73, 0.56}}};
constexpr int kKernelCount = sizeof(kKernels) / sizeof(kKernels[0]);
constexpr int kUnits = 256;           // compute units
constexpr int kChunks = 128;          // small matrices: workgroups that share the columns of one, at most

// The kernel with the least expected time.  The last round, when not full, costs less: nothing shares its units.
int kernel_for(const int64_t (&groups)[kKernelCount], int64_t slices, int planes) {
    int best = 0;
    double least = 1e300;
    for (int i = 0; i < kKernelCount; ++i) {
        const Kernel& c = kKernels[i];
        const int64_t slots = (int64_t)kUnits * c.beside, rest = groups[i] % slots;
        const double round = c.fixed + c.slice[planes] * (double)slices;
        const double t = round * ((double)(groups[i] / slots) + (rest ? 0.6 + 0.4 * (double)rest / (double)slots : 0.0));
        if (t < least) {
            least = t;
            best = i;
        }
    }
    return best;
}

int64_t Layout::bytes() const {
    if (small) return head() + sum_tiles * kGramValues * 8;
    return sums_at() + sum_tiles * kKernels[gram].tile * kKernels[gram].tile * 4;
}

// `planes`: of the Gram products' operands; `small`: in three launches, if the matrices allow it
int layout_of(const Call& k, const int* list, int count, int planes, bool small, Layout& l) {
    for (int i = 0; i < count; ++i) {
        Shape s;
        if (!shape_of(k.rows[list[i]], k.cols[list[i]], s)) return FC3D_ERANGE;
        if (s.m == 0) return FC3D_EINVAL;
        int at = i;                                           // insertion: equal ones keep their order
        for (; at > 0 && l.shape[at - 1].n < s.n; --at) {
            l.shape[at] = l.shape[at - 1];
            l.order[at] = l.order[at - 1];
        }
        l.shape[at] = s;
        l.order[at] = list[i];
    }
    int64_t prep = 0, depth = 0;
    int64_t groups[kKernelCount] = {};
    l.parts = l.halves = l.sum_tiles = 0;
    l.small = small;
    for (int i = 0; i < count; ++i) l.small = l.small && l.shape[i].m <= kSmall;
    if (l.small) {
        for (int i = 0; i < count; ++i) {
            // columns of a chunk, at most kChunks chunks (two at least are laid out: the product P takes their place)
            Shape& s = l.shape[i];
            s.mp = kSmall;
            s.np = ((s.n + kChunks - 1) / kChunks + 63) / 64 * 64;
            l.split[i] = (int)((s.n + s.np - 1) / s.np);
            l.sum_tiles += l.split[i] < 2 ? 2 : l.split[i];
            prep += (s.n + 63) / 64;
        }
        return prep >= (1 << 23) ? FC3D_ERANGE : FC3D_OK;
    }
    for (int i = 0; i < count; ++i) {
        const Shape& s = l.shape[i];
        l.parts += s.parts();
        l.halves += s.halves();
        prep += s.mp / 64 * (s.np / 64);
        for (int c = 0; c < kKernelCount; ++c) groups[c] += tiles_of(MUL, (int)s.mp, 0, 1, kKernels[c].tile);
        if (s.np / kSlice > depth) depth = s.np / kSlice;
    }
    if (prep >= (1 << 23) || l.parts >= (1 << 23)) return FC3D_ERANGE;      // workgroups of one launch
    // The Gram products: the kernel is picked for them once, since the sums of shared depth are laid out for its tile.
    // Where there are few tiles, the depth is shared out, eight slices at least to each workgroup, one round of them.
    l.gram = kernel_for(groups, depth, planes);
    const int tile = kKernels[l.gram].tile;
    int64_t tiles = groups[l.gram], slices = 0;
    for (int i = 0; i < count; ++i) slices += tiles_of(MUL, (int)l.shape[i].mp, 0, 1, tile) * (l.shape[i].np / kSlice);
    int64_t each = (slices + kUnits - 1) / kUnits;
    if (each < 8) each = 8;
    for (;; ++each) {
        int64_t all = 0;
        l.sum_tiles = 0;
        for (int i = 0; i < count; ++i) {
            const int64_t deep = l.shape[i].np / kSlice, t = tiles_of(MUL, (int)l.shape[i].mp, 0, 1, tile);
            int64_t split = (deep + each - 1) / each;
            const int64_t per = (deep + split - 1) / split;
            split = (deep + per - 1) / per;                   // no share without a slice
            if (tiles > kUnits) split = 1;
            l.split[i] = (int)split;
            all += t * split;
            if (split > 1) l.sum_tiles += t * split;
        }
        if (all <= kUnits || l.sum_tiles == 0) break;         // one round, or nothing left to share
    }
    return FC3D_OK;
}

int64_t groups_of(const Launch& a, const Table& t, int tile) {
    int64_t n = 0;
    for (int i = 0; i < t.count; ++i)
        for (int j = 0; j < 2; ++j) n += tiles_of(a.op[t.e[i].plan][j].kind, t.e[i].mp, t.e[i].np, t.e[i].split, tile);
    return n;
}

// (the names tell the kernels apart in a profile: tile, and planes of the operands)
template <int TILE, int WAVES>
int product(const Call& k, const Launch& a, int64_t groups, int p1, int p2) {
    constexpr const char* names[3] = {TILE == 64 ? "ns_product_64_1x1" : TILE == 96 ? "ns_product_96_1x1" : "ns_product_128_1x1",
                                      TILE == 64 ? "ns_product_64_2x1" : TILE == 96 ? "ns_product_96_2x1" : "ns_product_128_2x1",
                                      TILE == 64 ? "ns_product_64_2x2" : TILE == 96 ? "ns_product_96_2x2" : "ns_product_128_2x2"};
    const dim3 grid((unsigned)groups), block(WAVES * 64);
    if (p1 == 1) FC3D_LAUNCH(names[0], (ns_product_kernel<TILE, WAVES, 1, 1>), grid, block, 0, k.s, a);
    else if (p2 == 1) FC3D_LAUNCH(names[1], (ns_product_kernel<TILE, WAVES, 2, 1>), grid, block, 0, k.s, a);
    else FC3D_LAUNCH(names[2], (ns_product_kernel<TILE, WAVES, 2, 2>), grid, block, 0, k.s, a);
    return FC3D_OK;
}
template <int TILE>
int gram_sum(const Call& k, const Launch& a, int64_t groups) {
    constexpr const char* name = TILE == 64 ? "ns_gram_sum_64" : TILE == 96 ? "ns_gram_sum_96" : "ns_gram_sum_128";
    FC3D_LAUNCH(name, ns_gram_sum_kernel<TILE>, dim3((unsigned)groups), dim3(256), 0, k.s, a);
    return FC3D_OK;
}

template <typename F>
int by_type(int type, F&& f) {
    return type == FC3D_F32 ? f(float{}) : type == FC3D_BF16 ? f(__bf16{}) : f(_Float16{});
}

int run_small(const Call& k, const Layout& l, int count) {
    Table t = {};
    t.count = count;
    int64_t sums = 0, gram_groups = 0, apply_groups = 0;
    for (int i = 0; i < count; ++i) {
        const Shape& s = l.shape[i];
        const int at = l.order[i];
        t.e[i] = Matrix{k.g[at], k.mom ? k.mom[at] : nullptr, k.out[at], 0, (int)s.m, (int)s.n, (int)s.mp, (int)s.np,
                        k.lr ? k.lr[at] : 0.0f, 0, l.split[i], (int)sums, k.rows[at] > k.cols[at], 0};
        sums += l.split[i] < 2 ? 2 : l.split[i];
        gram_groups += l.split[i];
        apply_groups += (s.n + 63) / 64;
    }
    Matrix* table = reinterpret_cast<Matrix*>(k.ws);
    double* gram = reinterpret_cast<double*>(k.ws + l.head());
    return by_type(k.g_type, [&](auto zero) {
        typedef decltype(zero) T;
        FC3D_LAUNCH("ns_small_gram", ns_small_gram_kernel<T>, dim3((unsigned)gram_groups), dim3(256), 0, k.s, t, k.blend, table, gram);
        FC3D_LAUNCH("ns_small_chain", ns_small_chain_kernel, dim3((unsigned)count), dim3(1024), 0, k.s, table, gram, k.steps, k.a,
                    k.b, k.c, k.eps);
        FC3D_LAUNCH("ns_small_apply", ns_small_apply_kernel<T>, dim3((unsigned)apply_groups), dim3(256), 0, k.s, table, count,
                    k.blend, gram, k.out_type, (int)(k.lr != nullptr), k.decay);
        return FC3D_OK;
    });
}

int run_group(const Call& k, const Layout& l, const Scales& sc, int count) {
    Table t = {};
    t.count = count;
    const bool exact = is_exact(k);
    int64_t parts = 0, halves = 0, prep = 0, sums = 0;
    bool used[kPlans] = {};
    for (int i = 0; i < count; ++i) {
        const Shape& s = l.shape[i];
        const int at = l.order[i], plan = plan_of(k, sc.gain, s);
        t.e[i] = Matrix{k.g[at], k.mom ? k.mom[at] : nullptr, k.out[at], halves, (int)s.m, (int)s.n, (int)s.mp, (int)s.np,
                        k.lr ? k.lr[at] : 0.0f, (int)parts, l.split[i], (int)sums, k.rows[at] > k.cols[at], plan};
        used[plan] = true;
        parts += s.parts();
        halves += s.halves();
        prep += s.mp / 64 * (s.np / 64);
        if (l.split[i] > 1) sums += (int64_t)tiles_of(MUL, (int)s.mp, 0, 1, kKernels[l.gram].tile) * l.split[i];
    }
    double* squares = reinterpret_cast<double*>(k.ws);
    Matrix* table = reinterpret_cast<Matrix*>(k.ws + parts * 8);
    Norm* norms = reinterpret_cast<Norm*>(table + kMaxItems);
    _Float16* planes = reinterpret_cast<_Float16*>(k.ws + l.head());
    const auto first = [&](auto zero) {
        typedef decltype(zero) T;
        FC3D_LAUNCH("ns_norm", ns_norm_kernel<T>, dim3((unsigned)parts), dim3(256), 0, k.s, t, k.blend, squares, table);
        FC3D_LAUNCH("ns_prepare", ns_prepare_kernel<T>, dim3((unsigned)prep), dim3(256), 0, k.s, table, count, k.blend, squares,
                    k.eps, sc.x, (int)exact, planes, norms);
        return FC3D_OK;
    };
    if (const int rc = by_type(k.g_type, first)) return rc;

    static thread_local PlanOps ops[kPlans];
    int launches = 0;
    for (int p = 0; p < kPlans; ++p) {
        ops[p].count = 0;
        if (used[p]) ops_of(k, p, sc, exact, ops[p]);
        if (ops[p].count > launches) launches = ops[p].count;
    }
    Launch a = {};
    a.a = (float)k.a * sc.q;
    a.b = (float)k.b * sc.q / sc.a;
    a.out_type = k.out_type;
    a.step = k.lr != nullptr;
    a.decay = k.decay;
    a.matrices = count;
    a.table = table;
    a.planes = planes;
    a.norms = norms;
    a.gain = (float)std::log2(sc.gain);
    a.sums = reinterpret_cast<float*>(k.ws + l.sums_at());
    for (int i = 0; i < launches; ++i) {
        // An input taken as it is has one plane (the other is zero).  It is left out where no product of the launch needs it.
        bool gram = false;
        int p1 = 1, p2 = 1;
        for (int p = 0; p < kPlans; ++p)
            for (int j = 0; j < 2; ++j) {
                const Op& o = a.op[p][j] = i < ops[p].count ? ops[p].op[i][j] : Op{};
                if (o.kind == NONE) continue;
                gram = gram || o.kind == GRAM;
                if (!(o.exact && o.kind == GRAM)) p1 = 2;
                if (!o.exact) p2 = 2;
            }
        int64_t groups[kKernelCount], depth = 0;
        for (int c = 0; c < kKernelCount; ++c) groups[c] = groups_of(a, t, kKernels[c].tile);
        for (int j = 0; j < count; ++j) {
            const Op& o = a.op[t.e[j].plan][0];
            const int64_t d = o.kind == NONE ? 0 : o.kind == GRAM ? t.e[j].np / kSlice / t.e[j].split : t.e[j].mp / kSlice;
            if (d > depth) depth = d;
        }
        const int c = gram ? l.gram : kernel_for(groups, depth, p2 == 2 ? 0 : 1);
        const int rc = c == 0 ? product<64, 4>(k, a, groups[c], p1, p2) : c == 1 ? product<96, 4>(k, a, groups[c], p1, p2)
                                                                       : product<128, 8>(k, a, groups[c], p1, p2);
        if (rc != FC3D_OK) return rc;
        int64_t sum_groups = 0;
        for (int j = 0; j < count; ++j)
            if (a.op[t.e[j].plan][0].kind == GRAM && t.e[j].split > 1) sum_groups += tiles_of(MUL, t.e[j].mp, 0, 1, kKernels[c].tile);
        if (sum_groups) {
            const int tile = kKernels[c].tile;
            if (const int rc = tile == 64 ? gram_sum<64>(k, a, sum_groups) : tile == 96 ? gram_sum<96>(k, a, sum_groups)
                                                                                       : gram_sum<128>(k, a, sum_groups))
                return rc;
        }
    }
    return FC3D_OK;
}

bool known_type(int t) { return t >= FC3D_F32 && t <= FC3D_F16; }
bool off_align(const void* p, int type) { return (reinterpret_cast<uintptr_t>(p) & (type == FC3D_F32 ? 3u : 1u)) != 0; }

// Matrices of up to kTiny rows in a list with larger ones go through three launches of their own in 64 bits: a result of a
// few rows averages little.  Pairs of fp16 values left some fp32 results three times as far off as fp32 products do (2.2e-6
// against 6e-7), and a bf16 result's five steps at once cost up to 2e-3, as much as its rounding, where its rows were nearly
// dependent (rank 1 and noise of 0.01, 2 to 8 rows).  One tile of rows: 20 us for all of them together.
constexpr int kTiny = 16;
int64_t rows_of(const Call& k, int i) { return k.rows[i] < k.cols[i] ? k.rows[i] : k.cols[i]; }
bool mixed(const Call& k) {
    bool tiny = false, large = false;
    for (int i = 0; i < k.count; ++i) {
        tiny = tiny || rows_of(k, i) <= kTiny;
        large = large || rows_of(k, i) > kSmall;
    }
    return tiny && large;
}

// Matrices in groups of up to kMaxItems, one group after the other in the same workspace; `apart`: the tiny ones behind the
// rest.  A group ends too where its buffers, eight times its weights in fp32, would pass a GiB: what fills that fills the
// compute units several times over (32 matrices of 1024 x 1024), and 48 matrices of 4096 x 4096 would take 24 GiB.  `small`:
// of matrices of up to kSmall rows alone, which then need no such buffers.
constexpr int64_t kGroupBytes = (int64_t)1 << 30;
template <typename F>
int in_groups(const Call& k, bool apart, bool small, F&& f) {
    int list[kMaxItems];
    bool large = false;
    for (int i = 0; i < k.count; ++i) large = large || rows_of(k, i) > kSmall;
    for (int turn = 0; turn < (apart ? 2 : 1); ++turn) {
        int count = 0;
        int64_t bytes = 0;
        for (int i = 0; i < k.count; ++i) {
            if (apart && (rows_of(k, i) <= kTiny) != (turn == 1)) continue;
            Shape s;
            if (!shape_of(k.rows[i], k.cols[i], s)) return FC3D_ERANGE;
            const int64_t own = small && (turn == 1 || !large) ? 0 : 2 * s.halves();
            if (count == kMaxItems || (count > 0 && bytes + own > kGroupBytes)) {
                if (const int rc = f(list, count)) return rc;
                count = 0;
                bytes = 0;
            }
            list[count++] = i;
            bytes += own;
        }
        if (count > 0)
            if (const int rc = f(list, count)) return rc;
    }
    return FC3D_OK;
}
// The workspace is sized for every layout that a call with these sizes may take
int size_of(const Call& k, size_t& bytes) {
    bytes = 0;
    for (int small = 0; small < 2; ++small)
        for (int apart = 0; apart <= (int)(small && mixed(k)); ++apart)
            if (const int rc = in_groups(k, apart != 0, small != 0, [&](const int* list, int count) {
                    for (int planes = 0; planes <= 2; planes += 2) {
                        Layout l = {};
                        if (const int rc = layout_of(k, list, count, planes, small != 0, l)) return rc;
                        if ((size_t)l.bytes() > bytes) bytes = (size_t)l.bytes();
                    }
                    return (int)FC3D_OK;
                }))
                return rc;
    return FC3D_OK;
}

int run(const Call& k) {
    Scales sc = {};
    if (!scales_of(k, sc)) return FC3D_ERANGE;
    const bool small = small_of(k, sc.gain);
    return in_groups(k, small && mixed(k), small, [&](const int* list, int count) {
        Layout l = {};
        if (const int rc = layout_of(k, list, count, is_exact(k) ? 2 : 0, small, l)) return rc;
        return l.small ? run_small(k, l, count) : run_group(k, l, sc, count);
    });
}

int check_call(const Call& k) {
    if (k.count < 0 || !known_type(k.g_type) || !known_type(k.out_type)) return FC3D_EINVAL;
    if (k.steps < 1 || k.steps > 64 || !(k.eps >= 0.0) || !std::isfinite(k.a + k.b + k.c)) return FC3D_EINVAL;
    if (k.count == 0) return FC3D_OK;
    if (!k.g || !k.out || !k.rows || !k.cols || !k.ws) return FC3D_EINVAL;
    if (reinterpret_cast<uintptr_t>(k.ws) & 255u) return FC3D_EALIGN;
    for (int i = 0; i < k.count; ++i) {
        if (!k.g[i] || !k.out[i] || (k.mom && !k.mom[i]) || k.rows[i] <= 0 || k.cols[i] <= 0) return FC3D_EINVAL;
        if (off_align(k.g[i], k.g_type) || off_align(k.out[i], k.out_type) || (k.mom && off_align(k.mom[i], FC3D_F32))) return FC3D_EALIGN;
    }
    // sizes and coefficients are checked before the first launch, the latter alike for all types: a caller that works
    // on several lists is refused before the first one or not at all
    Call most = k;
    most.out_type = FC3D_BF16;
    Scales sc;
    if (!scales_of(most, sc)) return FC3D_ERANGE;
    size_t bytes;
    return size_of(k, bytes);
}

}  // namespace
}  // namespace fc3d

using namespace fc3d;

extern "C" size_t fc3d_orthogonalize_workspace(int count, const int64_t* rows, const int64_t* cols) {
    if (count <= 0 || !rows || !cols) return 0;
    Call k = {};
    k.count = count;
    k.rows = rows;
    k.cols = cols;
    size_t bytes = 0;
    return size_of(k, bytes) == FC3D_OK ? bytes : 0;
}

extern "C" int fc3d_orthogonalize(void* stream, int count, const void* const* g, void* const* out, const int64_t* rows,
                                  const int64_t* cols, int type, int steps, double a, double b, double c, double eps,
                                  void* workspace) {
    Call k = {};
    k.s = (hipStream_t)stream;
    k.count = count;
    k.g = g;
    k.out = out;
    k.rows = rows;
    k.cols = cols;
    k.g_type = k.out_type = type;
    k.steps = steps;
    k.a = a;
    k.b = b;
    k.c = c;
    k.eps = eps;
    k.ws = (char*)workspace;
    if (const int rc = check_call(k)) return rc;
    return run(k);
}

extern "C" int fc3d_muon_step(void* stream, int count, void* const* params, const void* const* grads, float* const* momenta,
                              const int64_t* rows, const int64_t* cols, const float* lr, int param_type, int grad_type,
                              double momentum, int nesterov, double decay, int steps, double a, double b, double c, double eps,
                              void* workspace) {
    if (count > 0 && (!momenta || !lr)) return FC3D_EINVAL;
    if (!(momentum >= 0.0 && momentum <= 1.0) || !std::isfinite(decay)) return FC3D_EINVAL;
    Call k = {};
    k.s = (hipStream_t)stream;
    k.count = count;
    k.g = grads;
    k.mom = momenta;
    k.out = params;
    k.rows = rows;
    k.cols = cols;
    k.lr = lr;
    k.g_type = grad_type;
    k.out_type = param_type;
    k.steps = steps;
    k.a = a;
    k.b = b;
    k.c = c;
    k.eps = eps;
    k.blend = Blend{(float)momentum, (float)(1.0 - momentum), nesterov};
    k.decay = (float)decay;
    k.ws = (char*)workspace;
    if (const int rc = check_call(k)) return rc;
    return run(k);
}
