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
// directions whose share of A is below its rounding, amplified a^(2L)-fold: five steps at once cost 1e-4 of the
// result in bad cases (measured in emulation, low rank plus noise), which is below the rounding of a 16-bit result;
// for fp32 results the segments are of two and three steps, or of one for matrices that are nearly square
// (n < 2 m, where the smallest singular values sit near zero), as accurate as step by step.
#include "fc3d_common.h"

#include <cmath>

namespace fc3d {
namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef float float16v __attribute__((ext_vector_type(16)));

constexpr int kTile = 64;             // products: output tile, and depth of one staged slice
constexpr int kMaxItems = 48;         // matrices of one launch (their descriptions travel as kernel arguments)
constexpr int kMaxJobs = 2 * kMaxItems;
constexpr int kChunk = 16384;         // elements of one workgroup of the norm pass

// A matrix's buffers, each a plane of hi values and one of lo values: X in two orders (the transpose twice: a segment
// reads one and writes the other), then the m x m matrices of the Gram form.
enum Buffer : uint8_t { BUF_X, BUF_XT0, BUF_XT1, BUF_A, BUF_Q, BUF_R, BUF_P0, BUF_P1, BUF_COUNT };

struct Job {                          // one product (or one matrix) of a launch
    int64_t base;                     // halves from the start of the workspace's planes to the matrix's buffers
    int m, n;                         // m <= n
    int first;                        // the launch's first workgroup that works on it
    uint8_t src1, src2, dst, op;      // buffers, and which of the launch's scales is the result's
    int slot;                         // the matrix's number in the call
};
template <int N>
struct Jobs {
    int count;
    Job e[N];
};
struct Io {                           // a matrix's tensors
    const void* g;
    float* mom;
    void* out;
    float lr;                         // learning rate times the shape's factor
    int tall;                         // the tensor is n x m
    int part0;                        // its first partial sum of squares
};
struct Ios {
    Io e[kMaxItems];
};

__host__ __device__ inline int padded(int v) { return (v + kTile - 1) / kTile * kTile; }

// The entry whose workgroups hold `block`
template <int N>
__device__ __forceinline__ int find_job(const Jobs<N>& t, int block) {
    int lo = 0, hi = t.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (t.e[mid].first <= block) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

__device__ __forceinline__ float ld_any(const void* p, int type, size_t i) {
    if (type == FC3D_F32) return static_cast<const float*>(p)[i];
    if (type == FC3D_BF16) return (float)static_cast<const __bf16*>(p)[i];
    return (float)static_cast<const _Float16*>(p)[i];
}
__device__ __forceinline__ void st_any(void* p, int type, size_t i, float v) {
    if (type == FC3D_F32) static_cast<float*>(p)[i] = v;
    else if (type == FC3D_BF16) static_cast<__bf16*>(p)[i] = (__bf16)v;
    else static_cast<_Float16*>(p)[i] = (_Float16)v;
}

struct Blend {                        // m' = beta m + (1 - beta) g;  u = (1 - beta) g + beta m' (nesterov) or m'
    float beta, rest;
    int nesterov;
};
__device__ __forceinline__ float blend(const Blend& k, float g, float mom_new) {
    return k.nesterov ? fmaf(k.beta, mom_new, k.rest * g) : mom_new;
}

// Sums of squares of the update per workgroup (64 bits: any fp32 input stays in range), and the momentum's update.
__global__ __launch_bounds__(256) void ns_norm_kernel(Jobs<kMaxItems> t, Ios io, int type, Blend k, double* __restrict__ parts) {
    __shared__ double red[4];
    const int i = find_job(t, blockIdx.x);
    const Io& o = io.e[i];
    const size_t count = (size_t)t.e[i].m * t.e[i].n;
    const size_t lo = (size_t)((int)blockIdx.x - t.e[i].first) * kChunk;
    const size_t hi = lo + kChunk < count ? lo + kChunk : count;
    double s = 0.0;
    for (size_t j = lo + threadIdx.x; j < hi; j += 256) {
        float u = ld_any(o.g, type, j);
        if (o.mom) {
            const float mn = fmaf(k.beta, o.mom[j], k.rest * u);
            o.mom[j] = mn;
            u = blend(k, u, mn);
        }
        s = fma((double)u, (double)u, s);
    }
#pragma unroll
    for (int q = 32; q > 0; q >>= 1) s += __shfl_xor(s, q, 64);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) parts[o.part0 + (int)blockIdx.x - t.e[i].first] = (red[0] + red[1]) + (red[2] + red[3]);
}

__device__ __forceinline__ void split_store(_Float16* p, size_t plane, size_t at, float v) {
    const _Float16 h = (_Float16)v;
    p[at] = h;
    p[plane + at] = (_Float16)(v - (float)h);
}

// X and its transpose, scaled by sx / (norm + eps), zero beyond the matrix, one 64 x 64 tile per workgroup.
// `exact` (16-bit input taken as it is): one plane that holds the input times a power of two, without rounding; the
// remaining factor in [1, 2) goes to rho and into the products that read X.
__global__ __launch_bounds__(256) void ns_prepare_kernel(Jobs<kMaxItems> t, Ios io, int type, Blend k, const double* __restrict__ parts,
                                                         double eps, float sx, int exact, _Float16* __restrict__ planes,
                                                         float* __restrict__ rho) {
    __shared__ float tile[kTile][kTile + 1];
    __shared__ double red[4];
    const int i = find_job(t, blockIdx.x);
    const Job& e = t.e[i];
    const Io& o = io.e[i];
    const int mp = padded(e.m), np = padded(e.n);
    const int count = (int)(((size_t)e.m * e.n + kChunk - 1) / kChunk);
    double s = 0.0;
    for (int q = threadIdx.x; q < count; q += 256) s += parts[o.part0 + q];
#pragma unroll
    for (int q = 32; q > 0; q >>= 1) s += __shfl_xor(s, q, 64);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    const double factor = (double)sx / (sqrt((red[0] + red[1]) + (red[2] + red[3])) + eps);
    int shift = 0;
    float rest = 1.0f;
    if (exact) {
        rest = 2.0f * (float)frexp(factor, &shift);          // factor = rest * 2^(shift - 1), rest in [1, 2)
        shift -= 1;
        if (!(factor < 1e300)) shift = 0;                    // a zero matrix with eps 0, or a NaN: 0 * inf below
        if (!(factor < 1e300) || factor == 0.0) rest = (float)factor;
    }
    const int block = (int)blockIdx.x - e.first, tn = np / kTile;
    const int i0 = block / tn * kTile, j0 = block % tn * kTile;
    if (block == 0 && threadIdx.x == 0) rho[e.slot] = rest;
    const int tx = threadIdx.x & 63, ty = threadIdx.x >> 6;
#pragma unroll
    for (int q = 0; q < 16; ++q) {
        const int fast = tx, slow = q * 4 + ty;              // fast: along the tensor's rows
        const int r = o.tall ? fast : slow, c = o.tall ? slow : fast;
        float v = 0.0f;
        if (i0 + r < e.m && j0 + c < e.n) {
            const size_t at = o.tall ? (size_t)(j0 + c) * e.m + (i0 + r) : (size_t)(i0 + r) * e.n + (j0 + c);
            v = ld_any(o.g, type, at);
            if (o.mom) v = blend(k, v, o.mom[at]);
            v = exact ? ldexpf(v, shift) : (float)((double)v * factor);
        }
        tile[r][c] = v;
    }
    __syncthreads();
    const size_t plane = (size_t)mp * np;
    _Float16* x = planes + e.base;
    _Float16* xt = x + 2 * plane;
#pragma unroll
    for (int q = 0; q < 16; ++q) {
        const int r = q * 4 + ty;
        split_store(x, plane, (size_t)(i0 + r) * np + j0 + tx, tile[r][tx]);
        split_store(xt, plane, (size_t)(j0 + r) * mp + i0 + tx, tile[tx][r]);
    }
}

// ---- products -----------------------------------------------------------------------------------------------
// D[i][j] = sum_k S1[i][k] S2[j][k]: both operands run along the depth in memory (a symmetric matrix is its own
// transpose, and X is kept in both orders), so one kernel serves every product.
enum Kind { GRAM, POLY, MUL, APPLY };

struct Product {
    _Float16* planes;
    const float* rho;
    float alpha[2];                   // sum -> stored value (scales of the operands and of the result), by Job::op
    float a, b;                       // POLY: Q = a I + b A + c A^2, in units of the stored result
    int use_rho;                      // the first segment of an input taken as it is
    // APPLY
    int last;                         // to the tensors, else back to X and its transpose
    int out_type, step;               // step: weights := decay * weights - lr * result
    float decay;
};

__device__ __forceinline__ _Float16* buffer(const Job& e, _Float16* planes, int id, int& ld, size_t& plane) {
    const int mp = padded(e.m), np = padded(e.n);
    const size_t xn = (size_t)mp * np, an = (size_t)mp * mp;
    if (id < BUF_A) {
        ld = id == BUF_X ? np : mp;
        plane = xn;
        return planes + e.base + (size_t)id * 2 * xn;
    }
    ld = mp;
    plane = an;
    return planes + e.base + 6 * xn + (size_t)(id - BUF_A) * 2 * an;
}

struct NoIos {};
// P1, P2: planes of the operands that count (1: the lo plane is zero)
template <int KIND, int P1, int P2, int N, typename IO>
__global__ __launch_bounds__(256) void ns_product_kernel(Jobs<N> t, IO io, Product a) {
    __shared__ half8 lds[(P1 + P2) * kTile * kTile / 8];
    const int w = find_job(t, blockIdx.x);
    const Job& e = t.e[w];
    const int block = (int)blockIdx.x - e.first;
    int ti, tj;
    if constexpr (KIND == APPLY) {
        const int tn = padded(e.n) / kTile;
        ti = block / tn;
        tj = block % tn;
    } else {                                                  // the upper triangle, column by column
        tj = (int)((sqrtf(8.0f * (float)block + 1.0f) - 1.0f) * 0.5f);
        while ((long)tj * (tj + 1) / 2 > block) --tj;
        while ((long)(tj + 1) * (tj + 2) / 2 <= block) ++tj;
        ti = block - (int)((long)tj * (tj + 1) / 2);
    }
    int ld1, ld2;
    size_t pl1, pl2;
    const _Float16* s1 = buffer(e, a.planes, e.src1, ld1, pl1) + (size_t)ti * kTile * ld1;
    const _Float16* s2 = buffer(e, a.planes, e.src2, ld2, pl2) + (size_t)tj * kTile * ld2;
    const int depth = KIND == GRAM ? padded(e.n) : padded(e.m);

    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int wi = (wave >> 1) * 32, wj = (wave & 1) * 32;
    // 16-byte pieces of a row of 64 values are stored at piece ^ (row & 7): eight rows read at one depth then lie in
    // different banks
    half8 next[(P1 + P2) * 2];
    const auto fetch = [&](int k0) {
#pragma unroll
        for (int p = 0; p < P1 + P2; ++p)
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                const int id = tid + 256 * q, row = id >> 3, piece = id & 7;
                const _Float16* src = p < P1 ? s1 + p * pl1 + (size_t)row * ld1 : s2 + (p - P1) * pl2 + (size_t)row * ld2;
                next[p * 2 + q] = *reinterpret_cast<const half8*>(src + k0 + piece * 8);
            }
    };
    const auto stage = [&]() {
#pragma unroll
        for (int p = 0; p < P1 + P2; ++p)
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                const int id = tid + 256 * q, row = id >> 3, piece = id & 7;
                lds[p * 512 + row * 8 + (piece ^ (row & 7))] = next[p * 2 + q];
            }
    };
    float16v acc = {};
    fetch(0);
    for (int k0 = 0; k0 < depth; k0 += kTile) {
        __syncthreads();
        stage();
        __syncthreads();
        if (k0 + kTile < depth) fetch(k0 + kTile);
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
            const int r1 = wi + (lane & 31), r2 = wj + (lane & 31), piece = kk * 2 + (lane >> 5);
            half8 f1[P1], f2[P2];
#pragma unroll
            for (int p = 0; p < P1; ++p) f1[p] = lds[p * 512 + r1 * 8 + (piece ^ (r1 & 7))];
#pragma unroll
            for (int p = 0; p < P2; ++p) f2[p] = lds[(P1 + p) * 512 + r2 * 8 + (piece ^ (r2 & 7))];
            if constexpr (P2 > 1) acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(f1[0], f2[1], acc, 0, 0, 0);
            if constexpr (P1 > 1) acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(f1[1], f2[0], acc, 0, 0, 0);
            acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(f1[0], f2[0], acc, 0, 0, 0);
        }
    }
    // lane: column (lane & 31) of its wavefront's 32 x 32, rows 8 (r / 4) + 4 (lane / 32) + r % 4
    float alpha = a.alpha[e.op];
    if constexpr (KIND == GRAM || KIND == APPLY)
        if (a.use_rho) alpha *= KIND == GRAM ? a.rho[e.slot] * a.rho[e.slot] : a.rho[e.slot];
    const int j = tj * kTile + wj + (lane & 31);
    int ld;
    size_t plane;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        const int i = ti * kTile + wi + 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3);
        float v = acc[r] * alpha;
        if constexpr (KIND == APPLY) {
            if (a.last) {
                if (i < e.m && j < e.n) {
                    const Io& o = io.e[w];
                    const size_t at = o.tall ? (size_t)j * e.m + i : (size_t)i * e.n + j;
                    if (a.step) v = fmaf(a.decay, ld_any(o.out, a.out_type, at), -o.lr * v);
                    st_any(o.out, a.out_type, at, v);
                }
            } else {
                _Float16* x = buffer(e, a.planes, BUF_X, ld, plane);
                split_store(x, plane, (size_t)i * ld + j, v);
                x = buffer(e, a.planes, e.dst, ld, plane);
                split_store(x, plane, (size_t)j * ld + i, v);
            }
        } else {
            if constexpr (KIND == POLY) {
                const _Float16* A = buffer(e, a.planes, e.src1, ld, plane);
                const size_t at = (size_t)i * ld + j;
                v = fmaf(a.b, (float)A[at] + (float)A[plane + at], v);
                if (i == j && i < e.m) v += a.a;
            }
            _Float16* d = buffer(e, a.planes, e.dst, ld, plane);
            // a tile on the diagonal computes each pair twice, with its cross terms in two orders: one of them counts
            if (ti != tj || i <= j) split_store(d, plane, (size_t)i * ld + j, v);
            if (ti != tj || i < j) split_store(d, plane, (size_t)j * ld + i, v);
        }
    }
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

struct Shape {
    int64_t m, n, mp, np;
    int64_t parts() const { return (m * n + kChunk - 1) / kChunk; }
    int64_t halves() const { return 6 * mp * np + (int64_t)(BUF_COUNT - BUF_A) * 2 * mp * mp; }
};
bool shape_of(int64_t rows, int64_t cols, Shape& s) {
    const int64_t most = 1 << 24;
    if (rows < 0 || cols < 0 || rows >= most || cols >= most) return false;
    s.m = rows < cols ? rows : cols;
    s.n = rows < cols ? cols : rows;
    s.mp = (s.m + kTile - 1) / kTile * kTile;
    s.np = (s.n + kTile - 1) / kTile * kTile;
    return (s.mp / kTile) * (s.np / kTile) < (1 << 22);       // workgroups of a launch
}

// Bytes of the workspace's head: the partial sums and one factor per matrix
int64_t head_bytes(int64_t parts) { return (parts * 8 + kMaxItems * 4 + 255) / 256 * 256; }

float pow2_below(double bound) { return (float)std::exp2(14.0 - std::ceil(std::log2(bound))); }     // bound * it <= 2^14

struct Scales {
    float x, a, r, q;                 // X, A, R = A Q, and Q with the running product
};
// Bounds on the spectra: singular values start in [0, 1] and stay below the polynomial's maximum over what they can be.
// false: the coefficients let them grow past what the fp16 pairs resolve.
bool scales_of(const Call& k, int longest, Scales& s) {
    double top = 1.0, all = 1.0;
    for (int i = 0; i < k.steps; ++i) {
        double next = 0.0;
        for (int j = 0; j <= 2048; ++j) {
            const double x = top * j / 2048.0, p = std::fabs(x * (k.a + x * x * (k.b + x * x * k.c)));
            if (!(p <= next)) next = p;
        }
        top = next * 1.01;
        if (!(top <= 16.0)) return false;
        if (top > all) all = top;
    }
    const double lam = all * all * 1.05;
    double q = 0.0, r = 0.0;
    for (int j = 0; j <= 2048; ++j) {
        const double x = lam * j / 2048.0, v = std::fabs(k.a + x * (k.b + x * k.c));
        if (v > q) q = v;
        if (v * x > r) r = v * x;
    }
    const double p = std::pow(q > 1.0 ? q : 1.0, longest);
    if (!(p <= 65536.0)) return false;
    s.x = pow2_below(all * 1.05);
    s.a = pow2_below(lam);
    s.r = pow2_below(r > 1e-3 ? r * 1.05 : 1e-3);
    s.q = pow2_below(p * 1.05);
    return true;
}

// The steps of one matrix in segments; segment lengths fall on step k with starts(k) / ends(k).
struct Segments {
    int first, rest;                  // length of the first one, of the others (the last may be shorter)
    bool starts(int k) const { return k == 0 || (k >= first && (k - first) % rest == 0); }
    bool ends(int k, int steps) const { return k == steps - 1 || starts(k + 1); }
};
// More than five steps of an fp32 result go one by one: near one the usual polynomial spreads neighbouring values
// (its slope is -1.4 at 0.75), so that every further step amplifies what the segments before it rounded.
Segments segments_of(int out_type, int steps, const Shape& s) {
    if (out_type != FC3D_F32) return {5, 5};
    if (s.n < 2 * s.m || steps > 5) return {1, 1};
    return {2, 3};
}

template <int N>
int64_t workgroups(Jobs<N>& t, int kind) {        // numbers the entries' workgroups, returns their sum
    int64_t sum = 0;
    for (int i = 0; i < t.count; ++i) {
        Job& e = t.e[i];
        const int64_t tm = padded(e.m) / kTile, tn = padded(e.n) / kTile;
        e.first = (int)sum;
        sum += kind == APPLY ? tm * tn : tm * (tm + 1) / 2;
    }
    return sum;
}

int run_group(const Call& k, int from, int count, const Shape* shapes, const Scales& sc) {
    Jobs<kMaxItems> all = {};
    Ios io = {};
    all.count = count;
    int64_t parts = 0, halves = 0, norm_groups = 0, prep_groups = 0;
    bool exact = k.g_type != FC3D_F32 && !k.mom;
    for (int i = 0; i < count; ++i) {
        const int at = from + i;
        const Shape& s = shapes[i];
        all.e[i] = Job{halves, (int)s.m, (int)s.n, 0, 0, 0, 0, 0, i};
        io.e[i] = Io{k.g[at], k.mom ? k.mom[at] : nullptr, k.out[at], k.lr ? k.lr[at] : 0.0f, k.rows[at] > k.cols[at], (int)parts};
        parts += s.parts();
        halves += s.halves();
    }
    double* sums = reinterpret_cast<double*>(k.ws);
    float* rho = reinterpret_cast<float*>(k.ws + parts * 8);
    _Float16* planes = reinterpret_cast<_Float16*>(k.ws + head_bytes(parts));

    Jobs<kMaxItems> t = all;
    for (int i = 0; i < count; ++i) {
        t.e[i].first = (int)norm_groups;
        norm_groups += shapes[i].parts();
    }
    FC3D_LAUNCH("ns_norm", ns_norm_kernel, dim3((unsigned)norm_groups), dim3(256), 0, k.s, t, io, k.g_type, k.blend, sums);
    for (int i = 0; i < count; ++i) {
        t.e[i].first = (int)prep_groups;
        prep_groups += shapes[i].mp / kTile * (shapes[i].np / kTile);
    }
    FC3D_LAUNCH("ns_prepare", ns_prepare_kernel, dim3((unsigned)prep_groups), dim3(256), 0, k.s, t, io, k.g_type, k.blend, sums,
                k.eps, sc.x, (int)exact, planes, rho);

    uint8_t xt[kMaxItems], p[kMaxItems];
    for (int i = 0; i < count; ++i) xt[i] = BUF_XT0;
    Product arg = {};
    arg.planes = planes;
    arg.rho = rho;
    arg.out_type = k.out_type;
    arg.step = k.lr != nullptr;
    arg.decay = k.decay;
    for (int step = 0; step < k.steps; ++step) {
        Segments seg[kMaxItems];
        uint8_t q[kMaxItems];
        Jobs<kMaxItems> one = {};
        // A = X X^T where a segment starts
        for (int i = 0; i < count; ++i) {
            seg[i] = segments_of(k.out_type, k.steps, shapes[i]);
            if (!seg[i].starts(step)) continue;
            Job& e = one.e[one.count++] = all.e[i];
            e.src1 = e.src2 = BUF_X;
            e.dst = BUF_A;
        }
        arg.use_rho = exact && step == 0;
        if (one.count) {
            const int64_t n = workgroups(one, GRAM);
            arg.alpha[0] = sc.a / (sc.x * sc.x);
            if (arg.use_rho)
                FC3D_LAUNCH("ns_gram", (ns_product_kernel<GRAM, 1, 1, kMaxItems, NoIos>), dim3((unsigned)n), dim3(256), 0, k.s,
                            one, NoIos{}, arg);
            else
                FC3D_LAUNCH("ns_gram", (ns_product_kernel<GRAM, 2, 2, kMaxItems, NoIos>), dim3((unsigned)n), dim3(256), 0, k.s,
                            one, NoIos{}, arg);
        }
        // Q = a I + b A + c A A; the first of a segment is its running product too
        one.count = 0;
        for (int i = 0; i < count; ++i) {
            Job& e = one.e[one.count++] = all.e[i];
            e.src1 = e.src2 = BUF_A;
            q[i] = e.dst = seg[i].starts(step) ? BUF_P0 : BUF_Q;
            if (seg[i].starts(step)) p[i] = BUF_P0;
        }
        const int64_t n = workgroups(one, POLY);
        arg.alpha[0] = (float)k.c * sc.q / (sc.a * sc.a);
        arg.a = (float)k.a * sc.q;
        arg.b = (float)k.b * sc.q / sc.a;
        FC3D_LAUNCH("ns_poly", (ns_product_kernel<POLY, 2, 2, kMaxItems, NoIos>), dim3((unsigned)n), dim3(256), 0, k.s, one,
                    NoIos{}, arg);
        // R = A Q where the segment goes on, P := P Q where it did not start here
        Jobs<kMaxJobs> two = {};
        for (int i = 0; i < count; ++i) {
            if (!seg[i].ends(step, k.steps)) {
                Job& e = two.e[two.count++] = all.e[i];
                e.src1 = BUF_A;
                e.src2 = q[i];
                e.dst = BUF_R;
                e.op = 0;
            }
            if (!seg[i].starts(step)) {
                Job& e = two.e[two.count++] = all.e[i];
                e.src1 = p[i];
                e.src2 = q[i];
                e.dst = p[i] = p[i] == BUF_P0 ? BUF_P1 : BUF_P0;
                e.op = 1;
            }
        }
        if (two.count) {
            const int64_t groups = workgroups(two, MUL);
            arg.alpha[0] = sc.r / (sc.a * sc.q);
            arg.alpha[1] = 1.0f / sc.q;
            FC3D_LAUNCH("ns_mul", (ns_product_kernel<MUL, 2, 2, kMaxJobs, NoIos>), dim3((unsigned)groups), dim3(256), 0, k.s, two,
                        NoIos{}, arg);
        }
        // A := R Q
        one.count = 0;
        for (int i = 0; i < count; ++i) {
            if (seg[i].ends(step, k.steps)) continue;
            Job& e = one.e[one.count++] = all.e[i];
            e.src1 = BUF_R;
            e.src2 = q[i];
            e.dst = BUF_A;
        }
        if (one.count) {
            const int64_t groups = workgroups(one, MUL);
            arg.alpha[0] = sc.a / (sc.r * sc.q);
            FC3D_LAUNCH("ns_mul", (ns_product_kernel<MUL, 2, 2, kMaxItems, NoIos>), dim3((unsigned)groups), dim3(256), 0, k.s, one,
                        NoIos{}, arg);
        }
        // X := P X where a segment ends, to the tensors behind the last one
        one.count = 0;
        Ios to = {};
        for (int i = 0; i < count; ++i) {
            if (!seg[i].ends(step, k.steps)) continue;
            to.e[one.count] = io.e[i];
            Job& e = one.e[one.count++] = all.e[i];
            e.src1 = p[i];
            e.src2 = xt[i];
            e.dst = xt[i] = xt[i] == BUF_XT0 ? BUF_XT1 : BUF_XT0;
        }
        if (one.count) {
            const int64_t groups = workgroups(one, APPLY);
            arg.last = step == k.steps - 1;
            arg.use_rho = exact && step < 5;          // the first segment of 16-bit results
            arg.alpha[0] = (arg.last ? 1.0f : sc.x) / (sc.q * sc.x);
            if (arg.use_rho)
                FC3D_LAUNCH("ns_apply", (ns_product_kernel<APPLY, 2, 1, kMaxItems, Ios>), dim3((unsigned)groups), dim3(256), 0, k.s,
                            one, to, arg);
            else
                FC3D_LAUNCH("ns_apply", (ns_product_kernel<APPLY, 2, 2, kMaxItems, Ios>), dim3((unsigned)groups), dim3(256), 0, k.s,
                            one, to, arg);
        }
    }
    return FC3D_OK;
}

bool known_type(int t) { return t >= FC3D_F32 && t <= FC3D_F16; }
bool off_align(const void* p, int type) { return (reinterpret_cast<uintptr_t>(p) & (type == FC3D_F32 ? 3u : 1u)) != 0; }

// Matrices in groups of kMaxItems, one group after the other in the same workspace.  `run`: false only sizes it.
int walk(const Call& k, bool run, size_t& bytes) {
    bytes = 0;
    Shape shapes[kMaxItems];
    Scales sc = {};
    if (run) {
        const int longest = k.out_type == FC3D_F32 ? 3 : 5;
        if (!scales_of(k, k.steps < longest ? k.steps : longest, sc)) return FC3D_ERANGE;
    }
    for (int from = 0; from < k.count; from += kMaxItems) {
        const int count = k.count - from < kMaxItems ? k.count - from : kMaxItems;
        int64_t parts = 0, halves = 0, tiles = 0;
        for (int i = 0; i < count; ++i) {
            if (!shape_of(k.rows[from + i], k.cols[from + i], shapes[i])) return FC3D_ERANGE;
            if (shapes[i].m == 0) return FC3D_EINVAL;
            parts += shapes[i].parts();
            halves += shapes[i].halves();
            tiles += shapes[i].mp / kTile * (shapes[i].np / kTile);
        }
        if (tiles >= (1 << 23) || parts >= (1 << 23)) return FC3D_ERANGE;      // workgroups of one launch
        const size_t need = (size_t)(head_bytes(parts) + halves * 2);
        if (need > bytes) bytes = need;
        if (run)
            if (const int rc = run_group(k, from, count, shapes, sc)) return rc;
    }
    return FC3D_OK;
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
    Scales sc;
    if (!scales_of(k, k.steps < 5 ? k.steps : 5, sc)) return FC3D_ERANGE;
    size_t bytes;
    return walk(k, false, bytes);
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
    return walk(k, false, bytes) == FC3D_OK ? bytes : 0;
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
    size_t bytes;
    return walk(k, true, bytes);
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
    size_t bytes;
    return walk(k, true, bytes);
}
