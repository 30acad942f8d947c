// Layer norm, forward and backward, for activations held in 32 or 16 bits.
//
//   y = act((x - mu) r w + b),   mu = mean_c x,   r = 1 / sqrt(mean_c (x - mu)^2 + eps)
//
// over `channels` values of each position; act is the identity or max(., 0).  With g = dy where the activation
// passes it and h = (x - mu) r:
//
//   dx = r (g w - mean_c(g w) - h mean_c(g w h)),   dw = sum_positions g h,   db = sum_positions g.
//
// Two memory orders: "rows" (the normalised axis is contiguous: inner == 1) and "planes" (a channel's positions are
// contiguous, the channels of one position lie `inner` values apart: images with the channel axis before the
// spatial ones).  Both are bound by memory: a value is read once, kept in registers while its position's
// statistics are formed (mean first, then the squares of the differences: no cancellation), and written once.
// Statistics, sums over positions and all arithmetic are 32 bits; a 16-bit result is rounded once, at its store.
// Sums over positions are kept per workgroup, written as partial sums and added in a fixed order by a second,
// small launch: no atomics, the same bits on every run.  A single workgroup's sums are the gradients.
#include "fc3d_common.h"

#include <type_traits>

namespace fc3d {
namespace {

typedef __bf16 bf16;
typedef _Float16 f16;

constexpr int kVec = 4;              // planes: values of one vector access (16 bytes of fp32, 8 of a 16-bit type)

template <typename T, int V>
struct Vec {
    T e[V];
};
template <int BYTES, int ALIGN>
struct Word;
template <>
struct Word<16, 4> {
    typedef uint32_t type __attribute__((ext_vector_type(4), aligned(4)));
};
template <>
struct Word<16, 2> {
    typedef uint32_t type __attribute__((ext_vector_type(4), aligned(2)));
};
template <>
struct Word<8, 2> {
    typedef uint32_t type __attribute__((ext_vector_type(2), aligned(2)));
};
// Vector accesses at the element's own alignment: rows of odd length and planes of odd size start anywhere, and
// global loads and stores take any address on this chip.
template <typename T, int V>
__device__ __forceinline__ Vec<T, V> ldv(const T* p) {
    Vec<T, V> r;
    if constexpr (V == 1) {
        r.e[0] = *p;
    } else {
        typedef typename Word<V * sizeof(T), sizeof(T)>::type word;
        const word w = *reinterpret_cast<const word*>(p);
        __builtin_memcpy(&r, &w, sizeof(r));
    }
    return r;
}
template <typename T, int V>
__device__ __forceinline__ void stv(T* p, const Vec<T, V>& v) {
    if constexpr (V == 1) {
        *p = v.e[0];
    } else {
        typedef typename Word<V * sizeof(T), sizeof(T)>::type word;
        word w;
        __builtin_memcpy(&w, &v, sizeof(v));
        *reinterpret_cast<word*>(p) = w;
    }
}
// The first n of V values (n <= 0: none); the rest reads as zero.
template <typename T, int V>
__device__ __forceinline__ Vec<T, V> ldv_n(const T* p, int n) {
    if (n >= V) return ldv<T, V>(p);
    Vec<T, V> r;
#pragma unroll
    for (int j = 0; j < V; ++j) r.e[j] = (T)0.0f;
#pragma unroll
    for (int j = 0; j < V; ++j)
        if (j < n) r.e[j] = p[j];
    return r;
}
template <typename T, int V>
__device__ __forceinline__ void stv_n(T* p, const Vec<T, V>& v, int n) {
    if (n >= V) {
        stv<T, V>(p, v);
        return;
    }
#pragma unroll
    for (int j = 0; j < V; ++j)
        if (j < n) p[j] = v.e[j];
}

// The same 16 bytes, of which the compiler knows nothing: what it has computed from them before does not count
template <typename T, int V>
__device__ __forceinline__ Vec<T, V> unknown(const Vec<T, V>& v) {
    typedef uint32_t word __attribute__((ext_vector_type(sizeof(v) / 4)));
    word w;
    __builtin_memcpy(&w, &v, sizeof(v));
    asm volatile("" : "+v"(w));
    Vec<T, V> r;
    __builtin_memcpy(&r, &w, sizeof(v));
    return r;
}

// A weight or bias: fp32 or the activations' 16-bit type (the same branch in every lane), `absent` without one
template <typename T>
__device__ __forceinline__ float param(const void* p, bool f32, long i, float absent) {
    if (!p) return absent;
    return f32 ? static_cast<const float*>(p)[i] : (float)static_cast<const T*>(p)[i];
}
__device__ __forceinline__ void put_param(void* p, int type, long i, float v) {
    if (type == FC3D_F32) static_cast<float*>(p)[i] = v;
    else if (type == FC3D_BF16) static_cast<bf16*>(p)[i] = (bf16)v;
    else static_cast<f16*>(p)[i] = (f16)v;
}

// Whether max(pre, 0) hands pre on; a NaN passes, in both directions
__device__ __forceinline__ bool passes(float pre) { return !(pre <= 0.0f); }

// N sums over the LPR lanes that share a row, the same bits in every lane.  Above one wavefront the wavefronts' sums
// meet in LDS; `slot` alternates between two areas, so that one barrier for all of them is enough.
template <int LPR, int BLOCK, int N>
__device__ __forceinline__ void group_sums(float (&v)[N], float* red, int slot) {
#pragma unroll
    for (int o = (LPR < 64 ? LPR : 64) / 2; o > 0; o >>= 1)
#pragma unroll
        for (int n = 0; n < N; ++n) v[n] += __shfl_xor(v[n], o, 64);
    if constexpr (LPR > 64) {
        float* a = red + slot * (BLOCK / 64) * N;
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int n = 0; n < N; ++n) a[(threadIdx.x >> 6) * N + n] = v[n];
        __syncthreads();
        a += threadIdx.x / LPR * (LPR / 64) * N;
#pragma unroll
        for (int n = 0; n < N; ++n) {
            v[n] = a[n];
#pragma unroll
            for (int i = 1; i < LPR / 64; ++i) v[n] += a[i * N + n];
        }
    }
}
template <int LPR, int BLOCK>
__device__ __forceinline__ float group_sum(float v, float* red, int slot) {
    float one[1] = {v};
    group_sums<LPR, BLOCK>(one, red, slot);
    return one[0];
}

// ---- rows -------------------------------------------------------------------------------------------------
// LPR lanes per row, E values each (vectors of 16 bytes, lane after lane); a workgroup takes rows
// blockIdx.x * (BLOCK / LPR) + k * gridDim.x * ..., its lanes keep their columns' weights.  The next row is loaded before
// the sums of the current one are formed, which would leave the memory idle otherwise (not with 1024 lanes per row, which
// have 128 registers: 4096 x 8192 fp32 44 us, 54 with the next row ahead).
template <typename T, int LPR, int E>
struct Row {
    static constexpr int V = 16 / sizeof(T), NV = E / V;
    Vec<T, V> v[NV];

    // even: the row is whole vectors.  A branch of lanes around a load makes its wait part of the branch, one load after the
    // other; so the lanes behind the row's end read its first values and put them away (backward, bf16, 32768 x 1024 46 ->
    // 39 us, 16384 x 2048 49 -> 44; fp32 81 -> 77).
    __device__ __forceinline__ void load(const T* row, int lane, int C, bool even) {
        if (even) {
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                const int c0 = (lane + k * LPR) * V;
                v[k] = ldv<T, V>(row + (c0 < C ? c0 : 0));
            }
#pragma unroll
            for (int k = 0; k < NV; ++k)
                if ((lane + k * LPR) * V >= C) v[k] = Vec<T, V>{};
        } else {
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                const int c0 = (lane + k * LPR) * V;
                v[k] = ldv_n<T, V>(row + (c0 < C ? c0 : 0), C - c0);
            }
        }
    }
    __device__ __forceinline__ void store(T* row, int lane, int C, bool even) const {
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int c0 = (lane + k * LPR) * V;
            if (c0 >= C) continue;
            if (even) stv<T, V>(row + c0, v[k]);
            else stv_n<T, V>(row + c0, v[k], C - c0);
        }
    }
};

// The weights or biases of a lane's columns, in whole vectors
template <typename T, int LPR, int E>
__device__ __forceinline__ void row_params(const void* p, bool f32, int lane, int C, float absent, float (&to)[E]) {
    constexpr int V = Row<T, LPR, E>::V, NV = E / V;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int c0 = (lane + k * LPR) * V, at = c0 < C ? c0 : 0;
        if (!p) {
#pragma unroll
            for (int j = 0; j < V; ++j) to[k * V + j] = absent;
        } else if (f32) {
#pragma unroll
            for (int h = 0; h < V; h += 4) {
                const Vec<float, 4> v = ldv_n<float, 4>(static_cast<const float*>(p) + at + (c0 + h < C ? h : 0), C - c0 - h);
#pragma unroll
                for (int j = 0; j < 4; ++j) to[k * V + h + j] = v.e[j];
            }
        } else {
            const Vec<T, V> v = ldv_n<T, V>(static_cast<const T*>(p) + at, C - c0);
#pragma unroll
            for (int j = 0; j < V; ++j) to[k * V + j] = (float)v.e[j];
        }
    }
}

template <typename T, int LPR, int BLOCK, int E>
__global__ __launch_bounds__(BLOCK) void ln_rows_fwd(const T* __restrict__ x, const void* __restrict__ w,
                                                     const void* __restrict__ b, bool w_f32, long rows, int C,
                                                     long x_stride, float eps, int relu, T* __restrict__ y,
                                                     float* __restrict__ mean, float* __restrict__ rstd) {
    constexpr int V = Row<T, LPR, E>::V, NV = E / V, RPB = BLOCK / LPR;
    __shared__ float red[LPR > 64 ? 2 * (BLOCK / 64) : 1];
    const int lane = threadIdx.x % LPR, sub = threadIdx.x / LPR;
    const float fc = (float)C;
    const bool even = C % V == 0;
    const long stride = (long)gridDim.x * RPB;
    long r = (long)blockIdx.x * RPB + sub;
    constexpr bool AHEAD = LPR < 1024 && LPR * E < 16384;
    Row<T, LPR, E> xv, ahead;
    if constexpr (AHEAD) xv.load(x + (r < rows ? r : 0) * x_stride, lane, C, even);
    float wv[E], bv[E];
    row_params<T, LPR, E>(w, w_f32, lane, C, 1.0f, wv);
    row_params<T, LPR, E>(b, w_f32, lane, C, 0.0f, bv);
    // every lane of a workgroup runs the same number of rounds: the sums above one wavefront hold barriers
    for (long r0 = (long)blockIdx.x * RPB; r0 < rows; r0 += stride, r += stride) {
        if constexpr (!AHEAD) xv.load(x + (r < rows ? r : 0) * x_stride, lane, C, even);
        else if (r0 + stride < rows) ahead.load(x + (r + stride < rows ? r + stride : 0) * x_stride, lane, C, even);
        float s = 0.0f;
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int j = 0; j < V; ++j) s += (float)xv.v[k].e[j];
        const float mu = group_sum<LPR, BLOCK>(s, red, 0) / fc;
        s = 0.0f;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int n = C - (lane + k * LPR) * V;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float d = j < n ? (float)xv.v[k].e[j] - mu : 0.0f;
                s = fmaf(d, d, s);
            }
        }
        const float rs = 1.0f / sqrtf(group_sum<LPR, BLOCK>(s, red, 1) / fc + eps);
        if (r < rows) {
#pragma unroll
            for (int k = 0; k < NV; ++k)
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    float v = fmaf(((float)xv.v[k].e[j] - mu) * rs, wv[k * V + j], bv[k * V + j]);
                    if (relu) v = passes(v) ? v : 0.0f;
                    xv.v[k].e[j] = (T)v;
                }
            xv.store(y + r * C, lane, C, even);
            if (mean && lane == 0) {
                mean[r] = mu;
                rstd[r] = rs;
            }
        }
        if constexpr (AHEAD) xv = ahead;
    }
}

// Where a backward launch leaves its sums of g h and of g: [gridDim.x][2][C] partial sums, or, of a single workgroup, the
// gradients themselves.
struct Sums {
    float* partial;
    void *dw, *db;        // either may be NULL, both are when no parameter asks for a gradient
    int type;
    __host__ __device__ __forceinline__ bool wanted() const { return dw || db; }
    __device__ __forceinline__ void put(int which, long C, long c, float v) const {
        if (gridDim.x > 1) partial[((long)blockIdx.x * 2 + which) * C + c] = v;
        else if (which ? db : dw) put_param(which ? db : dw, type, c, v);
    }
};

template <typename T, int LPR, int BLOCK, int E>
__global__ __launch_bounds__(BLOCK) void ln_rows_bwd(const T* __restrict__ dy, const T* __restrict__ x,
                                                     const void* __restrict__ w, const void* __restrict__ b, bool w_f32,
                                                     const float* __restrict__ mean, const float* __restrict__ rstd,
                                                     long rows, int C, long dy_stride, long x_stride, int relu,
                                                     T* __restrict__ dx, Sums sums) {
    constexpr int V = Row<T, LPR, E>::V, NV = E / V, RPB = BLOCK / LPR;
    __shared__ float red[LPR > 64 ? 4 * (BLOCK / 64) : 1];
    __shared__ float cols[RPB > 1 ? BLOCK * E : 1];
    const int lane = threadIdx.x % LPR, sub = threadIdx.x / LPR;
    const float fc = (float)C;
    const bool even = C % V == 0;
    const long stride = (long)gridDim.x * RPB;
    long r = (long)blockIdx.x * RPB + sub;
    constexpr bool AHEAD = LPR < 1024 && LPR * E < 16384;
    Row<T, LPR, E> xv, gv, next_x, next_g;
    float mu = 0.0f, rs = 0.0f;
    const auto load = [&](long r, Row<T, LPR, E>& xr, Row<T, LPR, E>& gr, float& m, float& s) {
        r = r < rows ? r : 0;
        xr.load(x + r * x_stride, lane, C, even);
        gr.load(dy + r * dy_stride, lane, C, even);
        m = mean[r];
        s = rstd[r];
    };
    if constexpr (AHEAD) load(r, xv, gv, mu, rs);
    float wv[E], aw[E], ab[E];
    row_params<T, LPR, E>(w, w_f32, lane, C, 1.0f, wv);
#pragma unroll
    for (int i = 0; i < E; ++i) {
        aw[i] = 0.0f;
        ab[i] = 0.0f;
    }
    int turn = 0;
    for (long r0 = (long)blockIdx.x * RPB; r0 < rows; r0 += stride, r += stride, turn ^= 1) {
        const bool live = r < rows;
        float next_mu = 0.0f, next_rs = 0.0f;
        if constexpr (!AHEAD) load(r, xv, gv, mu, rs);
        else if (r0 + stride < rows) load(r + stride, next_x, next_g, next_mu, next_rs);
        float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int n = live ? C - (lane + k * LPR) * V : 0;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const int i = k * V + j;
                const float h = ((float)xv.v[k].e[j] - mu) * rs;
                float g = (float)gv.v[k].e[j];
                if (relu) {                                   // (the biases are read again: they would cost a register each)
                    const int c = (lane + k * LPR) * V + j;
                    g = passes(fmaf(h, wv[i], c < C ? param<T>(b, w_f32, c, 0.0f) : 0.0f)) ? g : 0.0f;
                    gv.v[k].e[j] = (T)g;
                }
                if (j < n) {
                    const float gw = g * wv[i];
                    s1 += gw;
                    s2 = fmaf(gw, h, s2);
                    aw[i] = fmaf(g, h, aw[i]);
                    ab[i] += g;
                }
            }
        }
        float both[2] = {s1, s2};
        group_sums<LPR, BLOCK>(both, red, turn);
        const float m1 = both[0] / fc, m2 = both[1] / fc;
        if constexpr (sizeof(T) == 2 && LPR * E >= 16384) {   // to be unpacked again below: kept as fp32 it would not fit
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                xv.v[k] = unknown(xv.v[k]);
                gv.v[k] = unknown(gv.v[k]);
            }
        }
        if (live && dx) {
#pragma unroll
            for (int k = 0; k < NV; ++k)
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float h = ((float)xv.v[k].e[j] - mu) * rs;
                    xv.v[k].e[j] = (T)(rs * (fmaf((float)gv.v[k].e[j], wv[k * V + j], -m1) - h * m2));
                }
            xv.store(dx + r * C, lane, C, even);
        }
        if constexpr (AHEAD) {
            xv = next_x;
            gv = next_g;
            mu = next_mu;
            rs = next_rs;
        }
    }
    if (!sums.wanted()) return;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        float* a = which ? ab : aw;
        if constexpr (RPB > 1) {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < E; ++i) cols[(sub * E + i) * LPR + lane] = a[i];
            __syncthreads();
            for (int t = threadIdx.x; t < LPR * E; t += BLOCK) {
                float s = 0.0f;
#pragma unroll 4
                for (int q = 0; q < RPB; ++q) s += cols[q * E * LPR + t];
                const int i = t / LPR, c = (t % LPR + (i / V) * LPR) * V + i % V;
                if (c < C) sums.put(which, C, c, s);
            }
        } else {
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                const int c0 = (lane + k * LPR) * V;
#pragma unroll
                for (int j = 0; j < V; ++j)
                    if (c0 + j < C) sums.put(which, C, c0 + j, a[k * V + j]);
            }
        }
    }
}

// ---- planes -----------------------------------------------------------------------------------------------
// A workgroup is CL channel groups x PL positions; a lane holds E channels (cg, cg + CL, ...) of V neighbouring
// positions.  Lanes next to each other take neighbouring positions, so every load covers PL * V * sizeof(T)
// contiguous bytes of one channel.  Positions are counted in vectors over the whole batch (q = image * nvec + vector).
template <int CL, int PL>
constexpr int channel_groups() {      // sums that are left after the lanes of a wavefront have added theirs
    return PL >= 64 ? CL : CL > 64 / PL ? CL / (64 / PL) : 1;
}
template <int CL, int PL, int V>
__device__ __forceinline__ void channel_sums(float (&s)[V], float* red) {
    if constexpr (CL > 1) {
        const int pl = threadIdx.x % PL, cg = threadIdx.x / PL;
        constexpr int NG = channel_groups<CL, PL>(), GW = CL / NG;
#pragma unroll
        for (int o = PL; o < PL * GW; o <<= 1)
#pragma unroll
            for (int v = 0; v < V; ++v) s[v] += __shfl_xor(s[v], o, 64);
        if constexpr (NG > 1) {
            __syncthreads();                                  // the readers of the last sums are through
            if (cg % GW == 0)
#pragma unroll
                for (int v = 0; v < V; ++v) red[((cg / GW) * V + v) * PL + pl] = s[v];
            __syncthreads();
#pragma unroll
            for (int v = 0; v < V; ++v) {
                float a = red[v * PL + pl];
#pragma unroll
                for (int g = 1; g < NG; ++g) a += red[(g * V + v) * PL + pl];
                s[v] = a;
            }
        }
    }
}

// A lane's channels at n of V positions (n < V: the end of a plane).  A branch around a load of 16-bit values makes its wait
// part of the branch, one load after the other: there one branch goes around all of them, and channels behind the last
// read the first and are put away (32 x 64 x 65536 bf16: forward 152 -> 120 us, backward 271 -> 208).  fp32 values arrive in
// the registers that hold them and are faster with a branch each (224 against 235 us), or, backward with 8 channels a lane,
// with one branch around all and one per channel (322 against 332 and 353).
template <typename T, int V, int CL, int E, bool BWD>
__device__ __forceinline__ void plane_load(const T* p, int cg, int C, long inner, int n, Vec<T, V> (&to)[E]) {
    if constexpr (sizeof(T) == 4 && !(BWD && E == 8)) {
#pragma unroll
        for (int k = 0; k < E; ++k) {
            const int c = cg + k * CL;
            to[k] = ldv_n<T, V>(p + (c < C ? c : 0) * inner, c < C ? n : 0);
        }
        return;
    }
    if (n >= V) {
#pragma unroll
        for (int k = 0; k < E; ++k) {
            const int c = cg + k * CL;
            to[k] = Vec<T, V>{};
            if (sizeof(T) == 2 || c < C) to[k] = ldv<T, V>(p + (c < C ? c : 0) * inner);
        }
    } else {
#pragma unroll
        for (int k = 0; k < E; ++k) {
            const int c = cg + k * CL;
            to[k] = ldv_n<T, V>(p + (c < C ? c : 0) * inner, c < C ? n : 0);
        }
    }
    if (sizeof(T) == 2 && C < CL * E)
#pragma unroll
        for (int k = 0; k < E; ++k)
            if (cg + k * CL >= C) to[k] = Vec<T, V>{};
}
template <typename T, int V, int CL, int E>
__device__ __forceinline__ void plane_store(T* p, int cg, int C, long inner, int n, const Vec<T, V> (&v)[E]) {
    if (sizeof(T) == 2 && n >= V) {
#pragma unroll
        for (int k = 0; k < E; ++k)
            if (cg + k * CL < C) stv<T, V>(p + (cg + k * CL) * inner, v[k]);
    } else {
#pragma unroll
        for (int k = 0; k < E; ++k)
            if (cg + k * CL < C) stv_n<T, V>(p + (cg + k * CL) * inner, v[k], n);
    }
}

template <typename T, int V, int CL, int PL, int E>
__global__ __launch_bounds__(CL* PL) void ln_planes_fwd(const T* __restrict__ x, const void* __restrict__ w, const void* __restrict__ b, bool w_f32, unsigned nq, unsigned nvec, int C,
                                                        long inner, long x_stride, float eps, int relu, T* __restrict__ y,
                                                        float* __restrict__ mean, float* __restrict__ rstd) {
    __shared__ float red[CL > 1 ? channel_groups<CL, PL>() * PL * V : 1];
    const int pl = threadIdx.x % PL, cg = threadIdx.x / PL;
    const float fc = (float)C;
    float wv[E], bv[E];
#pragma unroll
    for (int k = 0; k < E; ++k) {
        const int c = cg + k * CL;
        wv[k] = c < C ? param<T>(w, w_f32, c, 1.0f) : 0.0f;
        bv[k] = c < C ? param<T>(b, w_f32, c, 0.0f) : 0.0f;
    }
    for (unsigned long q0 = (unsigned long)blockIdx.x * PL; q0 < nq; q0 += (unsigned long)gridDim.x * PL) {
        const bool live = q0 + pl < nq;
        const unsigned q = live ? (unsigned)(q0 + pl) : 0u;
        const unsigned img = q / nvec;
        const long p = (long)(q - img * nvec) * V;
        const int n = live ? (int)(inner - p < V ? inner - p : V) : 0;
        const T* xp = x + (long)img * x_stride + p;
        Vec<T, V> xv[E];
        plane_load<T, V, CL, E, false>(xp, cg, C, inner, n, xv);
        float mu[V], rs[V];
#pragma unroll
        for (int v = 0; v < V; ++v) {
            mu[v] = 0.0f;
#pragma unroll
            for (int k = 0; k < E; ++k) mu[v] += (float)xv[k].e[v];
        }
        channel_sums<CL, PL, V>(mu, red);
#pragma unroll
        for (int v = 0; v < V; ++v) {
            mu[v] /= fc;
            rs[v] = 0.0f;
#pragma unroll
            for (int k = 0; k < E; ++k) {
                const float d = cg + k * CL < C ? (float)xv[k].e[v] - mu[v] : 0.0f;
                rs[v] = fmaf(d, d, rs[v]);
            }
        }
        channel_sums<CL, PL, V>(rs, red);
#pragma unroll
        for (int v = 0; v < V; ++v) rs[v] = 1.0f / sqrtf(rs[v] / fc + eps);
#pragma unroll
        for (int k = 0; k < E; ++k)
#pragma unroll
            for (int v = 0; v < V; ++v) {
                float a = fmaf(((float)xv[k].e[v] - mu[v]) * rs[v], wv[k], bv[k]);
                if (relu) a = passes(a) ? a : 0.0f;
                xv[k].e[v] = (T)a;
            }
        plane_store<T, V, CL, E>(y + (long)img * inner * C + p, cg, C, inner, n, xv);
        if (mean && cg == 0) {
#pragma unroll
            for (int v = 0; v < V; ++v)
                if (v < n) {
                    mean[(long)img * inner + p + v] = mu[v];
                    rstd[(long)img * inner + p + v] = rs[v];
                }
        }
    }
}

template <typename T, int V, int CL, int PL, int E>
__global__ __launch_bounds__(CL* PL) void ln_planes_bwd(const T* __restrict__ dy, const T* __restrict__ x,
                                                        const void* __restrict__ w, const void* __restrict__ b, bool w_f32,
                                                        const float* __restrict__ mean, const float* __restrict__ rstd,
                                                        unsigned nq, unsigned nvec, int C, long inner, long dy_stride,
                                                        long x_stride, int relu, T* __restrict__ dx, Sums out) {
    __shared__ float red[CL > 1 ? channel_groups<CL, PL>() * PL * 2 * V : 1];
    __shared__ float wave_part[PL > 64 ? CL * (PL / 64) * E : 1];
    const int pl = threadIdx.x % PL, cg = threadIdx.x / PL;
    const float fc = (float)C;
    float wv[E], aw[E], ab[E];
#pragma unroll
    for (int k = 0; k < E; ++k) {
        const int c = cg + k * CL;
        wv[k] = c < C ? param<T>(w, w_f32, c, 1.0f) : 0.0f;
        aw[k] = 0.0f;
        ab[k] = 0.0f;
    }
    for (unsigned long q0 = (unsigned long)blockIdx.x * PL; q0 < nq; q0 += (unsigned long)gridDim.x * PL) {
        const bool live = q0 + pl < nq;
        const unsigned q = live ? (unsigned)(q0 + pl) : 0u;
        const unsigned img = q / nvec;
        const long p = (long)(q - img * nvec) * V;
        const int n = live ? (int)(inner - p < V ? inner - p : V) : 0;
        const T* xp = x + (long)img * x_stride + p;
        const T* gp = dy + (long)img * dy_stride + p;
        Vec<T, V> xv[E], gv[E];
        plane_load<T, V, CL, E, true>(xp, cg, C, inner, n, xv);
        plane_load<T, V, CL, E, true>(gp, cg, C, inner, n, gv);
        float mu[V], rs[V], sums[2 * V];                      // of g w, then of g w h
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const long at = (long)img * inner + p + (v < n ? v : 0);
            mu[v] = mean[at];
            rs[v] = rstd[at];
            sums[v] = 0.0f;
            sums[V + v] = 0.0f;
        }
#pragma unroll
        for (int k = 0; k < E; ++k) {
            const bool on = cg + k * CL < C;
            const float bias = relu && on ? param<T>(b, w_f32, cg + k * CL, 0.0f) : 0.0f;
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const float h = ((float)xv[k].e[v] - mu[v]) * rs[v];
                float g = (float)gv[k].e[v];
                if (relu) {
                    g = passes(fmaf(h, wv[k], bias)) ? g : 0.0f;
                    gv[k].e[v] = (T)g;
                }
                if (on && v < n) {
                    const float gw = g * wv[k];
                    sums[v] += gw;
                    sums[V + v] = fmaf(gw, h, sums[V + v]);
                    aw[k] = fmaf(g, h, aw[k]);
                    ab[k] += g;
                }
            }
        }
        channel_sums<CL, PL, 2 * V>(sums, red);
        if (dx) {
#pragma unroll
            for (int v = 0; v < 2 * V; ++v) sums[v] /= fc;
#pragma unroll
            for (int k = 0; k < E; ++k)
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    const float h = ((float)xv[k].e[v] - mu[v]) * rs[v];
                    xv[k].e[v] = (T)(rs[v] * (fmaf((float)gv[k].e[v], wv[k], -sums[v]) - h * sums[V + v]));
                }
            plane_store<T, V, CL, E>(dx + (long)img * inner * C + p, cg, C, inner, n, xv);
        }
    }
    if (!out.wanted()) return;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        float* a = which ? ab : aw;
#pragma unroll
        for (int k = 0; k < E; ++k)
#pragma unroll
            for (int o = (PL < 64 ? PL : 64) / 2; o > 0; o >>= 1) a[k] += __shfl_xor(a[k], o, 64);
        if constexpr (PL > 64) {
            constexpr int NW = PL / 64;
            __syncthreads();
            if ((threadIdx.x & 63) == 0)
#pragma unroll
                for (int k = 0; k < E; ++k) wave_part[(cg * NW + pl / 64) * E + k] = a[k];
            __syncthreads();
            for (int t = threadIdx.x; t < CL * E; t += CL * PL) {
                const int g = t / E, k = t % E, c = g + k * CL;
                float s = 0.0f;
#pragma unroll
                for (int i = 0; i < NW; ++i) s += wave_part[(g * NW + i) * E + k];
                if (c < C) out.put(which, C, c, s);
            }
        } else {
            if (pl == 0)
#pragma unroll
                for (int k = 0; k < E; ++k)
                    if (cg + k * CL < C) out.put(which, C, cg + k * CL, a[k]);
        }
    }
}

// ---- channels beyond what a workgroup's registers hold ------------------------------------------------------
// One workgroup per row (rows) or per 16 or 4 positions (planes), the values read once per sum and once for the
// result; the repeats come from the caches.  Loads are unrolled, several in flight: the wait for each would be all of the
// time of a small input.
constexpr int kLongBlock = 1024;

// NP: positions of a workgroup (rows: 1).  The sum over its lanes of the same position, in all of them.
template <int NP>
__device__ __forceinline__ float long_sum(float v, float* red) {
    __syncthreads();
#pragma unroll
    for (int o = NP; o < 64; o <<= 1) v += __shfl_xor(v, o, 64);
    if ((threadIdx.x & 63) < NP) red[(threadIdx.x >> 6) * NP + (threadIdx.x & 63)] = v;
    __syncthreads();
    v = 0.0f;
#pragma unroll
    for (int i = 0; i < kLongBlock / 64; ++i) v += red[i * NP + (threadIdx.x & (NP - 1))];
    return v;
}

template <typename T, int NP>
__global__ __launch_bounds__(kLongBlock) void ln_long_fwd(const T* __restrict__ x, const void* __restrict__ w, const void* __restrict__ b, bool w_f32, long positions, long C, long inner,
                                                          long x_stride, float eps, int relu, T* __restrict__ y,
                                                          float* __restrict__ mean, float* __restrict__ rstd) {
    __shared__ float red[kLongBlock / 64 * NP];
    constexpr int STEP = kLongBlock / NP;
    const int pl = threadIdx.x % NP, c0 = threadIdx.x / NP;
    for (long q0 = (long)blockIdx.x * NP; q0 < positions; q0 += (long)gridDim.x * NP) {
        const bool live = q0 + pl < positions;
        const long q = live ? q0 + pl : q0, img = q / inner, p = q - img * inner;
        const T* xp = x + img * x_stride + p;
        T* yp = y + img * inner * C + p;
        float s = 0.0f;
#pragma unroll 8
        for (long c = c0; c < C; c += STEP) s += (float)xp[c * inner];
        const float mu = long_sum<NP>(s, red) / (float)C;
        s = 0.0f;
#pragma unroll 8
        for (long c = c0; c < C; c += STEP) {
            const float d = (float)xp[c * inner] - mu;
            s = fmaf(d, d, s);
        }
        const float rs = 1.0f / sqrtf(long_sum<NP>(s, red) / (float)C + eps);
        if (live) {
#pragma unroll 8
        for (long c = c0; c < C; c += STEP) {
                float v = fmaf(((float)xp[c * inner] - mu) * rs, param<T>(w, w_f32, c, 1.0f), param<T>(b, w_f32, c, 0.0f));
                if (relu) v = passes(v) ? v : 0.0f;
                yp[c * inner] = (T)v;
            }
            if (mean && c0 == 0) {
                mean[q] = mu;
                rstd[q] = rs;
            }
        }
    }
}

template <typename T, int NP>
__global__ __launch_bounds__(kLongBlock) void ln_long_bwd(const T* __restrict__ dy, const T* __restrict__ x,
                                                          const void* __restrict__ w, const void* __restrict__ b, bool w_f32,
                                                          const float* __restrict__ mean, const float* __restrict__ rstd,
                                                          long positions, long C, long inner, long dy_stride,
                                                          long x_stride, int relu, T* __restrict__ dx) {
    __shared__ float red[kLongBlock / 64 * NP];
    constexpr int STEP = kLongBlock / NP;
    const int pl = threadIdx.x % NP, c0 = threadIdx.x / NP;
    for (long q0 = (long)blockIdx.x * NP; q0 < positions; q0 += (long)gridDim.x * NP) {
        const bool live = q0 + pl < positions;
        const long q = live ? q0 + pl : q0, img = q / inner, p = q - img * inner;
        const T* xp = x + img * x_stride + p;
        const T* gp = dy + img * dy_stride + p;
        const float mu = mean[q], rs = rstd[q];
        float s1 = 0.0f, s2 = 0.0f;
#pragma unroll 8
        for (long c = c0; c < C; c += STEP) {
            const float wc = param<T>(w, w_f32, c, 1.0f), h = ((float)xp[c * inner] - mu) * rs;
            float g = (float)gp[c * inner];
            if (relu) g = passes(fmaf(h, wc, param<T>(b, w_f32, c, 0.0f))) ? g : 0.0f;
            s1 += g * wc;
            s2 = fmaf(g * wc, h, s2);
        }
        const float m1 = long_sum<NP>(s1, red) / (float)C, m2 = long_sum<NP>(s2, red) / (float)C;
        if (live) {
            T* dp = dx + img * inner * C + p;
#pragma unroll 8
        for (long c = c0; c < C; c += STEP) {
                const float wc = param<T>(w, w_f32, c, 1.0f), h = ((float)xp[c * inner] - mu) * rs;
                float g = (float)gp[c * inner];
                if (relu) g = passes(fmaf(h, wc, param<T>(b, w_f32, c, 0.0f))) ? g : 0.0f;
                dp[c * inner] = (T)(rs * (fmaf(g, wc, -m1) - h * m2));
            }
        }
    }
}

// Sums over positions for the same case: a workgroup takes one share of the positions (blockIdx.y of gridDim.y) and 256
// channels (rows: a lane per channel) or four (planes: a wavefront per channel, a lane per position).
template <typename T, bool PLANES>
__global__ __launch_bounds__(256) void ln_long_params(const T* __restrict__ dy, const T* __restrict__ x,
                                                      const void* __restrict__ w, const void* __restrict__ b, bool w_f32,
                                                      const float* __restrict__ mean, const float* __restrict__ rstd,
                                                      long positions, long C, long inner, long dy_stride, long x_stride,
                                                      int relu, float* __restrict__ partial) {
    const long c = PLANES ? (long)blockIdx.x * 4 + (threadIdx.x >> 6) : (long)blockIdx.x * 256 + threadIdx.x;
    const long share = (positions + gridDim.y - 1) / gridDim.y;
    const long lo = (long)blockIdx.y * share, hi = lo + share < positions ? lo + share : positions;
    if (c >= C) return;
    float sw = 0.0f, sb = 0.0f;
    const float wc = param<T>(w, w_f32, c, 1.0f), bc = param<T>(b, w_f32, c, 0.0f);
#pragma unroll 4
    for (long q = lo + (PLANES ? (threadIdx.x & 63) : 0); q < hi; q += PLANES ? 64 : 1) {
        const long img = PLANES ? (long)((unsigned)q / (unsigned)inner) : q, p = PLANES ? q - img * inner : 0;
        const float h = ((float)x[img * x_stride + c * inner + p] - mean[q]) * rstd[q];
        float g = (float)dy[img * dy_stride + c * inner + p];
        if (relu) g = passes(fmaf(h, wc, bc)) ? g : 0.0f;
        sw = fmaf(g, h, sw);
        sb += g;
    }
    float* pw = partial + (long)blockIdx.y * 2 * C;
    if constexpr (PLANES) {
        sw = wave_sum(sw);
        sb = wave_sum(sb);
        if ((threadIdx.x & 63) > 0) return;
    }
    pw[c] = sw;
    pw[C + c] = sb;
}

// dw, db = sums of the n partial sums, 32 columns per workgroup and n shared out over 32 lanes of each
__global__ __launch_bounds__(1024) void ln_params_sum(const float* __restrict__ partial, int n, long C, int type,
                                                      void* __restrict__ dw, void* __restrict__ db) {
    __shared__ float red[32][33];
    const int col = threadIdx.x & 31, part = threadIdx.x >> 5;
    const long at = (long)blockIdx.x * 32 + col;                  // over [2][C]
    float s = 0.0f;
    if (at < 2 * C) {
#pragma unroll 8
        for (int i = part; i < n; i += 32) s += partial[(long)i * 2 * C + at];
    }
    red[part][col] = s;
    __syncthreads();
    if (part == 0 && at < 2 * C) {
        s = red[0][col];
#pragma unroll
        for (int i = 1; i < 32; ++i) s += red[i][col];
        if (at < C) {
            if (dw) put_param(dw, type, at, s);
        } else if (db) {
            put_param(db, type, at - C, s);
        }
    }
}

// ---- which kernel, how many workgroups ----------------------------------------------------------------------
constexpr int kRowsMax = 16 * 1024;               // rows: the widest that 1024 lanes of 16 values hold
constexpr int kPlanesMax = 1024;                  // planes: 128 channel groups of 8

// Workgroups of a launch that loops over its positions.  A backward launch leaves one row of partial sums per
// workgroup, which the second launch reads: no more of them than the compute units hold at a time.
constexpr long kRowsFwd = 1280, kRowsBwd = 512, kPlanesFwd = 1024, kPlanesBwd = 512, kLong = 4096;

struct Plan {
    bool rows, wide;      // wide: vectors along the positions (planes)
    bool fits;            // the register kernels hold a position's channels
    int lanes;            // rows: lanes per row; planes: channel groups
    int beside;           // rows, positions or vectors of positions of one workgroup
    int each;             // values (rows) or channels (planes) of a lane
    long units, most;     // workgroups that the positions fill once, and of a launch
    int64_t positions;
};

int elem_size(int type) { return type == FC3D_F32 ? 4 : 2; }

// What a lane holds and how many lanes share a position.  Rows, forward: 16 values a lane.  Rows, backward: 8, so that four
// or five wavefronts a SIMD hide each other's waits instead of three (16384 x 2048 bf16 54 -> 49 us, 8192 x 4096 87 -> 56);
// beyond 8192 values 512 lanes take 32, with twice the registers of 1024 lanes that take 16 (2048 x 16000 fp32 138 -> 116,
// bf16 129 -> 100 us).  Planes, forward: 8 channels.  Planes, backward, the fastest of 4 and 8
// channels a lane and of 128 to 1024 lanes: 16 x 128 x 16384 bf16 51 us with 4 on 512 lanes, 66 on 256; 32 x 64 x 65536 fp32
// 324 with 8, 356 with 4; 512 channels: fp32 46 with 4 on 1024 lanes, 47 with 8 on 512, bf16 50 and 47.
Plan plan_of(bool fwd, int type, int64_t outer, int64_t C, int64_t inner) {
    Plan p = {};
    p.rows = inner == 1;
    p.positions = outer * inner;
    const auto take = [&](int lanes, int beside, int each, long most) {
        p.lanes = lanes;
        p.beside = beside;
        p.each = each;
        p.most = most;
    };
    if (p.rows) {
        p.fits = C <= kRowsMax;
        const int block = fwd ? 256 : 512;
        if (C <= 64) take(8, block / 8, 8, 0);
        else if (C > 8192) take(fwd ? 1024 : 512, 1, fwd ? 16 : 32, 0);
        else if (C > 4096) take(1024, 1, 8, 0);
        else {
            int lanes = fwd ? 8 : 16;
            while (lanes * (fwd ? 16 : 8) < C) lanes *= 2;
            take(lanes, block / lanes, fwd ? 16 : 8, 0);
        }
        p.most = fwd ? kRowsFwd : kRowsBwd;
        p.units = p.fits ? (outer + p.beside - 1) / p.beside : outer;
    } else {
        p.fits = C <= kPlanesMax;
        // a plane that is no multiple of the vector leaves part of its last vector empty: single values where that
        // would idle a quarter of the lanes
        const int64_t nv = (inner + kVec - 1) / kVec;
        p.wide = inner * 4 >= nv * kVec * 3;
        if (fwd) {
            const int cl = C <= 8 ? 1 : C <= 32 ? 4 : C <= 64 ? 8 : C <= 128 ? 16 : C <= 256 ? 32 : C <= 512 ? 64 : 128;
            take(cl, cl <= 32 ? 256 / cl : cl == 64 ? 8 : 4, 8, kPlanesFwd);
        } else if (C <= 32) take(C <= 8 ? 2 : 8, C <= 8 ? 128 : 32, 4, 2 * kPlanesBwd);
        else if (C <= 64) take(8, 32, 8, kPlanesBwd);
        else if (C <= 128) take(32, 16, 4, kPlanesBwd);
        else if (C <= 256) take(64, 8, 4, kPlanesBwd);
        else if (C <= 512) type == FC3D_F32 ? take(128, 8, 4, kPlanesBwd) : take(64, 8, 8, kPlanesBwd);
        else take(128, 4, 8, kPlanesBwd);
        const int64_t nq = p.wide ? outer * nv : outer * inner;
        // beyond the registers: 16 positions fill the pieces that memory is read in (4 x 4096 x 1024 fp32 70 us, 277 with 4),
        // 4 spread a small input over more lanes (52 x 2048 x 8 fp32 7 us, 13 with 16)
        if (!p.fits) p.beside = p.positions * C > (1 << 20) ? 16 : 4;
        p.units = ((p.fits ? nq : p.positions) + p.beside - 1) / p.beside;
    }
    if (!p.fits) p.most = kLong;
    return p;
}

unsigned groups_of(const Plan& p) { return (unsigned)(p.units < p.most ? p.units : p.most); }
constexpr int kLongShares = 64;
// Of a backward plan.  Long axes: shares of 16 rows at least, or of 512 positions of planes, eight for each lane
int64_t partials_of(const Plan& p) {
    const int64_t shares = p.rows ? (p.positions + 15) / 16 : (p.positions + 511) / 512;
    return p.fits ? (int64_t)groups_of(p) : shares < kLongShares ? shares : kLongShares;
}
bool direct(const Plan& p) { return p.fits && groups_of(p) == 1; }       // the sums are the gradients: no workspace

int check_sizes(int x_type, int w_type, int64_t outer, int64_t C, int64_t inner) {
    if (x_type < FC3D_F32 || x_type > FC3D_F16) return FC3D_EINVAL;
    if (w_type != x_type && w_type != FC3D_F32) return FC3D_EINVAL;
    if (outer < 0 || C <= 0 || inner <= 0) return FC3D_EINVAL;
    const int64_t most = (int64_t)1 << 31;
    if (C >= (1 << 24) || inner >= most || outer >= most || (outer > 0 && outer * inner >= most)) return FC3D_ERANGE;
    return FC3D_OK;
}

bool aligned_to(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (uintptr_t)(bytes - 1)) == 0; }

struct FwdArgs {
    hipStream_t s;
    const void *x, *w, *b;
    bool w_f32;
    int64_t outer, C, inner, x_stride;
    float eps;
    int relu;
    void* y;
    float *mean, *rstd;
};
struct BwdArgs {
    hipStream_t s;
    const void *dy, *x, *w, *b;
    bool w_f32;
    const float *mean, *rstd;
    int64_t outer, C, inner, dy_stride, x_stride;
    int relu;
    void* dx;
    Sums sums;
};

template <typename T, int LPR, int BLOCK, int E>
int rows_launch(const FwdArgs& a, unsigned groups) {
    FC3D_LAUNCH("layer_norm_fwd", (ln_rows_fwd<T, LPR, BLOCK, E>), dim3(groups), dim3(BLOCK), 0, a.s, (const T*)a.x, a.w, a.b,
                a.w_f32, (long)a.outer, (int)a.C, (long)a.x_stride, a.eps, a.relu, (T*)a.y, a.mean, a.rstd);
    return FC3D_OK;
}
template <typename T, int LPR, int BLOCK, int E>
int rows_launch(const BwdArgs& a, unsigned groups) {
    FC3D_LAUNCH("layer_norm_bwd", (ln_rows_bwd<T, LPR, BLOCK, E>), dim3(groups), dim3(BLOCK), 0, a.s, (const T*)a.dy,
                (const T*)a.x, a.w, a.b, a.w_f32, a.mean, a.rstd, (long)a.outer, (int)a.C, (long)a.dy_stride,
                (long)a.x_stride, a.relu, (T*)a.dx, a.sums);
    return FC3D_OK;
}
template <typename T, int V, int CL, int PL, int E>
int planes_launch(const FwdArgs& a, unsigned groups) {
    const unsigned nvec = (unsigned)((a.inner + V - 1) / V), nq = (unsigned)(a.outer * nvec);
    FC3D_LAUNCH("layer_norm_fwd", (ln_planes_fwd<T, V, CL, PL, E>), dim3(groups), dim3(CL * PL), 0, a.s, (const T*)a.x, a.w,
                a.b, a.w_f32, nq, nvec, (int)a.C, (long)a.inner, (long)a.x_stride, a.eps, a.relu, (T*)a.y, a.mean, a.rstd);
    return FC3D_OK;
}
template <typename T, int V, int CL, int PL, int E>
int planes_launch(const BwdArgs& a, unsigned groups) {
    const unsigned nvec = (unsigned)((a.inner + V - 1) / V), nq = (unsigned)(a.outer * nvec);
    FC3D_LAUNCH("layer_norm_bwd", (ln_planes_bwd<T, V, CL, PL, E>), dim3(groups), dim3(CL * PL), 0, a.s, (const T*)a.dy,
                (const T*)a.x, a.w, a.b, a.w_f32, a.mean, a.rstd, nq, nvec, (int)a.C, (long)a.inner, (long)a.dy_stride,
                (long)a.x_stride, a.relu, (T*)a.dx, a.sums);
    return FC3D_OK;
}
template <typename T, int V>
int planes_of(const FwdArgs& a, const Plan& p, unsigned groups) {
    switch (p.lanes) {
        case 1: return planes_launch<T, V, 1, 256, 8>(a, groups);
        case 4: return planes_launch<T, V, 4, 64, 8>(a, groups);
        case 8: return planes_launch<T, V, 8, 32, 8>(a, groups);
        case 16: return planes_launch<T, V, 16, 16, 8>(a, groups);
        case 32: return planes_launch<T, V, 32, 8, 8>(a, groups);
        case 64: return planes_launch<T, V, 64, 8, 8>(a, groups);
        default: return planes_launch<T, V, 128, 4, 8>(a, groups);
    }
}
template <typename T, int V>
int planes_of(const BwdArgs& a, const Plan& p, unsigned groups) {
    constexpr bool F32 = sizeof(T) == 4;
    switch (p.lanes) {
        case 2: return planes_launch<T, V, 2, 128, 4>(a, groups);
        case 8: return p.each == 8 ? planes_launch<T, V, 8, 32, 8>(a, groups) : planes_launch<T, V, 8, 32, 4>(a, groups);
        case 32: return planes_launch<T, V, 32, 16, 4>(a, groups);
        case 64:
            if constexpr (!F32)
                if (p.each == 8) return planes_launch<T, V, 64, 8, 8>(a, groups);
            return planes_launch<T, V, 64, 8, 4>(a, groups);
        default:
            if constexpr (F32)
                if (p.each == 4) return planes_launch<T, V, 128, 8, 4>(a, groups);
            return planes_launch<T, V, 128, 4, 8>(a, groups);
    }
}
template <typename T>
int rows_of(const FwdArgs& a, const Plan& p, unsigned groups) {
    switch (p.lanes) {
        case 8: return p.each == 8 ? rows_launch<T, 8, 256, 8>(a, groups) : rows_launch<T, 8, 256, 16>(a, groups);
        case 16: return rows_launch<T, 16, 256, 16>(a, groups);
        case 32: return rows_launch<T, 32, 256, 16>(a, groups);
        case 64: return rows_launch<T, 64, 256, 16>(a, groups);
        case 128: return rows_launch<T, 128, 256, 16>(a, groups);
        case 256: return rows_launch<T, 256, 256, 16>(a, groups);
        default: return p.each == 8 ? rows_launch<T, 1024, 1024, 8>(a, groups) : rows_launch<T, 1024, 1024, 16>(a, groups);
    }
}
template <typename T>
int rows_of(const BwdArgs& a, const Plan& p, unsigned groups) {
    switch (p.lanes) {
        case 8: return rows_launch<T, 8, 512, 8>(a, groups);
        case 16: return rows_launch<T, 16, 512, 8>(a, groups);
        case 32: return rows_launch<T, 32, 512, 8>(a, groups);
        case 64: return rows_launch<T, 64, 512, 8>(a, groups);
        case 128: return rows_launch<T, 128, 512, 8>(a, groups);
        case 256: return rows_launch<T, 256, 512, 8>(a, groups);
        case 512: return p.each == 8 ? rows_launch<T, 512, 512, 8>(a, groups) : rows_launch<T, 512, 512, 32>(a, groups);
        default: return rows_launch<T, 1024, 1024, 8>(a, groups);
    }
}
// The register kernel of a plan, forward or backward by the arguments' type
template <typename T, typename A>
int registers_of(const A& a, const Plan& p) {
    const unsigned groups = groups_of(p);
    if (p.rows) return rows_of<T>(a, p, groups);
    return p.wide ? planes_of<T, kVec>(a, p, groups) : planes_of<T, 1>(a, p, groups);
}

template <typename T, int NP>
int long_of(const FwdArgs& a, const Plan& p) {
    FC3D_LAUNCH("layer_norm_fwd", (ln_long_fwd<T, NP>), dim3(groups_of(p)), dim3(kLongBlock), 0, a.s, (const T*)a.x, a.w,
                a.b, a.w_f32, (long)(a.outer * a.inner), (long)a.C, (long)a.inner, (long)a.x_stride, a.eps, a.relu, (T*)a.y,
                a.mean, a.rstd);
    return FC3D_OK;
}
template <typename T, int NP>
int long_of(const BwdArgs& a, const Plan& p) {
    const T *dy = (const T*)a.dy, *x = (const T*)a.x;
    const long positions = (long)(a.outer * a.inner);
    if (a.dx)
        FC3D_LAUNCH("layer_norm_bwd", (ln_long_bwd<T, NP>), dim3(groups_of(p)), dim3(kLongBlock), 0, a.s, dy, x, a.w, a.b,
                    a.w_f32, a.mean, a.rstd, positions, (long)a.C, (long)a.inner, (long)a.dy_stride, (long)a.x_stride,
                    a.relu, (T*)a.dx);
    if (a.sums.wanted())
        FC3D_LAUNCH("layer_norm_params", (ln_long_params<T, (NP > 1)>),
                    dim3((unsigned)(NP > 1 ? (a.C + 3) / 4 : (a.C + 255) / 256), (unsigned)partials_of(p)), dim3(256), 0, a.s, dy, x, a.w, a.b,
                    a.w_f32, a.mean, a.rstd, positions, (long)a.C, (long)a.inner, (long)a.dy_stride, (long)a.x_stride,
                    a.relu, a.sums.partial);
    return FC3D_OK;
}

template <typename T, typename A>
int kernel_of(const A& a, const Plan& p) {
    if (p.fits) return registers_of<T>(a, p);
    return p.rows ? long_of<T, 1>(a, p) : p.beside == 4 ? long_of<T, 4>(a, p) : long_of<T, 16>(a, p);
}
template <typename A>
int type_of(const A& a, const Plan& p, int x_type) {
    return x_type == FC3D_F32 ? kernel_of<float>(a, p) : x_type == FC3D_BF16 ? kernel_of<bf16>(a, p) : kernel_of<f16>(a, p);
}

__global__ __launch_bounds__(256) void ln_params_clear(long C, int type, void* __restrict__ dw, void* __restrict__ db) {
    const long i = (long)blockIdx.x * 256 + threadIdx.x;
    if (i < C) {
        if (dw) put_param(dw, type, i, 0.0f);
        if (db) put_param(db, type, i, 0.0f);
    }
}

}  // namespace
}  // namespace fc3d

using namespace fc3d;

extern "C" int fc3d_layer_norm_fwd(void* stream, const void* x, int x_type, const void* weight, const void* bias, int w_type,
                                   int64_t outer, int64_t channels, int64_t inner, int64_t x_stride, float eps, int relu,
                                   void* y, float* mean, float* rstd) {
    if (const int rc = check_sizes(x_type, w_type, outer, channels, inner)) return rc;
    if (!(eps >= 0.0f) || (mean == nullptr) != (rstd == nullptr)) return FC3D_EINVAL;
    if (outer == 0) return FC3D_OK;
    if (!x || !y || x_stride < 0) return FC3D_EINVAL;
    if (!aligned_to(x, elem_size(x_type)) || !aligned_to(y, elem_size(x_type)) || !aligned_to(weight, elem_size(w_type)) ||
        !aligned_to(bias, elem_size(w_type)) || !aligned_to(mean, 4) || !aligned_to(rstd, 4))
        return FC3D_EALIGN;
    const FwdArgs a = {(hipStream_t)stream, x, weight, bias, w_type == FC3D_F32, outer, channels, inner, x_stride, eps, relu,
                       y, mean, rstd};
    return type_of(a, plan_of(true, x_type, outer, channels, inner), x_type);
}

extern "C" size_t fc3d_layer_norm_bwd_workspace(int x_type, int64_t outer, int64_t channels, int64_t inner) {
    if (check_sizes(x_type, x_type, outer, channels, inner) != FC3D_OK || outer == 0) return 0;
    const Plan p = plan_of(false, x_type, outer, channels, inner);
    return direct(p) ? 0 : (size_t)partials_of(p) * 2 * (size_t)channels * sizeof(float);
}

extern "C" int fc3d_layer_norm_bwd(void* stream, const void* dy, const void* x, int x_type, const void* weight,
                                   const void* bias, int w_type, const float* mean, const float* rstd, int64_t outer,
                                   int64_t channels, int64_t inner, int64_t dy_stride, int64_t x_stride, int relu, void* dx,
                                   void* dw, void* db, void* workspace) {
    if (const int rc = check_sizes(x_type, w_type, outer, channels, inner)) return rc;
    if (!dx && !dw && !db) return FC3D_OK;
    if (!aligned_to(dw, elem_size(w_type)) || !aligned_to(db, elem_size(w_type))) return FC3D_EALIGN;
    if (outer == 0) {
        if (!dw && !db) return FC3D_OK;
        FC3D_LAUNCH("layer_norm_params", ln_params_clear, dim3((unsigned)((channels + 255) / 256)), dim3(256), 0,
                    (hipStream_t)stream, (long)channels, w_type, dw, db);
        return FC3D_OK;
    }
    const Plan p = plan_of(false, x_type, outer, channels, inner);
    if (!dy || !x || !mean || !rstd || dy_stride < 0 || x_stride < 0 || ((dw || db) && !workspace)) return FC3D_EINVAL;
    if (!aligned_to(dy, elem_size(x_type)) || !aligned_to(x, elem_size(x_type)) || !aligned_to(dx, elem_size(x_type)) ||
        !aligned_to(weight, elem_size(w_type)) || !aligned_to(bias, elem_size(w_type)) || !aligned_to(mean, 4) ||
        !aligned_to(rstd, 4) || !aligned_to(workspace, 4))
        return FC3D_EALIGN;
    const BwdArgs a = {(hipStream_t)stream, dy, x, weight, bias, w_type == FC3D_F32, mean, rstd, outer, channels, inner,
                       dy_stride, x_stride, relu, dx, Sums{(float*)workspace, dw, db, w_type}};
    const int rc = type_of(a, p, x_type);
    if (rc != FC3D_OK || !a.sums.wanted() || direct(p)) return rc;
    FC3D_LAUNCH("layer_norm_params_sum", ln_params_sum, dim3((unsigned)((2 * channels + 31) / 32)), dim3(1024), 0, a.s,
                a.sums.partial, (int)partials_of(p), (long)channels, w_type, dw, db);
    return FC3D_OK;
}
