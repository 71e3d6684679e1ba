// Root-mean-square norm of rows with the residual's addition:
//     h = x + r,   rstd = 1 / sqrt(mean(h^2) + eps),   y = h rstd w          (one pass: the row stays in registers between its sum and its output)
// its gradient, with g = dy w and xh = h rstd,
//     dx = rstd (g - xh mean(g xh)) + dh,   dw = sum over rows of dy xh,
// and its output in 8 bits: s = max|y| / 448 over the row or over each group of its columns, q = e4m3(y / s).
//
// Bound by HBM: a few operations for each value read or written.  A row is taken by 8, 16, 32, 64, 256 or 1024 lanes, so that a lane holds at most 32 values of it (one to
// eight loads of sixteen bytes, all in flight before the first is used) and the sum is one exchange inside a wave, or one through LDS.  The weights of a lane's
// columns are read once and stay in registers for all the rows that its workgroup takes.  Rows may start anywhere (odd widths, strides): the part reads sixteen
// bytes from any address; only a row's last, partial piece goes value by value.
//
// Measured (a large copy: 5.2 TB/s): 131072 rows of 512, fp32, with residual: 185 us = 5.8 TB/s, backward 206 us = 5.2; 8192 rows of 8192, bf16: 111 us = 4.8, backward 142 us = 4.7 and
// 5 us for dw; 8192 rows of 4096, bf16 to 8 bits with residual: 39 us = 6.0; 5000 rows of 717, fp16, a scale to 128 columns: 9.7 us; one row: 4 us, a launch's latency.
#include "ogmm_common.h"
#include <algorithm>
#include <type_traits>

namespace {

using namespace ogmm;

constexpr int MAX_D = 32768;
constexpr float E4M3_MAX = 448.0f;

template <class T, int N>
struct __attribute__((packed, aligned(sizeof(T)))) Piece { T v[N]; };
template <int N>
struct __attribute__((packed, aligned(1))) Bytes { uint32_t w[N / 4]; };

// values [c, c + N) of a row of D; zeros behind its end
template <int N, class T>
__device__ __forceinline__ void load(const T* __restrict__ row, int c, int D, float (&out)[N]) {
    if (c + N <= D) {
        const Piece<T, N> p = *reinterpret_cast<const Piece<T, N>*>(row + c);
#pragma unroll
        for (int k = 0; k < N; ++k) out[k] = static_cast<float>(p.v[k]);
    } else {
#pragma unroll
        for (int k = 0; k < N; ++k) out[k] = c + k < D ? static_cast<float>(row[c + k]) : 0.0f;
    }
}

// sixteen bytes as they lie in memory, to be widened when they are used: a wide row's values take half the registers
struct Raw { uint32_t w[4]; };
template <class T>
__device__ __forceinline__ Raw fetch(const T* __restrict__ row, int c, int D) {
    constexpr int N = 16 / sizeof(T);
    if (c + N <= D) return __builtin_bit_cast(Raw, *reinterpret_cast<const Piece<T, N>*>(row + c));
    Piece<T, N> p;
#pragma unroll
    for (int k = 0; k < N; ++k) p.v[k] = c + k < D ? row[c + k] : static_cast<T>(0.0f);
    return __builtin_bit_cast(Raw, p);
}
template <class T>
__device__ __forceinline__ float value(const Raw& r, int k) {
    if constexpr (sizeof(T) == 4) return __uint_as_float(r.w[k]);
    else if constexpr (std::is_same_v<T, __bf16>) return __uint_as_float(k & 1 ? r.w[k / 2] & 0xffff0000u : r.w[k / 2] << 16);
    else return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(k & 1 ? r.w[k / 2] >> 16 : r.w[k / 2] & 0xffff)));
}

template <int N, class T>
__device__ __forceinline__ void store(T* __restrict__ row, int c, int D, const float (&x)[N]) {
    if (c + N <= D) {
        Piece<T, N> p;
#pragma unroll
        for (int k = 0; k < N; ++k) p.v[k] = static_cast<T>(x[k]);
        *reinterpret_cast<Piece<T, N>*>(row + c) = p;
    } else {
#pragma unroll
        for (int k = 0; k < N; ++k)
            if (c + k < D) row[c + k] = static_cast<T>(x[k]);
    }
}

// Sum (or maximum) over the LANES lanes of one row; every lane gets it.  `slot` alternates between rows, so that one barrier a row is enough.
template <int LANES, bool MAX>
__device__ __forceinline__ float over_row(float v, float* lds, int& slot) {
#pragma unroll
    for (int o = 1; o < (LANES < 64 ? LANES : 64); o <<= 1) {
        const float u = __shfl_xor(v, o, 64);
        v = MAX ? fmaxf(v, u) : v + u;
    }
    if constexpr (LANES > 64) {
        constexpr int W = LANES / 64;
        float* s = lds + slot * W;
        slot ^= 1;
        if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
        __syncthreads();
        v = s[0];
#pragma unroll
        for (int i = 1; i < W; ++i) v = MAX ? fmaxf(v, s[i]) : v + s[i];
    }
    return v;
}

template <int LANES> constexpr int THREADS = LANES > 256 ? LANES : 256;

// Squares of fp32 or bf16 values leave fp32 from 2^64 on, and below 2^-50 come near the end of its normal numbers: the sum is formed again from the values times a power of two then
__device__ __forceinline__ bool squares_fit(float ss, float eps) { return ss < INFINITY && (ss > 0x1p-100f || eps > 0x1p-70f); }


struct NormArgs {
    const void *x, *r, *w;
    int64_t ldx, ldr, rows;
    int D, group;
    float eps;
    void *y, *h;
    float *rstd, *scales;
};

// Q8: y in 8 bits with scales
template <class T, class W, int LANES, int ITEMS, bool Q8>
__global__ __launch_bounds__(THREADS<LANES>) void rms_norm_kernel(const NormArgs a) {
    constexpr int VEC = 16 / sizeof(T), PER = THREADS<LANES> / LANES;
    __shared__ float lds[2 * (LANES > 64 ? LANES / 64 : 1)];
    int slot = 0;
    const int lane = threadIdx.x % LANES, D = a.D;
    float w[ITEMS][VEC];
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) load<VEC>(static_cast<const W*>(a.w), (i * LANES + lane) * VEC, D, w[i]);
    for (int64_t row0 = static_cast<int64_t>(blockIdx.x) * PER; row0 < a.rows; row0 += static_cast<int64_t>(gridDim.x) * PER) {
        const int64_t row = row0 + threadIdx.x / LANES;
        const bool here = LANES > 64 || row < a.rows;          // (a row's lanes agree; lanes of one wave may hold several rows and take part in the exchange)
        const T* x = static_cast<const T*>(a.x) + row * a.ldx;
        float h[ITEMS][VEC];
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) load<VEC>(x, (i * LANES + lane) * VEC, here ? D : 0, h[i]);
        if (a.r) {
            const T* r = static_cast<const T*>(a.r) + row * a.ldr;
            float u[ITEMS][VEC];
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) load<VEC>(r, (i * LANES + lane) * VEC, here ? D : 0, u[i]);
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
#pragma unroll
                for (int k = 0; k < VEC; ++k) h[i][k] += u[i][k];
                // (the stored sum is rounded to the type of the stream it belongs to; the norm below takes the sum itself)
                store<VEC>(static_cast<T*>(a.h) + row * D, (i * LANES + lane) * VEC, here ? D : 0, h[i]);
            }
        }
        float ss = 0.0f;
#pragma unroll
        for (int i = 0; i < ITEMS; ++i)
#pragma unroll
            for (int k = 0; k < VEC; ++k) ss = fmaf(h[i][k], h[i][k], ss);
        ss = over_row<LANES, false>(ss, lds, slot);
        float rstd = 1.0f / sqrtf(ss / D + a.eps), k = 1.0f;          // rstd: of h as it stands here, k times the row
        if constexpr (!std::is_same_v<T, _Float16>)
            if (!squares_fit(ss, a.eps)) {          // (a row's lanes agree)
                k = ss < 1.0f ? 0x1p72f : 0x1p-72f;
                ss = 0.0f;
#pragma unroll
                for (int i = 0; i < ITEMS; ++i)
#pragma unroll
                    for (int j = 0; j < VEC; ++j) {
                        h[i][j] *= k;
                        ss = fmaf(h[i][j], h[i][j], ss);
                    }
                ss = over_row<LANES, false>(ss, lds, slot);
                rstd = 1.0f / sqrtf(ss / D + a.eps * k * k);
            }
        if constexpr (!Q8) {
            if (a.rstd && here && lane == 0) a.rstd[row] = rstd * k;
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
#pragma unroll
                for (int k = 0; k < VEC; ++k) h[i][k] = h[i][k] * rstd * w[i][k];
                store<VEC>(static_cast<T*>(a.y) + row * D, (i * LANES + lane) * VEC, here ? D : 0, h[i]);
            }
        } else {
            // rstd > 0 leaves y / s as it is where both lack it: t = h w, s = rstd max|t| / 448, q = e4m3(t 448 / max|t|), one rounding less than through y
            const int groups = a.group ? (D + a.group - 1) / a.group : 1;
            float top[ITEMS];
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
                top[i] = 0.0f;
#pragma unroll
                for (int k = 0; k < VEC; ++k) {
                    h[i][k] *= w[i][k];
                    top[i] = fmaxf(top[i], fabsf(h[i][k]));
                }
            }
            if (a.group) {
                for (int o = 1; o < a.group / VEC; o <<= 1)          // (a group's lanes are neighbours in one wave: 32, 64 or 128 columns)
#pragma unroll
                    for (int i = 0; i < ITEMS; ++i) top[i] = fmaxf(top[i], __shfl_xor(top[i], o, 64));
            } else {
                float m = top[0];
#pragma unroll
                for (int i = 1; i < ITEMS; ++i) m = fmaxf(m, top[i]);
                m = over_row<LANES, true>(m, lds, slot);
#pragma unroll
                for (int i = 0; i < ITEMS; ++i) top[i] = m;
            }
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
                const int c = (i * LANES + lane) * VEC;
                float s = top[i] * rstd / E4M3_MAX;
                if (s < 1.17549435e-38f) s = 0.0f;          // (below the normal numbers the quotient y / s would not be defined to 4 bits)
                const float up = top[i] < 1e-30f ? 0x1p100f : 1.0f;          // 448 / max|t| stays finite
                const float inv = s == 0.0f ? 0.0f : E4M3_MAX / (top[i] * up);
                if (here && c < D && (a.group ? c % a.group == 0 : c == 0)) a.scales[row * groups + (a.group ? c / a.group : 0)] = s;
                float q[VEC];
#pragma unroll
                for (int k = 0; k < VEC; ++k) q[k] = h[i][k] * up * inv;
                Bytes<VEC> b;
#pragma unroll
                for (int k = 0; k < VEC; k += 4)
                    b.w[k / 4] = (__builtin_amdgcn_cvt_pk_fp8_f32(q[k], q[k + 1], 0, false) & 0xffff) | __builtin_amdgcn_cvt_pk_fp8_f32(q[k + 2], q[k + 3], 0, false) << 16;
                uint8_t* o = static_cast<uint8_t*>(a.y) + row * D + c;
                if (here && c + VEC <= D) *reinterpret_cast<Bytes<VEC>*>(o) = b;
                else
#pragma unroll
                    for (int k = 0; k < VEC; ++k)
                        if (here && c + k < D) o[k] = static_cast<uint8_t>(b.w[k / 4] >> (k % 4 * 8));
            }
        }
    }
}

struct BwdArgs {
    const void *dy, *h, *r, *w, *dh;
    const float* rstd;
    int64_t lddy, ldh, ldr, lddh, rows;
    int D;
    void* dx;
    float* part;          // [gridDim.x][D]: each workgroup's share of dw
};

// RES: the sum is formed again from its two 16-bit summands.  Its stored form is off by half a step of the type, which dw -- a sum of terms of either sign -- passes on as it is: its error
// was 1.4 times that of its own rounding (8192 rows of 8192, bf16: 142 us, 115 from the stored sum: a fifth matrix to read, at the same 4.7 TB/s)
template <class T, class W, int LANES, int ITEMS, bool RES>
__global__ __launch_bounds__(THREADS<LANES>, (LANES > 256 ? 4 : 2)) void rms_norm_bwd_kernel(const BwdArgs a) {
    constexpr int VEC = 16 / sizeof(T), PER = THREADS<LANES> / LANES;
    __shared__ float lds[2 * (LANES > 64 ? LANES / 64 : 1)];
    __shared__ float share[PER > 1 ? PER * LANES * VEC : 1];
    int slot = 0;
    const int lane = threadIdx.x % LANES, D = a.D;
    // the weights: in registers in 32 bits, or where 1024 lanes or four loads of every input leave few of those in the rows' own 16
    constexpr bool RAW_W = sizeof(W) == 2 && (LANES > 256 || (RES && ITEMS > 2));
    constexpr int WVEC = 16 / sizeof(W);
    Raw w_raw[RAW_W ? ITEMS : 1];
    float w[RAW_W ? 1 : ITEMS][VEC], dw[ITEMS][VEC];
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
        if constexpr (RAW_W) w_raw[i] = fetch<W>(static_cast<const W*>(a.w), (i * LANES + lane) * VEC, D);
        else load<VEC>(static_cast<const W*>(a.w), (i * LANES + lane) * VEC, D, w[i]);
#pragma unroll
        for (int k = 0; k < VEC; ++k) dw[i][k] = 0.0f;
    }
    static_assert(!RAW_W || WVEC == VEC, "weights");
    auto weight = [&](int i, int k) {
        if constexpr (RAW_W) return value<W>(w_raw[i], k);
        else return w[i][k];
    };
    const float inv_d = 1.0f / D;
    // Where the registers allow it, the next row is on its way while this one is worked on (8192 rows of 8192 from the summands, four inputs of four loads: 142 us without it, 253
    // with it, for what then spills)
    constexpr bool AHEAD = LANES <= 256 && !(RES && ITEMS > 2);
    Raw rg[ITEMS], rh[ITEMS], ru[ITEMS], rr[RES ? ITEMS : 1];
    float rstd = 0.0f;
    auto fetch_row = [&](Raw (&g)[ITEMS], Raw (&h)[ITEMS], Raw (&u)[ITEMS], Raw* x, float& r, int64_t row) {          // (a row's lanes agree on whether it is there)
        const int d = row < a.rows ? D : 0;
        r = d ? a.rstd[row] : 0.0f;
        const T *pg = static_cast<const T*>(a.dy) + row * a.lddy, *ph = static_cast<const T*>(a.h) + row * a.ldh, *pu = static_cast<const T*>(a.dh) + row * a.lddh,
                *pr = static_cast<const T*>(a.r) + row * a.ldr;
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            g[i] = fetch<T>(pg, (i * LANES + lane) * VEC, d);
            h[i] = fetch<T>(ph, (i * LANES + lane) * VEC, d);
            if constexpr (RES) x[i] = fetch<T>(pr, (i * LANES + lane) * VEC, d);
            if (a.dh) u[i] = fetch<T>(pu, (i * LANES + lane) * VEC, d);
        }
    };
    auto sum = [&](int i, int k) {
        if constexpr (RES) return value<T>(rh[i], k) + value<T>(rr[i], k);
        else return value<T>(rh[i], k);
    };
    const int64_t step = static_cast<int64_t>(gridDim.x) * PER;
    int64_t row = static_cast<int64_t>(blockIdx.x) * PER + threadIdx.x / LANES;
    if constexpr (AHEAD) fetch_row(rg, rh, ru, rr, rstd, row);
    for (int64_t row0 = static_cast<int64_t>(blockIdx.x) * PER; row0 < a.rows; row0 += step, row += step) {
        if constexpr (!AHEAD) fetch_row(rg, rh, ru, rr, rstd, row);
        Raw ng[AHEAD ? ITEMS : 1], nh[AHEAD ? ITEMS : 1], nu[AHEAD ? ITEMS : 1], nr[AHEAD && RES ? ITEMS : 1];
        float next_rstd = 0.0f;
        if constexpr (AHEAD)
            if (row0 + step < a.rows) fetch_row(ng, nh, nu, nr, next_rstd, row + step);
        float dot = 0.0f;
#pragma unroll
        for (int i = 0; i < ITEMS; ++i)
#pragma unroll
            for (int k = 0; k < VEC; ++k) {
                const float g = value<T>(rg[i], k), xh = sum(i, k) * rstd;
                dw[i][k] = fmaf(g, xh, dw[i][k]);
                dot = fmaf(g * weight(i, k), xh, dot);
            }
        dot = over_row<LANES, false>(dot, lds, slot) * inv_d;
        const int d = row < a.rows ? D : 0;
        // (widened once more below: kept wide across the exchange, the row would take twice the registers)
        if constexpr (sizeof(T) == 2)
#pragma unroll
            for (int i = 0; i < ITEMS; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    asm volatile("" : "+v"(rg[i].w[j]), "+v"(rh[i].w[j]));
                    if constexpr (RES) asm volatile("" : "+v"(rr[i].w[j]));
                }
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            float dx[VEC];
#pragma unroll
            for (int k = 0; k < VEC; ++k) {
                dx[k] = rstd * (value<T>(rg[i], k) * weight(i, k) - sum(i, k) * rstd * dot);
                if (a.dh) dx[k] += value<T>(ru[i], k);
            }
            store<VEC>(static_cast<T*>(a.dx) + row * D, (i * LANES + lane) * VEC, d, dx);
        }
        if constexpr (AHEAD) {
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
                rg[i] = ng[i];
                rh[i] = nh[i];
                ru[i] = nu[i];
                if constexpr (RES) rr[i] = nr[i];
            }
            rstd = next_rstd;
        }
    }
    float* part = a.part + static_cast<int64_t>(blockIdx.x) * D;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
        if constexpr (PER == 1) {
            store<VEC>(part, (i * LANES + lane) * VEC, D, dw[i]);
        } else {          // the workgroup's rows side by side: one sum over them, in their order
            __syncthreads();
#pragma unroll
            for (int k = 0; k < VEC; ++k) share[threadIdx.x * VEC + k] = dw[i][k];
            __syncthreads();
            for (int e = threadIdx.x; e < LANES * VEC; e += THREADS<LANES>) {
                float s = 0.0f;
                for (int p = 0; p < PER; ++p) s += share[p * LANES * VEC + e];
                const int c = i * LANES * VEC + e;
                if (c < D) part[c] = s;
            }
        }
    }
}

// dw[c] = sum over the workgroups' shares, in fp64: 64 columns to a workgroup, sixteen slices of the shares beside each other.  A share is summed in fp32, over the rows of a lane (131072 rows of 512,
// fp32: 64 of them) and those side by side in a workgroup, which is most of dw's error: 1.7e-7 of its 2-norm, where fp64 throughout gives 5.8e-8 and its own rounding is 2.5e-8
template <class W>
__global__ __launch_bounds__(1024) void rms_norm_dw_kernel(const float* __restrict__ part, int n, int D, W* __restrict__ dw) {
    __shared__ double lds[16][64];
    const int c = blockIdx.x * 64 + (threadIdx.x & 63), s = threadIdx.x >> 6;
    double acc = 0.0;
    if (c < D)
#pragma unroll 8
        for (int i = s; i < n; i += 16) acc += part[static_cast<int64_t>(i) * D + c];
    lds[s][threadIdx.x & 63] = acc;
    __syncthreads();
    if (s == 0 && c < D) {
        for (int i = 1; i < 16; ++i) acc += lds[i][threadIdx.x];
        dw[c] = static_cast<W>(static_cast<float>(acc));
    }
}

// Lanes to a row and loads of sixteen bytes to a lane: the fewest lanes that keep a lane at four loads (narrow rows: two), so that narrow rows share a workgroup and the sum over a
// row takes few exchanges; the widest fp32 rows take eight
template <class T, class F>
int with_shape(int D, int least_lanes, F&& f) {
    constexpr int VEC = 16 / sizeof(T);
    using std::integral_constant;
    auto go = [&](auto lanes, auto items) { return f(lanes, items); };
    const int n = (D + VEC - 1) / VEC;
#define OGMM_SHAPE(L, I) if (n <= L * I && least_lanes <= L) return go(integral_constant<int, L>(), integral_constant<int, I>())
    OGMM_SHAPE(8, 1);
    OGMM_SHAPE(8, 2);
    OGMM_SHAPE(16, 2);
    OGMM_SHAPE(32, 2);
    OGMM_SHAPE(64, 2);
    OGMM_SHAPE(64, 4);
    OGMM_SHAPE(256, 2);
    OGMM_SHAPE(256, 4);
    OGMM_SHAPE(1024, 2);
    OGMM_SHAPE(1024, 4);
    if constexpr (sizeof(T) == 4) OGMM_SHAPE(1024, 8);
#undef OGMM_SHAPE
    return fail("rms_norm: rows of %d values are too wide", D);
}

// workgroups: as many as the rows need, and no more than fill the 256 CUs a few times over (each reads the weights once)
inline int blocks_for(int64_t rows, int per, int most) { return static_cast<int>(std::min<int64_t>((rows + per - 1) / per, most)); }

template <class T, class W>
int launch_norm(const NormArgs& a, bool q8, hipStream_t stream) {
    return with_shape<T>(a.D, a.group ? 64 : 1, [&](auto lanes, auto items) {
        constexpr int L = decltype(lanes)::value, I = decltype(items)::value;
        const int blocks = blocks_for(a.rows, THREADS<L> / L, L > 256 ? 1024 : 4096);
        if (q8) rms_norm_kernel<T, W, L, I, true><<<blocks, THREADS<L>, 0, stream>>>(a);
        else rms_norm_kernel<T, W, L, I, false><<<blocks, THREADS<L>, 0, stream>>>(a);
        return check_launch("ogmm_rms_norm");
    });
}

// dw's shares are written and read again (blocks x D x 4 bytes): two workgroups to a CU for wide rows, four for narrow ones, whose waves have fewer bytes on their way each
// (131072 fp32 rows of 512: 206 us with two, 216 with four)
constexpr int BWD_BLOCKS = 1024;

template <class T, class W>
int launch_bwd(const BwdArgs& a, void* dw, hipStream_t stream) {
    return with_shape<T>(a.D, 1, [&](auto lanes, auto items) {
        constexpr int L = decltype(lanes)::value, I = decltype(items)::value;
        const int blocks = blocks_for(a.rows, THREADS<L> / L, L > 32 ? BWD_BLOCKS / 2 : BWD_BLOCKS);
        if constexpr (sizeof(T) == 2) {
            if (blocks && a.r) rms_norm_bwd_kernel<T, W, L, I, true><<<blocks, THREADS<L>, 0, stream>>>(a);
        }
        if (blocks && !a.r) rms_norm_bwd_kernel<T, W, L, I, false><<<blocks, THREADS<L>, 0, stream>>>(a);
        rms_norm_dw_kernel<W><<<(a.D + 63) / 64, 1024, 0, stream>>>(a.part, blocks, a.D, static_cast<W*>(dw));
        return check_launch("ogmm_rms_norm_bwd");
    });
}

template <class F>
int with_types(const char* who, int type, int wtype, F&& f) {
    if (type == OGMM_F32 && wtype == OGMM_F32) return f(float(), float());
    if (type == OGMM_BF16 && wtype == OGMM_BF16) return f(__bf16(), __bf16());
    if (type == OGMM_BF16 && wtype == OGMM_F32) return f(__bf16(), float());
    if (type == OGMM_F16 && wtype == OGMM_F16) return f(_Float16(), _Float16());
    if (type == OGMM_F16 && wtype == OGMM_F32) return f(_Float16(), float());
    return fail("%s: rows of type %d with weights of type %d are not supported", who, type, wtype);
}

int check_rows(const char* who, int64_t rows, int D) {
    OGMM_REQUIRE(rows >= 0, "%s: negative number of rows", who);
    OGMM_REQUIRE(D >= 1 && D <= MAX_D, "%s: rows of %d values (1 to %d are supported)", who, D, MAX_D);
    return 0;
}

}  // namespace

extern "C" int ogmm_rms_norm(const void* x, int64_t ldx, const void* residual, int64_t ldr, const void* weight, int64_t rows, int D, int type, int weight_type, float eps,
                             void* y, void* h, float* rstd, void* stream) {
    if (check_rows("ogmm_rms_norm", rows, D)) return 1;
    OGMM_REQUIRE(weight && (!rows || (x && y)) && (!rows || !residual || h), "ogmm_rms_norm: missing argument");
    OGMM_REQUIRE(eps >= 0.0f, "ogmm_rms_norm: eps must not be negative");
    if (!rows) return 0;
    const NormArgs a{x, residual, weight, ldx, ldr, rows, D, 0, eps, y, h, rstd, nullptr};
    return with_types("ogmm_rms_norm", type, weight_type, [&](auto t, auto w) { return launch_norm<decltype(t), decltype(w)>(a, false, as_stream(stream)); });
}

extern "C" int ogmm_rms_norm_q8(const void* x, int64_t ldx, const void* residual, int64_t ldr, const void* weight, int64_t rows, int D, int type, int weight_type, float eps,
                                int group, void* q, float* scales, void* h, void* stream) {
    if (check_rows("ogmm_rms_norm_q8", rows, D)) return 1;
    OGMM_REQUIRE(weight && (!rows || (x && q && scales)) && (!rows || !residual || h), "ogmm_rms_norm_q8: missing argument");
    OGMM_REQUIRE(eps >= 0.0f, "ogmm_rms_norm_q8: eps must not be negative");
    OGMM_REQUIRE(group == 0 || group == 32 || group == 64 || group == 128, "ogmm_rms_norm_q8: group must be 0 (the row), 32, 64 or 128 columns, got %d", group);
    if (!rows) return 0;
    const NormArgs a{x, residual, weight, ldx, ldr, rows, D, group, eps, q, h, nullptr, scales};
    return with_types("ogmm_rms_norm_q8", type, weight_type, [&](auto t, auto w) { return launch_norm<decltype(t), decltype(w)>(a, true, as_stream(stream)); });
}

extern "C" int64_t ogmm_rms_norm_bwd_workspace_bytes(int64_t rows, int D) {
    if (rows < 0 || D < 1) return -1;
    return std::max<int64_t>(1, std::min<int64_t>(rows, BWD_BLOCKS)) * D * static_cast<int64_t>(sizeof(float));
}

extern "C" int ogmm_rms_norm_bwd(const void* dy, int64_t lddy, const void* h, int64_t ldh, const void* residual, int64_t ldr, const void* weight, const float* rstd, const void* dh, int64_t lddh, int64_t rows,
                                 int D, int type, int weight_type, void* dx, void* dweight, void* workspace, void* stream) {
    if (check_rows("ogmm_rms_norm_bwd", rows, D)) return 1;
    OGMM_REQUIRE(weight && dweight && workspace && (!rows || (dy && h && rstd && dx)), "ogmm_rms_norm_bwd: missing argument");
    OGMM_REQUIRE(!residual || type != OGMM_F32, "ogmm_rms_norm_bwd: fp32 rows are given as their sum");
    const BwdArgs a{dy, h, residual, weight, dh, rstd, lddy, ldh, ldr, lddh, rows, D, dx, static_cast<float*>(workspace)};
    return with_types("ogmm_rms_norm_bwd", type, weight_type, [&](auto t, auto w) { return launch_bwd<decltype(t), decltype(w)>(a, dweight, as_stream(stream)); });
}
