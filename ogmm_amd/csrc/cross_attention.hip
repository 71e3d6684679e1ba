// Cross attention to states of another length (include/ogmm_hip.h, L1), forward and backward.
//
// Simple form: one wave to a query row (forward, dq) or to a key row (dk, dv); scores are formed 64 at a time, a lane each, and never reach memory.
#include "ogmm_common.h"
#include <math.h>
#include <type_traits>

namespace {

using namespace ogmm;

struct Args : ogmm_xattn {};

__device__ __forceinline__ int clamp_len(const int32_t* lens, int b, int n) { return lens ? max(0, min(n, lens[b])) : n; }

__device__ __forceinline__ bool admitted(const Args& a, int b, int n, int len) { return n < len && (!a.key_mask || a.key_mask[b * a.mask_b + n]); }

template <class T>
__device__ __forceinline__ float dot(const float* __restrict__ u, const T* __restrict__ x, int d) {
    float s = 0.0f;
    for (int c = 0; c < d; ++c) s = fmaf(u[c], static_cast<float>(x[c]), s);
    return s;
}

// rows of q: waves over (b, h, n)
template <class T>
__global__ __launch_bounds__(256) void xattn_fwd_kernel(const Args a) {
    __shared__ float qs[4][128];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, d = a.d;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * 4 + wave;
    if (row >= static_cast<int64_t>(a.B) * a.H * a.Nq) return;
    const int n = row % a.Nq, h = row / a.Nq % a.H, b = row / a.Nq / a.H, hk = h / (a.H / a.Hkv);
    const T *q = static_cast<const T*>(a.q) + b * a.q_b + n * a.q_n + h * a.q_h;
    const T *k = static_cast<const T*>(a.k) + b * a.k_b + hk * a.k_h, *v = static_cast<const T*>(a.v) + b * a.v_b + hk * a.v_h;
    const int len = n < clamp_len(a.q_lens, b, a.Nq) ? clamp_len(a.kv_lens, b, a.Nk) : 0;
    for (int c = lane; c < d; c += 64) qs[wave][c] = static_cast<float>(q[c]) * a.scale;
    float m = -INFINITY, l = 0.0f, o0 = 0.0f, o1 = 0.0f;
    for (int j0 = 0; j0 < len; j0 += 64) {
        const int j = j0 + lane;
        const float s = admitted(a, b, j, len) ? dot(qs[wave], k + j * a.k_n, d) : -INFINITY;
        const float top = fmaxf(m, wave_max(s));
        if (top == -INFINITY) continue;
        const float p = expf(s - top), f = expf(m - top);
        m = top;
        l = l * f + wave_sum(p);
        o0 *= f;
        o1 *= f;
        for (int i = 0; i < 64 && j0 + i < len; ++i) {
            const float pi = __shfl(p, i, 64);
            if (pi == 0.0f) continue;
            const T* vi = v + static_cast<int64_t>(j0 + i) * a.v_n;
            if (lane < d) o0 = fmaf(pi, static_cast<float>(vi[lane]), o0);
            if (lane + 64 < d) o1 = fmaf(pi, static_cast<float>(vi[lane + 64]), o1);
        }
    }
    T* o = static_cast<T*>(a.o) + ((static_cast<int64_t>(b) * a.Nq + n) * a.H + h) * d;
    const float inv = l > 0.0f ? 1.0f / l : l;
    if (lane < d) o[lane] = static_cast<T>(o0 * inv);
    if (lane + 64 < d) o[lane + 64] = static_cast<T>(o1 * inv);
    if (a.lse && lane == 0) a.lse[row] = l == 0.0f ? -INFINITY : m + logf(l);
}

template <class T>
__global__ __launch_bounds__(256) void xattn_dq_kernel(const Args a) {
    __shared__ float qs[4][128], gs[4][128];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, d = a.d;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * 4 + wave;
    if (row >= static_cast<int64_t>(a.B) * a.H * a.Nq) return;
    const int n = row % a.Nq, h = row / a.Nq % a.H, b = row / a.Nq / a.H, hk = h / (a.H / a.Hkv);
    const T *q = static_cast<const T*>(a.q) + b * a.q_b + n * a.q_n + h * a.q_h, *g = static_cast<const T*>(a.dout) + b * a.do_b + n * a.do_n + h * a.do_h;
    const T *k = static_cast<const T*>(a.k) + b * a.k_b + hk * a.k_h, *v = static_cast<const T*>(a.v) + b * a.v_b + hk * a.v_h;
    const int64_t at = ((static_cast<int64_t>(b) * a.Nq + n) * a.H + h) * d;
    const T* o = static_cast<const T*>(a.o) + at;
    T* dq = static_cast<T*>(a.dq) + at;
    const float lse = a.lse[row];
    const int len = n < clamp_len(a.q_lens, b, a.Nq) && lse != -INFINITY ? clamp_len(a.kv_lens, b, a.Nk) : 0;
    float delta = 0.0f, s0 = 0.0f, s1 = 0.0f;
    for (int c = lane; c < d; c += 64) {
        qs[wave][c] = static_cast<float>(q[c]) * a.scale;
        gs[wave][c] = static_cast<float>(g[c]);
        if (len) delta = fmaf(gs[wave][c], static_cast<float>(o[c]), delta);
    }
    delta = wave_sum(delta);
    for (int j0 = 0; j0 < len; j0 += 64) {
        const int j = j0 + lane;
        float ds = 0.0f;
        if (admitted(a, b, j, len)) ds = expf(dot(qs[wave], k + j * a.k_n, d) - lse) * (dot(gs[wave], v + j * a.v_n, d) - delta);
        for (int i = 0; i < 64 && j0 + i < len; ++i) {
            const float si = __shfl(ds, i, 64);
            if (si == 0.0f) continue;
            const T* ki = k + static_cast<int64_t>(j0 + i) * a.k_n;
            if (lane < d) s0 = fmaf(si, static_cast<float>(ki[lane]), s0);
            if (lane + 64 < d) s1 = fmaf(si, static_cast<float>(ki[lane + 64]), s1);
        }
    }
    if (lane < d) dq[lane] = static_cast<T>(s0 * a.scale);
    if (lane + 64 < d) dq[lane + 64] = static_cast<T>(s1 * a.scale);
}

// rows of k and v: waves over (b, hk, j); a key's sum runs over the query heads that share it
template <class T>
__global__ __launch_bounds__(256) void xattn_dkv_kernel(const Args a) {
    __shared__ float ks[4][128], vs[4][128];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, d = a.d;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * 4 + wave;
    if (row >= static_cast<int64_t>(a.B) * a.Hkv * a.Nk) return;
    const int j = row % a.Nk, hk = row / a.Nk % a.Hkv, b = row / a.Nk / a.Hkv, G = a.H / a.Hkv;
    const T *k = static_cast<const T*>(a.k) + b * a.k_b + j * a.k_n + hk * a.k_h, *v = static_cast<const T*>(a.v) + b * a.v_b + j * a.v_n + hk * a.v_h;
    const int rows = admitted(a, b, j, clamp_len(a.kv_lens, b, a.Nk)) ? clamp_len(a.q_lens, b, a.Nq) : 0;
    for (int c = lane; c < d; c += 64) {
        ks[wave][c] = static_cast<float>(k[c]) * a.scale;
        vs[wave][c] = static_cast<float>(v[c]);
    }
    float k0 = 0.0f, k1 = 0.0f, v0 = 0.0f, v1 = 0.0f;
    for (int h = hk * G; h < (hk + 1) * G; ++h)
        for (int n0 = 0; n0 < rows; n0 += 64) {
            const int n = n0 + lane;
            float p = 0.0f, ds = 0.0f;
            if (n < rows) {
                const T *q = static_cast<const T*>(a.q) + b * a.q_b + n * a.q_n + h * a.q_h, *g = static_cast<const T*>(a.dout) + b * a.do_b + n * a.do_n + h * a.do_h;
                const T* o = static_cast<const T*>(a.o) + ((static_cast<int64_t>(b) * a.Nq + n) * a.H + h) * d;
                float delta = 0.0f;
                for (int c = 0; c < d; ++c) delta = fmaf(static_cast<float>(g[c]), static_cast<float>(o[c]), delta);
                p = expf(dot(ks[wave], q, d) - a.lse[(static_cast<int64_t>(b) * a.H + h) * a.Nq + n]);
                ds = p * (dot(vs[wave], g, d) - delta);
            }
            for (int i = 0; i < 64 && n0 + i < rows; ++i) {
                const float pi = __shfl(p, i, 64), si = __shfl(ds, i, 64);
                const T *q = static_cast<const T*>(a.q) + b * a.q_b + (n0 + i) * a.q_n + h * a.q_h;
                const T *g = static_cast<const T*>(a.dout) + b * a.do_b + (n0 + i) * a.do_n + h * a.do_h;
                if (lane < d) { v0 = fmaf(pi, static_cast<float>(g[lane]), v0); k0 = fmaf(si, static_cast<float>(q[lane]), k0); }
                if (lane + 64 < d) { v1 = fmaf(pi, static_cast<float>(g[lane + 64]), v1); k1 = fmaf(si, static_cast<float>(q[lane + 64]), k1); }
            }
        }
    const int64_t at = ((static_cast<int64_t>(b) * a.Nk + j) * a.Hkv + hk) * d;
    T *dk = static_cast<T*>(a.dk) + at, *dv = static_cast<T*>(a.dv) + at;
    if (lane < d) { dk[lane] = static_cast<T>(k0 * a.scale); dv[lane] = static_cast<T>(v0); }
    if (lane + 64 < d) { dk[lane + 64] = static_cast<T>(k1 * a.scale); dv[lane + 64] = static_cast<T>(v1); }
}

int check(const char* who, const ogmm_xattn* a) {
    OGMM_REQUIRE(a, "%s: missing argument", who);
    OGMM_REQUIRE(a->B >= 0 && a->Nq >= 0 && a->Nk >= 0 && a->H >= 1 && a->Hkv >= 1, "%s: B = %d, Nq = %d, Nk = %d, H = %d, Hkv = %d", who, a->B, a->Nq, a->Nk, a->H, a->Hkv);
    OGMM_REQUIRE(a->H % a->Hkv == 0, "%s: %d query heads over %d key heads", who, a->H, a->Hkv);
    OGMM_REQUIRE(a->d >= 8 && a->d <= 128 && a->d % 8 == 0, "%s: head width %d (multiples of 8 up to 128 are supported)", who, a->d);
    OGMM_REQUIRE(a->type == OGMM_F32 || a->type == OGMM_BF16 || a->type == OGMM_F16, "%s: unknown type %d", who, a->type);
    const int64_t e = a->type == OGMM_F32 ? 4 : 2;
    const int64_t strides[] = {a->q_b, a->q_n, a->q_h, a->k_b, a->k_n, a->k_h, a->v_b, a->v_n, a->v_h};
    for (int64_t s : strides) OGMM_REQUIRE(s * e % 16 == 0, "%s: a stride of %lld elements is not a multiple of 16 bytes", who, static_cast<long long>(s));
    OGMM_REQUIRE(aligned16(a->q) && aligned16(a->k) && aligned16(a->v) && aligned16(a->o), "%s: addresses must be multiples of 16 bytes", who);
    OGMM_REQUIRE(isfinite(a->scale), "%s: scale must be finite", who);
    // (a workgroup takes several rows, so this keeps every grid below 2^31 workgroups and a row's number within 32 bits)
    OGMM_REQUIRE(static_cast<double>(a->B) * a->H * a->Nq < 2147483648.0 && static_cast<double>(a->B) * a->Hkv * a->Nk < 2147483648.0, "%s: more than 2^31 rows", who);
    const bool rows = a->B && a->Nq, keys = a->B && a->Nk;
    OGMM_REQUIRE(!rows || (a->q && a->o), "%s: missing argument", who);
    OGMM_REQUIRE(!keys || (a->k && a->v), "%s: missing argument", who);
    return 0;
}

template <class F>
int with_type(int type, F&& f) {
    if (type == OGMM_F32) return f(float());
    if (type == OGMM_BF16) return f(__bf16());
    return f(_Float16());
}

}  // namespace

extern "C" int64_t ogmm_xattn_workspace_bytes(const ogmm_xattn* a, int backward) { return 0; }

extern "C" int ogmm_xattn_fwd(const ogmm_xattn* a, void* stream) {
    if (check("ogmm_xattn_fwd", a)) return 1;
    const int64_t rows = static_cast<int64_t>(a->B) * a->H * a->Nq;
    if (!rows) return 0;
    return with_type(a->type, [&](auto t) {
        xattn_fwd_kernel<decltype(t)><<<static_cast<uint32_t>((rows + 3) / 4), 256, 0, as_stream(stream)>>>(Args{*a});
        return check_launch("ogmm_xattn_fwd");
    });
}

extern "C" int ogmm_xattn_bwd(const ogmm_xattn* a, void* stream) {
    if (check("ogmm_xattn_bwd", a)) return 1;
    const int64_t e = a->type == OGMM_F32 ? 4 : 2;
    OGMM_REQUIRE(a->do_b * e % 16 == 0 && a->do_n * e % 16 == 0 && a->do_h * e % 16 == 0 && aligned16(a->dout), "ogmm_xattn_bwd: dout's address and strides must be multiples of 16 bytes");
    OGMM_REQUIRE(aligned16(a->dq) && aligned16(a->dk) && aligned16(a->dv), "ogmm_xattn_bwd: addresses must be multiples of 16 bytes");
    const int64_t rows = static_cast<int64_t>(a->B) * a->H * a->Nq, keys = static_cast<int64_t>(a->B) * a->Hkv * a->Nk;
    OGMM_REQUIRE(!rows || (a->dout && a->lse && a->dq), "ogmm_xattn_bwd: missing argument");
    OGMM_REQUIRE(!keys || (a->dk && a->dv), "ogmm_xattn_bwd: missing argument");
    if (!rows && !keys) return 0;
    return with_type(a->type, [&](auto t) {
        if (rows) xattn_dq_kernel<decltype(t)><<<static_cast<uint32_t>((rows + 3) / 4), 256, 0, as_stream(stream)>>>(Args{*a});
        if (keys) xattn_dkv_kernel<decltype(t)><<<static_cast<uint32_t>((keys + 3) / 4), 256, 0, as_stream(stream)>>>(Args{*a});
        return check_launch("ogmm_xattn_bwd");
    });
}
