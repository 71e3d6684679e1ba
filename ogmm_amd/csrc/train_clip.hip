// Global norm of many gradient tensors, and their clipping:  n = inv_scale sqrt(sum g^2),  c = min(1, max_norm / (n + 1e-6)),  out = g * (inv_scale c).
//
// Bound by HBM: every value is read once for the norm, and read and written once more where the factor is not one.  The tensors travel as a table in the
// kernel arguments (no copy, nothing kept between calls, capturable); each workgroup takes an equal run of their values, so a hundred small tensors
// fill the part as well as one large one.  Squares are summed in fp64: four or eight of them in fp32 first, where
// that is inside its range.  Every sum has a fixed order: results repeat bit for bit.
//
// Measured: 150 fp32 tensors, 13 M values: 14 us for the norm and 4 for finding that nothing changes (52 MB, out of the last-level cache), under 30 us of listing them on the host;
// 400 bf16 tensors, 300 M values, clipped to fp32: 2 x 80 us for the norm = 3.8 TB/s (a large sum reads at 3.95), 3 x 128 us for the product = 4.7 TB/s (a copy: 5.2).
#include "ogmm_common.h"
#include <algorithm>
#include <exception>
#include <math.h>
#include <vector>

namespace {

using namespace ogmm;

constexpr int THREADS = 1024;
// 512 workgroups of 1024 threads are all the waves that the 256 CUs hold; with one partial sum each the second kernel can add them up by itself in every workgroup
constexpr int MAX_BLOCKS = 512;
constexpr uint32_t CHUNK = 4096;            // what the work is dealt in: a load of sixteen bytes for each thread (fp32)
constexpr int64_t PIECE = 1 << 30;          // a longer tensor goes into the table as several pieces, so that sizes fit 32 bits

// A launch's tensors; the kernel argument segment is 4 KB: 230 tensors by one address, or 156 by two (out of place)
template <int N, bool OUT>
struct Table {
    void* g[N];
    float* out[OUT ? N : 1];
    uint32_t count[N];
    uint32_t first[N + 1];          // chunks before this tensor's
    uint8_t type[N];
};
using InPlace = Table<230, false>;
using OutOfPlace = Table<156, true>;
static_assert(sizeof(InPlace) <= 4032 && sizeof(OutOfPlace) <= 4032, "kernel arguments");

__device__ __forceinline__ float half_bits(uint32_t h, int type) {
    if (type == OGMM_BF16) return __uint_as_float(h << 16);
    return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(h)));
}

// Workgroups take runs of `run` chunks in turn (few tensors: one run each): f(tensor, first value, how many) for each tensor that a run touches
template <int N, bool OUT, class F>
__device__ __forceinline__ void over_runs(const Table<N, OUT>& t, int n, uint32_t run, F&& f) {
    const uint32_t chunks = t.first[n];
    int lo = 0;
    for (uint32_t c = blockIdx.x * run; c < chunks; c += (gridDim.x - 1) * run) {
        const uint32_t end = min(c + run, chunks);
        for (int hi = n - 1; lo < hi;) {          // the last tensor whose first chunk is not behind c
            const int mid = (lo + hi + 1) >> 1;
            if (t.first[mid] <= c) lo = mid; else hi = mid - 1;
        }
        for (;; ++lo) {
            const uint32_t stop = min(end, t.first[lo + 1]), off = (c - t.first[lo]) * CHUNK;
            f(lo, off, min((stop - c) * CHUNK, t.count[lo] - off));
            c = stop;
            if (c >= end) break;
        }
        if (end == chunks) break;
    }
}

__device__ __forceinline__ double block_sum(double v, double* lds) {
    v = wave_sum_d(v);
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    double s = 0.0;
    for (int i = 0; i < THREADS / 64; ++i) s += lds[i];
    return s;
}

// bytes at an address of any alignment that the element has
template <int BYTES> struct __attribute__((packed, aligned(2))) Packed { uint32_t w[BYTES / 4]; };

// f(values, where) over a run's values, VEC to a thread at once and AHEAD loads in flight; f1(place) for single ones: those in front of the first place at which `by` (the run's first
// value as it is read or written) is aligned to VEC values of its own, and the last few.  A tensor may start anywhere in a bucket, and loads that straddle lines cost more.
template <int BYTES, int VEC, int AHEAD, class P, class F, class F1>
__device__ __forceinline__ void over_values(const char* __restrict__ p, const P* by, uint32_t len, F&& f, F1&& f1) {
    constexpr uint32_t ROUND = THREADS * VEC;
    constexpr int E = BYTES / VEC;
    const uint32_t lead = min(len, static_cast<uint32_t>(-(reinterpret_cast<uintptr_t>(by) / sizeof(P)) % VEC)), tail = (len - lead) % VEC;
    uint32_t at = lead + threadIdx.x * VEC;
    for (; at + (AHEAD - 1) * ROUND + VEC <= len; at += AHEAD * ROUND) {
        Packed<BYTES> b[AHEAD];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) b[u] = *reinterpret_cast<const Packed<BYTES>*>(p + static_cast<size_t>(at + u * ROUND) * E);
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) f(b[u], at + u * ROUND);
    }
    if (at + VEC <= len) {          // what is left, fewer than AHEAD: together too
        Packed<BYTES> b[AHEAD - 1];
#pragma unroll
        for (int u = 0; u < AHEAD - 1; ++u)
            if (at + u * ROUND + VEC <= len) b[u] = *reinterpret_cast<const Packed<BYTES>*>(p + static_cast<size_t>(at + u * ROUND) * E);
#pragma unroll
        for (int u = 0; u < AHEAD - 1; ++u)
            if (at + u * ROUND + VEC <= len) f(b[u], at + u * ROUND);
    }
    if (threadIdx.x < lead) f1(threadIdx.x);
    if (threadIdx.x < tail) f1(len - tail + threadIdx.x);
}

// acc += the squares of N values.  They are added up in fp32 first, where their sum stands well inside its range (their roundings are of random sign, 2^-24 at most); a group outside
// it -- 1e-19 and 1e19 are the roots -- is formed in fp64.  A conversion to fp64 and its multiplication take six times an fp32 one.
template <int N>
__device__ __forceinline__ void add_squares(double& acc, const float (&x)[N]) {
    float s = x[0] * x[0];
#pragma unroll
    for (int k = 1; k < N; ++k) s = fmaf(x[k], x[k], s);
    if (s > 1e-30f && s < 1e30f) {
        acc += s;
    } else {
#pragma unroll
        for (int k = 0; k < N; ++k) acc = fma(static_cast<double>(x[k]), static_cast<double>(x[k]), acc);
    }
}

template <int N, bool OUT>
__global__ __launch_bounds__(THREADS, 8) void grad_squares_kernel(const Table<N, OUT> t, int n, uint32_t run, double* __restrict__ partial) {
    __shared__ double lds[THREADS / 64];
    double acc = 0.0;
    over_runs(t, n, run, [&](int i, uint32_t off, uint32_t len) {
        const int type = t.type[i];
        if (type == OGMM_F32) {
            const float* p = static_cast<const float*>(t.g[i]) + off;
            over_values<16, 4, 4>(reinterpret_cast<const char*>(p), p, len,
                [&](const Packed<16>& b, uint32_t) {
                    const float x[4] = {__uint_as_float(b.w[0]), __uint_as_float(b.w[1]), __uint_as_float(b.w[2]), __uint_as_float(b.w[3])};
                    add_squares(acc, x);
                },
                [&](uint32_t e) { const double x = p[e]; acc = fma(x, x, acc); });
        } else {
            const uint16_t* p = static_cast<const uint16_t*>(t.g[i]) + off;
            over_values<16, 8, 4>(reinterpret_cast<const char*>(p), p, len,
                [&](const Packed<16>& b, uint32_t) {
                    float x[8];
#pragma unroll
                    for (int k = 0; k < 4; ++k) { x[2 * k] = half_bits(b.w[k] & 0xffff, type); x[2 * k + 1] = half_bits(b.w[k] >> 16, type); }
                    add_squares(acc, x);
                },
                [&](uint32_t e) { const double x = half_bits(p[e], type); acc = fma(x, x, acc); });
        }
    });
    const double s = block_sum(acc, lds);
    if (threadIdx.x == 0) partial[blockIdx.x] = s;
}

__device__ __forceinline__ double norm_of(const double* __restrict__ partial, int partials, double inv_scale, double* lds) {
    double acc = 0.0;
    for (int i = threadIdx.x; i < partials; i += THREADS) acc += partial[i];
    return sqrt(block_sum(acc, lds)) * inv_scale;
}

__global__ __launch_bounds__(THREADS) void grad_norm_finish_kernel(const double* __restrict__ partial, int partials, double inv_scale, float* __restrict__ norm) {
    __shared__ double lds[THREADS / 64];
    const double n = norm_of(partial, partials, inv_scale, lds);
    if (threadIdx.x == 0) *norm = static_cast<float>(n);
}

template <int N, bool OUT>
__global__ __launch_bounds__(THREADS, 8) void grad_clip_kernel(const Table<N, OUT> t, int n, uint32_t run, const double* __restrict__ partial, int partials, double inv_scale, double max_norm,
                                                            float* __restrict__ norm) {
    __shared__ double lds[THREADS / 64];
    const double total = norm_of(partial, partials, inv_scale, lds);
    if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = static_cast<float>(total);
    double c = max_norm / (total + 1e-6);
    if (c > 1.0 || (isinf(max_norm) && isinf(total))) c = 1.0;          // (without a limit nothing is clipped; a NaN stays one: the gradients become NaN as they do in a plain product)
    const float f = static_cast<float>(c * inv_scale);
    if (!OUT && f == 1.0f) return;          // nothing changes
    over_runs(t, n, run, [&](int i, uint32_t off, uint32_t len) {
        const int type = t.type[i];
        if (type == OGMM_F32) {
            const float* p = static_cast<const float*>(t.g[i]) + off;
            float* o = OUT ? t.out[OUT ? i : 0] + off : static_cast<float*>(t.g[i]) + off;
            over_values<16, 4, 4>(reinterpret_cast<const char*>(p), o, len,
                [&](Packed<16> b, uint32_t e) {
#pragma unroll
                    for (int k = 0; k < 4; ++k) b.w[k] = __float_as_uint(__uint_as_float(b.w[k]) * f);
                    *reinterpret_cast<Packed<16>*>(o + e) = b;
                },
                [&](uint32_t e) { o[e] = p[e] * f; });
        } else if (OUT) {          // four values to a thread: its sixteen bytes of output lie beside its neighbours'
            const uint16_t* p = static_cast<const uint16_t*>(t.g[i]) + off;
            float* o = t.out[OUT ? i : 0] + off;
            over_values<8, 4, 8>(reinterpret_cast<const char*>(p), o, len,
                [&](const Packed<8>& b, uint32_t e) {
                    Packed<16> r;
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        r.w[2 * k] = __float_as_uint(half_bits(b.w[k] & 0xffff, type) * f);
                        r.w[2 * k + 1] = __float_as_uint(half_bits(b.w[k] >> 16, type) * f);
                    }
                    *reinterpret_cast<Packed<16>*>(o + e) = r;
                },
                [&](uint32_t e) { o[e] = half_bits(p[e], type) * f; });
        } else {
            uint16_t* p = static_cast<uint16_t*>(t.g[i]) + off;
            over_values<16, 8, 4>(reinterpret_cast<const char*>(p), p, len,
                [&](Packed<16> b, uint32_t e) {
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        b.w[k] = to_half_bits(half_bits(b.w[k] & 0xffff, type) * f, type) | static_cast<uint32_t>(to_half_bits(half_bits(b.w[k] >> 16, type) * f, type)) << 16;
                    *reinterpret_cast<Packed<16>*>(p + e) = b;
                },
                [&](uint32_t e) { p[e] = to_half_bits(half_bits(p[e], type) * f, type); });
        }
    });
}

struct Item { void* g; float* out; uint32_t count; uint8_t type; };

size_t width(int type) { return type == OGMM_F32 ? 4 : 2; }

int check_list(const char* who, int n, const void* const* grads, const int64_t* numel, const int32_t* types) {
    OGMM_REQUIRE(n >= 0 && (n == 0 || (grads && numel && types)), "%s: missing argument", who);
    for (int i = 0; i < n; ++i) {
        OGMM_REQUIRE(numel[i] >= 0, "%s: tensor %d has a negative size", who, i);
        OGMM_REQUIRE(types[i] == OGMM_F32 || types[i] == OGMM_BF16 || types[i] == OGMM_F16, "%s: tensor %d has an unknown type %d", who, i, types[i]);
        OGMM_REQUIRE(!numel[i] || grads[i], "%s: tensor %d is null", who, i);
        OGMM_REQUIRE(reinterpret_cast<uintptr_t>(grads[i]) % width(types[i]) == 0, "%s: tensor %d is not aligned to its elements", who, i);
    }
    return 0;
}

// A value that two entries of the list write, or that one writes and another reads, would come out by chance: refused.
int check_apart(const char* who, int n, const void* const* grads, const int64_t* numel, const int32_t* types, void* const* out) {
    struct Span { uintptr_t lo, hi; int i; };
    std::vector<Span> w;
    w.reserve(n);
    for (int i = 0; i < n; ++i)
        if (numel[i]) {
            const uintptr_t lo = reinterpret_cast<uintptr_t>(out ? out[i] : grads[i]);
            w.push_back({lo, lo + numel[i] * (out ? 4 : width(types[i])), i});
        }
    std::sort(w.begin(), w.end(), [](const Span& a, const Span& b) { return a.lo < b.lo; });
    for (size_t k = 1; k < w.size(); ++k)
        OGMM_REQUIRE(w[k].lo >= w[k - 1].hi, "%s: tensors %d and %d share memory that is written", who, w[k - 1].i, w[k].i);
    if (!out) return 0;
    for (int i = 0; i < n; ++i) {
        if (!numel[i]) continue;
        const uintptr_t lo = reinterpret_cast<uintptr_t>(grads[i]), hi = lo + numel[i] * width(types[i]);
        auto it = std::upper_bound(w.begin(), w.end(), lo, [](uintptr_t v, const Span& s) { return v < s.hi; });          // the first span that ends behind lo
        for (; it != w.end() && it->lo < hi; ++it)
            OGMM_REQUIRE(it->i == i && it->lo == lo && types[i] == OGMM_F32, "%s: an output shares memory with gradient %d", who, i);
    }
    return 0;
}

void pieces_of(int n, const void* const* grads, const int64_t* numel, const int32_t* types, void* const* out, std::vector<Item>& items) {
    items.reserve(n);
    for (int i = 0; i < n; ++i)
        for (int64_t at = 0; at < numel[i]; at += PIECE)
            items.push_back({const_cast<char*>(static_cast<const char*>(grads[i])) + at * width(types[i]), out ? static_cast<float*>(out[i]) + at : nullptr,
                             static_cast<uint32_t>(std::min(PIECE, numel[i] - at)), static_cast<uint8_t>(types[i])});
}

template <class T, bool OUT>
int fill(T& t, const std::vector<Item>& items, size_t from) {
    constexpr size_t cap = sizeof(t.count) / sizeof(t.count[0]);
    const int n = static_cast<int>(std::min(cap, items.size() - from));
    uint32_t at = 0;
    for (int k = 0; k < n; ++k) {
        const Item& it = items[from + k];
        t.g[k] = it.g;
        if (OUT) t.out[OUT ? k : 0] = it.out;
        t.count[k] = it.count;
        t.type[k] = it.type;
        t.first[k] = at;
        at += (it.count + CHUNK - 1) / CHUNK;
    }
    t.first[n] = at;
    return n;
}

// How `chunks` are dealt: equal runs, one to a workgroup as long as that is 16 chunks or less.  (13 M values of 150 tensors: one run each 14 us, single chunks in turn 19; 300 M: runs
// of 65536 values keep the workgroups' reads closer together than one run each would)
struct Deal { int blocks; uint32_t run; };
Deal deal(uint32_t chunks) {
    const uint32_t rounds = std::max<uint32_t>(1, (chunks + 16 * MAX_BLOCKS - 1) / (16 * MAX_BLOCKS)), run = std::max<uint32_t>(1, (chunks + MAX_BLOCKS * rounds - 1) / (MAX_BLOCKS * rounds));
    return {static_cast<int>(std::min<uint32_t>((chunks + run - 1) / run, MAX_BLOCKS)), run};
}

int launch_squares(const std::vector<Item>& items, double* partial, int* partials, hipStream_t stream) {
    *partials = 0;
    for (size_t from = 0; from < items.size();) {
        InPlace t;
        const int n = fill<InPlace, false>(t, items, from);
        const Deal d = deal(t.first[n]);
        grad_squares_kernel<<<d.blocks, THREADS, 0, stream>>>(t, n, d.run, partial + *partials);
        *partials += d.blocks;
        from += n;
    }
    return check_launch("ogmm_grad_norm");
}

template <class T, bool OUT>
void launch_clip(const std::vector<Item>& items, const double* partial, int partials, double inv_scale, double max_norm, float* norm, hipStream_t stream) {
    for (size_t from = 0; from < items.size();) {
        T t;
        const int n = fill<T, OUT>(t, items, from);
        const Deal d = deal(t.first[n]);
        grad_clip_kernel<<<d.blocks, THREADS, 0, stream>>>(t, n, d.run, partial, partials, inv_scale, max_norm, from ? nullptr : norm);
        from += n;
    }
}

}  // namespace

extern "C" int64_t ogmm_grad_norm_workspace_bytes(int n, const int64_t* numel) {
    if (n < 0 || (n && !numel)) return -1;
    int64_t pieces = 0;
    for (int i = 0; i < n; ++i) pieces += numel[i] <= 0 ? 0 : (numel[i] + PIECE - 1) / PIECE;
    return std::max<int64_t>(1, (pieces + 229) / 230) * MAX_BLOCKS * static_cast<int64_t>(sizeof(double));
}

// (the lists are held in vectors: an allocation that fails becomes an error code at the C boundary)
template <class F>
static int guarded(const char* who, F&& f) {
    try {
        return f();
    } catch (const std::exception& e) {
        return ogmm::fail("%s: %s", who, e.what());
    }
}

extern "C" int ogmm_grad_norm(int n, const void* const* grads, const int64_t* numel, const int32_t* types, float inv_scale, float* norm, void* workspace, void* stream) {
    OGMM_REQUIRE(norm && workspace, "ogmm_grad_norm: missing argument");
    OGMM_REQUIRE(isfinite(inv_scale) && inv_scale > 0.0f, "ogmm_grad_norm: inv_scale must be positive and finite");
    if (check_list("ogmm_grad_norm", n, grads, numel, types)) return 1;
    return guarded("ogmm_grad_norm", [&] {
        std::vector<Item> items;
        pieces_of(n, grads, numel, types, nullptr, items);
        int partials;
        double* partial = static_cast<double*>(workspace);
        if (launch_squares(items, partial, &partials, as_stream(stream))) return 1;
        grad_norm_finish_kernel<<<1, THREADS, 0, as_stream(stream)>>>(partial, partials, inv_scale, norm);
        return check_launch("ogmm_grad_norm");
    });
}

extern "C" int ogmm_clip_grads(int n, const void* const* grads, const int64_t* numel, const int32_t* types, void* const* out, float inv_scale, float max_norm, float* norm,
                               void* workspace, void* stream) {
    OGMM_REQUIRE(norm && workspace, "ogmm_clip_grads: missing argument");
    OGMM_REQUIRE(isfinite(inv_scale) && inv_scale > 0.0f, "ogmm_clip_grads: inv_scale must be positive and finite");
    OGMM_REQUIRE(max_norm >= 0.0f, "ogmm_clip_grads: max_norm must not be negative");
    if (check_list("ogmm_clip_grads", n, grads, numel, types)) return 1;
    for (int i = 0; out && i < n; ++i)
        OGMM_REQUIRE(!numel[i] || (out[i] && reinterpret_cast<uintptr_t>(out[i]) % 4 == 0), "ogmm_clip_grads: output %d is null or not aligned to its elements", i);
    return guarded("ogmm_clip_grads", [&] {
        if (check_apart("ogmm_clip_grads", n, grads, numel, types, out)) return 1;
        std::vector<Item> items;
        pieces_of(n, grads, numel, types, out, items);
        int partials;
        double* partial = static_cast<double*>(workspace);
        if (launch_squares(items, partial, &partials, as_stream(stream))) return 1;
        if (items.empty())
            grad_norm_finish_kernel<<<1, THREADS, 0, as_stream(stream)>>>(partial, 0, inv_scale, norm);
        else if (out)
            launch_clip<OutOfPlace, true>(items, partial, partials, inv_scale, max_norm, norm, as_stream(stream));
        else
            launch_clip<InPlace, false>(items, partial, partials, inv_scale, max_norm, norm, as_stream(stream));
        return check_launch("ogmm_clip_grads");
    });
}
