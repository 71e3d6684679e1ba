// Global norm of many gradient tensors, and their clipping:  n = inv_scale sqrt(sum g^2),  c = min(1, max_norm / (n + 1e-6)),  out = g * (inv_scale c).
//
// Bound by HBM: every value is read once for the norm, and read and written once more where the factor is not one.  The tensors travel as a table in the
// kernel arguments (no copy, nothing kept between calls, capturable); they are cut into chunks that the workgroups of one launch take in turn, so a hundred
// small tensors fill the part as well as one large one.  Squares are formed and summed in fp64 from the first value on: fp32 squares of gradients below 1e-19
// or above 1e19 leave its range, and the fp64 FMA rate is several times what the stream of values needs.  Every sum has a fixed order: results repeat bit for bit.
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

template <int N, bool OUT>
__device__ __forceinline__ int tensor_of(const Table<N, OUT>& t, int n, uint32_t chunk) {
    int lo = 0, hi = n - 1;          // the last tensor whose first chunk is not behind `chunk` (empty tensors share it with their successor)
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (t.first[mid] <= chunk) lo = mid; else hi = mid - 1;
    }
    return lo;
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

// f(values, where) over a chunk's values, VEC to a thread at once and four loads in flight; f1(place) for the last few
template <int BYTES, int VEC, class F, class F1>
__device__ __forceinline__ void over_chunk(const char* __restrict__ p, uint32_t len, F&& f, F1&& f1) {
    constexpr uint32_t ROUND = THREADS * VEC;
    constexpr int E = BYTES / VEC;
    uint32_t at = threadIdx.x * VEC;
    for (; at + 3 * ROUND + VEC <= len; at += 4 * ROUND) {
        Packed<BYTES> b[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) b[u] = *reinterpret_cast<const Packed<BYTES>*>(p + (at + u * ROUND) * E);
#pragma unroll
        for (int u = 0; u < 4; ++u) f(b[u], at + u * ROUND);
    }
    for (; at + VEC <= len; at += ROUND) f(*reinterpret_cast<const Packed<BYTES>*>(p + at * E), at);
    if (threadIdx.x < len % VEC) f1(len - len % VEC + threadIdx.x);
}

template <int N, bool OUT>
__global__ __launch_bounds__(THREADS) void grad_squares_kernel(const Table<N, OUT> t, int n, uint32_t chunks, uint32_t chunk_len, double* __restrict__ partial) {
    __shared__ double lds[THREADS / 64];
    double acc = 0.0;
    for (uint32_t c = blockIdx.x; c < chunks; c += gridDim.x) {
        const int i = tensor_of(t, n, c);
        const uint32_t off = (c - t.first[i]) * chunk_len, len = min(chunk_len, t.count[i] - off);
        const int type = t.type[i];
        if (type == OGMM_F32) {
            const float* p = static_cast<const float*>(t.g[i]) + off;
            over_chunk<16, 4>(reinterpret_cast<const char*>(p), len,
                [&](const Packed<16>& b, uint32_t) {
#pragma unroll
                    for (int k = 0; k < 4; ++k) { const double x = __uint_as_float(b.w[k]); acc = fma(x, x, acc); }
                },
                [&](uint32_t e) { const double x = p[e]; acc = fma(x, x, acc); });
        } else {
            const uint16_t* p = static_cast<const uint16_t*>(t.g[i]) + off;
            over_chunk<16, 8>(reinterpret_cast<const char*>(p), len,
                [&](const Packed<16>& b, uint32_t) {
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const double x = half_bits(b.w[k] & 0xffff, type), y = half_bits(b.w[k] >> 16, type);
                        acc = fma(x, x, acc);
                        acc = fma(y, y, acc);
                    }
                },
                [&](uint32_t e) { const double x = half_bits(p[e], type); acc = fma(x, x, acc); });
        }
    }
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
__global__ __launch_bounds__(THREADS) void grad_clip_kernel(const Table<N, OUT> t, int n, uint32_t chunks, uint32_t chunk_len, const double* __restrict__ partial,
                                                            int partials, double inv_scale, double max_norm, float* __restrict__ norm) {
    __shared__ double lds[THREADS / 64];
    const double total = norm_of(partial, partials, inv_scale, lds);
    if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = static_cast<float>(total);
    double c = max_norm / (total + 1e-6);
    if (c > 1.0) c = 1.0;          // (a NaN stays one: the gradients become NaN as they do in a plain product)
    const float f = static_cast<float>(c * inv_scale);
    if (!OUT && f == 1.0f) return;          // nothing changes
    for (uint32_t ch = blockIdx.x; ch < chunks; ch += gridDim.x) {
        const int i = tensor_of(t, n, ch);
        const uint32_t off = (ch - t.first[i]) * chunk_len, len = min(chunk_len, t.count[i] - off);
        const int type = t.type[i];
        if (type == OGMM_F32) {
            const float* p = static_cast<const float*>(t.g[i]) + off;
            float* o = OUT ? t.out[OUT ? i : 0] + off : static_cast<float*>(t.g[i]) + off;
            over_chunk<16, 4>(reinterpret_cast<const char*>(p), len,
                [&](Packed<16> b, uint32_t e) {
#pragma unroll
                    for (int k = 0; k < 4; ++k) b.w[k] = __float_as_uint(__uint_as_float(b.w[k]) * f);
                    *reinterpret_cast<Packed<16>*>(o + e) = b;
                },
                [&](uint32_t e) { o[e] = p[e] * f; });
        } else if (OUT) {          // four values to a thread: its sixteen bytes of output lie beside its neighbours'
            const uint16_t* p = static_cast<const uint16_t*>(t.g[i]) + off;
            float* o = t.out[OUT ? i : 0] + off;
            over_chunk<8, 4>(reinterpret_cast<const char*>(p), len,
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
            over_chunk<16, 8>(reinterpret_cast<const char*>(p), len,
                [&](Packed<16> b, uint32_t e) {
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        b.w[k] = to_half_bits(half_bits(b.w[k] & 0xffff, type) * f, type) | static_cast<uint32_t>(to_half_bits(half_bits(b.w[k] >> 16, type) * f, type)) << 16;
                    *reinterpret_cast<Packed<16>*>(p + e) = b;
                },
                [&](uint32_t e) { p[e] = to_half_bits(half_bits(p[e], type) * f, type); });
        }
    }
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

// Chunks so large that a workgroup takes about eight of them, within 4096 values (one load of sixteen bytes a thread) and 32768
uint32_t chunk_length(int64_t total) {
    uint32_t len = 4096;
    while (len < 32768 && total > static_cast<int64_t>(len) * MAX_BLOCKS * 8) len *= 2;
    return len;
}

template <class T, bool OUT>
int fill(T& t, const std::vector<Item>& items, size_t from, uint32_t len, uint32_t* chunks) {
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
        at += (it.count + len - 1) / len;
    }
    t.first[n] = at;
    *chunks = at;
    return n;
}

int64_t total_of(const std::vector<Item>& items) {
    int64_t s = 0;
    for (const Item& it : items) s += it.count;
    return s;
}

int launch_squares(const std::vector<Item>& items, uint32_t len, double* partial, int* partials, hipStream_t stream) {
    *partials = 0;
    for (size_t from = 0; from < items.size();) {
        InPlace t;
        uint32_t chunks;
        const int n = fill<InPlace, false>(t, items, from, len, &chunks);
        const int blocks = static_cast<int>(std::min<uint32_t>(chunks, MAX_BLOCKS));
        grad_squares_kernel<<<blocks, THREADS, 0, stream>>>(t, n, chunks, len, partial + *partials);
        *partials += blocks;
        from += n;
    }
    return check_launch("ogmm_grad_norm");
}

template <class T, bool OUT>
void launch_clip(const std::vector<Item>& items, uint32_t len, const double* partial, int partials, double inv_scale, double max_norm, float* norm, hipStream_t stream) {
    for (size_t from = 0; from < items.size();) {
        T t;
        uint32_t chunks;
        const int n = fill<T, OUT>(t, items, from, len, &chunks);
        grad_clip_kernel<<<std::min<uint32_t>(chunks, MAX_BLOCKS), THREADS, 0, stream>>>(t, n, chunks, len, partial, partials, inv_scale, max_norm, from ? nullptr : norm);
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
        if (launch_squares(items, chunk_length(total_of(items)), partial, &partials, as_stream(stream))) return 1;
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
        const uint32_t len = chunk_length(total_of(items));
        int partials;
        double* partial = static_cast<double*>(workspace);
        if (launch_squares(items, len, partial, &partials, as_stream(stream))) return 1;
        if (items.empty())
            grad_norm_finish_kernel<<<1, THREADS, 0, as_stream(stream)>>>(partial, 0, inv_scale, norm);
        else if (out)
            launch_clip<OutOfPlace, true>(items, len, partial, partials, inv_scale, max_norm, norm, as_stream(stream));
        else
            launch_clip<InPlace, false>(items, len, partial, partials, inv_scale, max_norm, norm, as_stream(stream));
        return check_launch("ogmm_clip_grads");
    });
}
