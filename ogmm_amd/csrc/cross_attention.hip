// Cross attention to states of another length (include/ogmm_hip.h, L1), forward and backward.
//
// Forward, one pass over the keys with a running maximum and sum.  A workgroup has four waves; a wave owns 32 query rows and forms S^T = K Q^T, so that a lane holds one
// query's scores (32x32 result: column = lane % 32, rows 8 (i / 4) + 4 (lane / 32) + i % 4): maximum, exponential and sum stay inside the lane but for one exchange with
// lane ^ 32, and P^T is the next product's operand as it lies, O^T = V^T P^T, with V's keys taken in the order in which the lanes hold them.  The G query heads of a key
// head are rows of one tile (row = n G + g): their keys are read once.
#include "ogmm_common.h"
#include <algorithm>
#include <math.h>
#include <type_traits>

namespace {

using namespace ogmm;

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

struct Args : ogmm_xattn {
    int G, rows;                   // query heads to a key head, query rows to a key head (Nq G)
    int tiles, splits;             // row tiles, parts of the keys
    uint32_t items, per_xcd;       // workgroups in all, and of one XCD
    float* part;                   // splits > 1: [items of a split][rows of a tile][d] sums and, behind them, (maximum, sum) pairs
    float* part_ml;
};

__device__ __forceinline__ int clamp_len(const int32_t* lens, int b, int n) { return lens ? max(0, min(n, lens[b])) : n; }

// Workgroups go to the XCDs in turn; those of one (batch, key head) read the same keys, so each XCD gets a run of neighbours for its own L2
__device__ __forceinline__ uint32_t item_of(const Args& a) { return blockIdx.x % 8 * a.per_xcd + blockIdx.x / 8; }

// ---- products of 32x32 tiles, sixteen bytes of either operand to a lane: row lane % 32, byte 16 (lane / 32) of a 32-byte chunk of the contraction
__device__ __forceinline__ void mma(f32x16& c, u32x4 a, u32x4 b, __bf16) {
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ void mma(f32x16& c, u32x4 a, u32x4 b, _Float16) {
    c = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ void mma(f32x16& c, u32x4 a, u32x4 b, float) {
#pragma unroll
    for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a[j]), __uint_as_float(b[j]), c, 0, 0, 0);
}

// A matrix of rows in LDS: ROW bytes and a gap that sets neighbouring rows 16 (or 32) bytes apart in the banks
template <class T, int DP, int PAD>
struct Tile {
    static constexpr int ROW = DP * sizeof(T), PITCH = ROW + PAD, CHUNKS = ROW / 32, DB = DP / 32;

    // row lane % 32 of a block of 32 rows, chunk s of its channels
    static __device__ __forceinline__ u32x4 row_chunk(const char* lds, int row0, int s) {
        const int lane = threadIdx.x & 63;
        return *reinterpret_cast<const u32x4*>(lds + (row0 + (lane & 31)) * PITCH + 32 * s + 16 * (lane >> 5));
    }

    // c[db] += X^T Y for the 32 rows from row0 as contraction: X = this matrix (its channels are the result's rows), y = 32 rows x 32 columns as a product's result holds it.
    // 16-bit: channel 32 db + row of the result; the transposing read gives a lane four rows of one channel.  fp32: channel DB row + db.
    static __device__ __forceinline__ void mul_t(f32x16 (&c)[DB], const char* lds, int row0, const u32x4 (&y)[sizeof(T) == 4 ? 4 : 2]) {
        const int lane = threadIdx.x & 63;
        if constexpr (sizeof(T) == 2) {
            const char* p = lds + (row0 + 4 * (lane >> 5) + (lane & 15) / 4) * PITCH + (lane & 16) * 2 + (lane & 3) * 8;
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int db = 0; db < DB; ++db) {
                    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + 16 * t * PITCH + 64 * db));
                    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + (16 * t + 8) * PITCH + 64 * db));
                    mma(c[db], __builtin_bit_cast(u32x4, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7)), y[t], T());
                }
        } else {
            const char* p = lds + (row0 + 4 * (lane >> 5)) * PITCH + (lane & 31) * 4 * DB;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                float x[DB];
                __builtin_memcpy(x, __builtin_assume_aligned(p + (8 * (i / 4) + i % 4) * PITCH, DB == 3 ? 4 : 4 * DB), 4 * DB);
#pragma unroll
                for (int db = 0; db < DB; ++db) c[db] = __builtin_amdgcn_mfma_f32_32x32x2f32(x[db], __uint_as_float(y[i / 4][i % 4]), c[db], 0, 0, 0);
            }
        }
    }

    // the channel of element i of block db of such a result
    static __device__ __forceinline__ int channel(int db, int i) {
        const int r = 8 * (i / 4) + 4 * ((threadIdx.x & 63) >> 5) + i % 4;
        return sizeof(T) == 2 ? 32 * db + r : DB * r + db;
    }
};

// a result's 32x32 values as the next product's operand
template <class T>
__device__ __forceinline__ void as_operand(u32x4 (&y)[sizeof(T) == 4 ? 4 : 2], const f32x16& x) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 16; ++i) y[i / 4][i % 4] = __float_as_uint(x[i]);
    } else {
        typedef T t8 __attribute__((ext_vector_type(8)));
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            t8 v;
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = static_cast<T>(x[8 * t + i]);          // (rounded to nearest: one half step of the type on each weight, its sum stays fp32)
            y[t] = __builtin_bit_cast(u32x4, v);
        }
    }
}

__device__ __forceinline__ float other_half(float v) { return __shfl_xor(v, 32, 64); }

// Which of the 64 keys from n0 are admitted, one bit each (the same in every wave)
__device__ __forceinline__ uint64_t key_bits(const Args& a, int b, int n0, int len) {
    const int n = n0 + (threadIdx.x & 63);
    return __ballot(n < len && (!a.key_mask || a.key_mask[b * a.mask_b + n]));
}

template <class T, int DP, bool KEY_WAVES>
struct Fwd {
    // keys of a tile: enough products between two barriers, and so little LDS that two workgroups share a CU
    static constexpr int KT = KEY_WAVES ? 128 : sizeof(T) == 4 && DP > 64 ? 32 : 64;
    using K = Tile<T, DP, 16>;
    using V = Tile<T, DP, sizeof(T) == 4 ? 16 : 32>;
    static constexpr int ROWS = KEY_WAVES ? 32 : 128;
    static constexpr int TILE_BYTES = KT * (K::PITCH + V::PITCH);
    // the four waves' sums side by side at the end
    static constexpr int LDS = KEY_WAVES ? std::max(TILE_BYTES, 4 * 32 * (DP + 4) * 4 + 4 * 32 * 8) : TILE_BYTES;
    static constexpr int CPR = K::ROW / 16, PASSES = KT * CPR / 256;          // chunks of sixteen bytes to a row, rounds of 256 threads to a tile
};

// rows [n0, n0 + KT) of k or v in registers (rows behind the padded end: some row that is there; channels behind d: zeros)
template <class T, int CPR, int PASSES>
__device__ __forceinline__ void fetch(u32x4 (&r)[PASSES], const T* __restrict__ x, int64_t step, int n0, int n, int d) {
    const int c = threadIdx.x % CPR;
    const bool there = c * 16 < d * static_cast<int>(sizeof(T));
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
        const int row = min(n0 + static_cast<int>(threadIdx.x) / CPR + i * (256 / CPR), n - 1);
        r[i] = u32x4{0, 0, 0, 0};
        if (there) r[i] = *reinterpret_cast<const u32x4*>(reinterpret_cast<const char*>(x + row * step) + 16 * c);
    }
}

// ... and from there to LDS; a row that is not admitted becomes zeros: what stands there may be anything, and 0 x NaN is no 0
template <int PITCH, int CPR, int PASSES, int WORDS>
__device__ __forceinline__ void put(char* lds, const u32x4 (&r)[PASSES], const uint64_t (&bits)[WORDS], bool full) {
    const int c = threadIdx.x % CPR;
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
        const int row = static_cast<int>(threadIdx.x) / CPR + i * (256 / CPR);
        u32x4 v = r[i];
        if (!full && !(bits[WORDS == 1 ? 0 : row >> 6] >> (row & 63) & 1)) v = u32x4{0, 0, 0, 0};
        *reinterpret_cast<u32x4*>(lds + row * PITCH + 16 * c) = v;
    }
}

template <class T, int DP, bool KEY_WAVES>
__global__ __launch_bounds__(256, (Fwd<T, DP, KEY_WAVES>::LDS > 81920 ? 1 : 2)) void xattn_fwd_kernel(const Args a) {
    using S = Fwd<T, DP, KEY_WAVES>;
    using K = typename S::K;
    using V = typename S::V;
    constexpr int KT = S::KT, WORDS = KT > 64 ? KT / 64 : 1, BLOCKS = KEY_WAVES ? 1 : KT / 32, DB = K::DB;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    char *lds_k = lds, *lds_v = lds + KT * K::PITCH;
    const uint32_t item = item_of(a);
    if (item >= a.items) return;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int split = item % a.splits, tile = item / a.splits % a.tiles, bh = item / a.splits / a.tiles, hk = bh % a.Hkv, b = bh / a.Hkv;
    const int len = clamp_len(a.kv_lens, b, a.Nk), q_rows = clamp_len(a.q_lens, b, a.Nq) * a.G;
    const T *k = static_cast<const T*>(a.k) + b * a.k_b + hk * a.k_h, *v = static_cast<const T*>(a.v) + b * a.v_b + hk * a.v_h;
    // this lane's query row
    const int row = tile * S::ROWS + (KEY_WAVES ? 0 : wave * 32) + (lane & 31), n = row / a.G, g = row - n * a.G;
    const bool row_there = row < q_rows;
    u32x4 q[K::CHUNKS];
    const float c = a.scale == 0.0f ? 1.0f : fabsf(a.scale) * LOG2E;          // (scale = 0: no score, whatever the queries are)
    {
        const char* p = reinterpret_cast<const char*>(static_cast<const T*>(a.q) + b * a.q_b + n * a.q_n + (hk * a.G + g) * a.q_h);
        const uint32_t flip = a.scale < 0.0f ? (sizeof(T) == 4 ? 0x80000000u : 0x80008000u) : 0u;          // a negative scale: the queries' signs
#pragma unroll
        for (int s = 0; s < K::CHUNKS; ++s) {
            q[s] = u32x4{0, 0, 0, 0};
            if (row_there && a.scale != 0.0f && 32 * s + 16 * (lane >> 5) < a.d * static_cast<int>(sizeof(T))) q[s] = *reinterpret_cast<const u32x4*>(p + 32 * s + 16 * (lane >> 5)) ^ flip;
        }
    }
    const int key_tiles = tile * S::ROWS < q_rows ? (len + KT - 1) / KT : 0, per = (key_tiles + a.splits - 1) / a.splits;
    const int end = min(key_tiles, (split + 1) * per);
    float m = -INFINITY, l = 0.0f;          // m: of scale S log2(e), the running maximum or up to 8 below it
    f32x16 o[DB] = {};
    u32x4 rk[S::PASSES], rv[S::PASSES];
    uint64_t bits[WORDS], next_bits[WORDS];
    auto next = [&](int t) {          // the first tile from t on that has an admitted key
        for (; t < end; ++t) {
            uint64_t any = 0;
#pragma unroll
            for (int w = 0; w < WORDS; ++w) any |= next_bits[w] = key_bits(a, b, t * KT + 64 * w, KT < 64 ? min(len, (t + 1) * KT) : len);
            if (any) break;
        }
        return t;
    };
    int t = next(split * per);
    if (t < end) {
        fetch<T, S::CPR>(rk, k, a.k_n, t * KT, a.Nk, a.d);
        fetch<T, S::CPR>(rv, v, a.v_n, t * KT, a.Nk, a.d);
    }
    while (t < end) {
        constexpr uint64_t ALL = KT < 64 ? (uint64_t(1) << (KT & 63)) - 1 : ~uint64_t(0);
        bool full = true;
#pragma unroll
        for (int w = 0; w < WORDS; ++w) { bits[w] = next_bits[w]; full &= bits[w] == ALL; }
        put<K::PITCH, S::CPR>(lds_k, rk, bits, full);
        put<V::PITCH, S::CPR>(lds_v, rv, bits, full);
        __syncthreads();
        t = next(t + 1);
        if (t < end) {
            fetch<T, S::CPR>(rk, k, a.k_n, t * KT, a.Nk, a.d);
            fetch<T, S::CPR>(rv, v, a.v_n, t * KT, a.Nk, a.d);
        }
        f32x16 s[BLOCKS] = {};
#pragma unroll
        for (int j = 0; j < BLOCKS; ++j)
#pragma unroll
            for (int u = 0; u < K::CHUNKS; ++u) mma(s[j], K::row_chunk(lds_k, KEY_WAVES ? wave * 32 : 32 * j, u), q[u], T());
        if (!full) {
#pragma unroll
            for (int j = 0; j < BLOCKS; ++j) {
                const int key0 = KEY_WAVES ? wave * 32 : 32 * j;
                const uint32_t mine = static_cast<uint32_t>(bits[WORDS == 1 ? 0 : key0 >> 6] >> (key0 & 63)) >> (4 * (lane >> 5));
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (!(mine >> (8 * (i / 4) + i % 4) & 1)) s[j][i] = -INFINITY;
            }
        }
        float top = s[0][0];
#pragma unroll
        for (int j = 0; j < BLOCKS; ++j)
#pragma unroll
            for (int i = 0; i < 16; ++i) top = fmaxf(top, s[j][i]);
        top = fmaxf(top, other_half(top)) * c;
        // The sums are brought to a new maximum only where it rose by more than 2^8: weights up to 2^8 keep their relative precision in every type
        if (__ballot(top > m + 8.0f)) {
            const float up = fmaxf(m, top), f = up == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - up);
            m = up;
            l *= f;
#pragma unroll
            for (int db = 0; db < DB; ++db)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[db][i] *= f;
        }
        const float shift = m == -INFINITY ? 0.0f : m;
#pragma unroll
        for (int j = 0; j < BLOCKS; ++j) {
            float part = 0.0f;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                s[j][i] = __builtin_amdgcn_exp2f(fmaf(s[j][i], c, -shift));
                part += s[j][i];
            }
            l += part;
            u32x4 p[sizeof(T) == 4 ? 4 : 2];
            as_operand<T>(p, s[j]);
            V::mul_t(o, lds_v, KEY_WAVES ? wave * 32 : 32 * j, p);
        }
        __syncthreads();
    }
    l += other_half(l);
    if (!row_there) {          // (behind q_lens: it has looked at keys with the zeros it was given)
        m = -INFINITY;
        l = 0.0f;
#pragma unroll
        for (int db = 0; db < DB; ++db) o[db] = f32x16{};
    }
    if constexpr (KEY_WAVES) {          // the four waves' sums, at their common maximum
        float* sums = reinterpret_cast<float*>(lds);                                   // [wave][row][DP + 4]
        float2* ml = reinterpret_cast<float2*>(lds + 4 * 32 * (DP + 4) * 4);           // [wave][row]
        if (lane < 32) ml[wave * 32 + lane] = make_float2(m, l);
        __syncthreads();
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < 4; ++w) top = fmaxf(top, ml[w * 32 + (lane & 31)].x);
        const float f = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - top);
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int i = 0; i < 16; ++i) sums[(wave * 32 + (lane & 31)) * (DP + 4) + K::channel(db, i)] = o[db][i] * f;
        __syncthreads();
        const int r = threadIdx.x >> 3;          // eight threads to a row
        const int out_row = tile * 32 + r;
        float2 all = make_float2(-INFINITY, 0.0f);
        for (int w = 0; w < 4; ++w) all.x = fmaxf(all.x, ml[w * 32 + r].x);
        for (int w = 0; w < 4; ++w)
            if (ml[w * 32 + r].x != -INFINITY) all.y += ml[w * 32 + r].y * __builtin_amdgcn_exp2f(ml[w * 32 + r].x - all.x);
        if (out_row < a.rows) {
            const int on = out_row / a.G, og = out_row - on * a.G;
            const float inv = a.splits > 1 ? 1.0f : all.y > 0.0f ? 1.0f / all.y : all.y;
            float* part = a.splits > 1 ? a.part + (static_cast<int64_t>(item) * 32 + r) * a.d : nullptr;
            T* out = static_cast<T*>(a.o) + ((static_cast<int64_t>(b) * a.Nq + on) * a.H + hk * a.G + og) * a.d;
            for (int ch = threadIdx.x & 7; ch < a.d; ch += 8) {
                float x = 0.0f;
#pragma unroll
                for (int w = 0; w < 4; ++w) x += sums[(w * 32 + r) * (DP + 4) + ch];
                if (part) part[ch] = x;
                else out[ch] = static_cast<T>(x * inv);
            }
            if ((threadIdx.x & 7) == 0) {
                if (a.splits > 1) reinterpret_cast<float2*>(a.part_ml)[static_cast<int64_t>(item) * 32 + r] = all;
                else if (a.lse) a.lse[(static_cast<int64_t>(b) * a.H + hk * a.G + og) * a.Nq + on] = all.y == 0.0f ? -INFINITY : (all.x + log2f(all.y)) * LN2;
            }
        }
    } else {
        if (row >= a.rows) return;
        if (a.splits > 1) {
            float* part = a.part + (static_cast<int64_t>(item) * S::ROWS + wave * 32 + (lane & 31)) * a.d;
            if (lane < 32) reinterpret_cast<float2*>(a.part_ml)[static_cast<int64_t>(item) * S::ROWS + wave * 32 + lane] = make_float2(m, l);
#pragma unroll
            for (int db = 0; db < DB; ++db)
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (K::channel(db, i) < a.d) part[K::channel(db, i)] = o[db][i];
            return;
        }
        const float inv = l > 0.0f ? 1.0f / l : l;
        T* out = static_cast<T*>(a.o) + ((static_cast<int64_t>(b) * a.Nq + n) * a.H + hk * a.G + g) * a.d;
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if (K::channel(db, i) < a.d) out[K::channel(db, i)] = static_cast<T>(o[db][i] * inv);
        if (a.lse && lane < 32) a.lse[(static_cast<int64_t>(b) * a.H + hk * a.G + g) * a.Nq + n] = l == 0.0f ? -INFINITY : (m + log2f(l)) * LN2;
    }
}

// Joins the parts of the keys: one wave to a query row
template <class T>
__global__ __launch_bounds__(256) void xattn_join_kernel(const Args a, int tile_rows) {
    const int64_t w = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    if (w >= static_cast<int64_t>(a.B) * a.Hkv * a.rows) return;
    const int row = w % a.rows, bh = w / a.rows, hk = bh % a.Hkv, b = bh / a.Hkv, tile = row / tile_rows, n = row / a.G, g = row - n * a.G;
    const int64_t first = (static_cast<int64_t>(bh) * a.tiles + tile) * a.splits;
    const float2* ml = reinterpret_cast<const float2*>(a.part_ml);
    float top = -INFINITY;
    for (int s = lane; s < a.splits; s += 64) top = fmaxf(top, ml[(first + s) * tile_rows + row % tile_rows].x);
    top = wave_max(top);
    float l = 0.0f, o0 = 0.0f, o1 = 0.0f;
    for (int s = 0; s < a.splits; ++s) {
        const int64_t at = (first + s) * tile_rows + row % tile_rows;
        const float2 x = ml[at];
        if (x.x == -INFINITY) continue;
        const float f = __builtin_amdgcn_exp2f(x.x - top);
        l = fmaf(x.y, f, l);
        if (lane < a.d) o0 = fmaf(a.part[at * a.d + lane], f, o0);
        if (lane + 64 < a.d) o1 = fmaf(a.part[at * a.d + lane + 64], f, o1);
    }
    const float inv = l > 0.0f ? 1.0f / l : l;
    T* out = static_cast<T*>(a.o) + ((static_cast<int64_t>(b) * a.Nq + n) * a.H + hk * a.G + g) * a.d;
    if (lane < a.d) out[lane] = static_cast<T>(o0 * inv);
    if (lane + 64 < a.d) out[lane + 64] = static_cast<T>(o1 * inv);
    if (a.lse && lane == 0) a.lse[(static_cast<int64_t>(b) * a.H + hk * a.G + g) * a.Nq + n] = l == 0.0f ? -INFINITY : (top + log2f(l)) * LN2;
}

__device__ __forceinline__ bool admitted(const Args& a, int b, int n, int len) { return n < len && (!a.key_mask || a.key_mask[b * a.mask_b + n]); }

template <class T>
__device__ __forceinline__ float dot(const float* __restrict__ u, const T* __restrict__ x, int d) {
    float s = 0.0f;
    for (int c = 0; c < d; ++c) s = fmaf(u[c], static_cast<float>(x[c]), s);
    return s;
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


// ---- host
template <class F>
int with_type(int type, F&& f) {
    if (type == OGMM_F32) return f(float());
    if (type == OGMM_BF16) return f(__bf16());
    return f(_Float16());
}

template <class F>
int with_width(int d, F&& f) {
    using std::integral_constant;
    if (d <= 32) return f(integral_constant<int, 32>());
    if (d <= 64) return f(integral_constant<int, 64>());
    return f(integral_constant<int, 128>());
}

// Up to 32 query rows of a key head (single tokens): one row tile, and the four waves of its workgroup take different keys.
bool few_rows(const ogmm_xattn* a) { return static_cast<int64_t>(a->Nq) * (a->H / a->Hkv) <= 32; }

Args forward_args(const ogmm_xattn* x, float* ws) {
    Args a{};
    static_cast<ogmm_xattn&>(a) = *x;
    a.G = a.H / a.Hkv;
    a.rows = a.Nq * a.G;
    const int tile_rows = few_rows(x) ? 32 : 128;
    a.tiles = (a.rows + tile_rows - 1) / tile_rows;
    // Where the row tiles alone do not give every CU two workgroups, the keys are cut, into parts of at least 256
    const int64_t base = static_cast<int64_t>(a.B) * a.Hkv * a.tiles;
    a.splits = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(512 / std::max<int64_t>(base, 1), (a.Nk + 255) / 256)));
    a.items = static_cast<uint32_t>(base * a.splits);
    a.per_xcd = (a.items + 7) / 8;
    a.part_ml = ws;
    a.part = ws ? ws + static_cast<int64_t>(a.items) * tile_rows * 2 : nullptr;
    return a;
}

template <class T, int DP, bool KEY_WAVES>
int launch_fwd(const Args& a, hipStream_t stream) {
    using S = Fwd<T, DP, KEY_WAVES>;
    if constexpr (S::LDS > 65536) {
        static PerDeviceOnce once;
        if (once.first() && hipFuncSetAttribute(reinterpret_cast<const void*>(&xattn_fwd_kernel<T, DP, KEY_WAVES>), hipFuncAttributeMaxDynamicSharedMemorySize, S::LDS) != hipSuccess)
            return fail("ogmm_xattn_fwd: %d bytes of LDS are not available", S::LDS);
    }
    xattn_fwd_kernel<T, DP, KEY_WAVES><<<a.per_xcd * 8, 256, S::LDS, stream>>>(a);
    if (a.splits > 1) {
        const int64_t rows = static_cast<int64_t>(a.B) * a.Hkv * a.rows;
        xattn_join_kernel<T><<<static_cast<uint32_t>((rows + 3) / 4), 256, 0, stream>>>(a, S::ROWS);
    }
    return check_launch("ogmm_xattn_fwd");
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

}  // namespace

extern "C" int64_t ogmm_xattn_workspace_bytes(const ogmm_xattn* a, int backward) {
    if (!a || a->B < 1 || a->Nq < 1 || a->Nk < 0 || a->H < 1 || a->Hkv < 1 || backward) return 0;
    const Args f = forward_args(a, nullptr);
    return f.splits > 1 ? static_cast<int64_t>(f.items) * (few_rows(a) ? 32 : 128) * (a->d + 2) * static_cast<int64_t>(sizeof(float)) : 0;
}

extern "C" int ogmm_xattn_fwd(const ogmm_xattn* x, void* stream) {
    if (check("ogmm_xattn_fwd", x)) return 1;
    if (!x->B || !x->Nq) return 0;
    const Args a = forward_args(x, static_cast<float*>(x->workspace));
    OGMM_REQUIRE(a.splits == 1 || a.workspace, "ogmm_xattn_fwd: missing workspace");
    const bool few = few_rows(x);
    return with_type(x->type, [&](auto t) {
        return with_width(x->d, [&](auto w) {
            using T = decltype(t);
            constexpr int DP = decltype(w)::value;
            return few ? launch_fwd<T, DP, true>(a, as_stream(stream)) : launch_fwd<T, DP, false>(a, as_stream(stream));
        });
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
        if (rows) xattn_dq_kernel<decltype(t)><<<static_cast<uint32_t>((rows + 3) / 4), 256, 0, as_stream(stream)>>>([&] { Args g{}; static_cast<ogmm_xattn&>(g) = *a; return g; }());
        if (keys) xattn_dkv_kernel<decltype(t)><<<static_cast<uint32_t>((keys + 3) / 4), 256, 0, as_stream(stream)>>>([&] { Args g{}; static_cast<ogmm_xattn&>(g) = *a; return g; }());
        return check_launch("ogmm_xattn_bwd");
    });
}
