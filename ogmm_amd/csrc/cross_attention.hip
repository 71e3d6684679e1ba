// Cross attention to states of another length (include/ogmm_hip.h, L1), forward and backward.
//
// Forward, one pass over the keys with a running maximum and sum.  A workgroup has four waves or eight; a wave owns 32 query rows and forms S^T = K Q^T, so that a lane holds
// one query's scores (32x32 result: column = lane % 32, rows 8 (i / 4) + 4 (lane / 32) + i % 4): maximum, exponential and sum stay inside the lane but for one exchange with
// lane ^ 32, and P^T is the next product's operand as it lies, O^T = V^T P^T, with V's keys taken in the order in which the lanes hold them.  The G query heads of a key
// head are rows of one tile (row = n G + g): their keys are read once.
//
// What bounds it, measured: many rows in 16 bits: matrix and vector instructions together (heads of 128: the matrix pipes are busy a third of the time, the exponentials, sums and
// roundings take as long, and both wait at a tile's barrier): 64 x 1024 rows to 717 keys, 4 heads of 128, fp16 153 us = 630 TFLOP/s; 4 x 4096 to 4096, 16 heads over 4, bf16 724 us = 760;
// 4096 rows to 2048 ragged, masked keys, 16 heads of 64 over 4, bf16 173 us.  16 x 1024 rows to 717 ragged keys, 4 heads of 128, fp32 197 us = 93 TFLOP/s of the 154 that a
// large product reaches: the fp32 matrix pipes, busy 79 % of the cycles in which a CU works and 68 % of the time.
// One row: the keys' bytes: 16 requests of up to 12288 states, 4 key heads of 128, 56 us and 5 to join the parts, 302 MB at 5.4 TB/s; one token to 1024 states: 9 + 3 us, two launches' latency.
#include "ogmm_common.h"
#include <algorithm>
#include <atomic>
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
constexpr int WEIGHT_LOG2 = 12;          // the forward's weights are 2^12 at most

struct Args : ogmm_xattn {
    int G, rows;                   // query heads to a key head, query rows to a key head (Nq G)
    int tiles, splits;             // row tiles, parts of the keys
    uint32_t items, run;           // workgroups that have work, and neighbours among them that one XCD takes
    float* part;                   // splits > 1: [items of a split][rows of a tile][d] sums and, behind them, (maximum, sum) pairs
    float* part_ml;
};

__device__ __forceinline__ int clamp_len(const int32_t* lens, int b, int n) { return lens ? max(0, min(n, lens[b])) : n; }

// Workgroups go to the XCDs in turn.  Tiles of one (batch, key head) read the same keys, so an XCD gets runs of neighbours for its own L2; runs are dealt in turn, and so
// short (at least 64 of them where there are that many tiles) that batch entries of different lengths come out even.
__device__ __forceinline__ uint32_t item_of(const Args& a) {
    const uint32_t xcd = blockIdx.x % 8, at = blockIdx.x / 8;
    return (at / a.run * 8 + xcd) * a.run + at % a.run;
}

// The batch entry that comes b-th: where lengths differ the longest first, so that the last workgroups to start are the shortest (up to 64 entries: a lane ranks one)
__device__ __forceinline__ int batch_of(const Args& a, int b) {
    if (!a.kv_lens || a.B > 64 || a.B == 1) return b;
    const int lane = threadIdx.x & 63, mine = lane < a.B ? clamp_len(a.kv_lens, lane, a.Nk) : -1;
    int rank = 0;
    for (int i = 0; i < a.B; ++i) {
        const int other = __builtin_amdgcn_readlane(mine, i);
        rank += other > mine || (other == mine && i < lane);
    }
    return __ffsll(static_cast<unsigned long long>(__ballot(lane < a.B && rank == b))) - 1;
}

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

// A matrix of rows in LDS, with a gap between rows that keeps both of its readers off each other's banks.  Clocks of a CU for a wave's instruction, eight waves, at gaps of 0, 16, 32
// and 48 bytes: sixteen bytes of each of 32 rows 64.1, 4.7, 8.1, 4.6 (rows of 256 bytes) and 16.1, 5.6, 5.3, 5.4 (128 bytes); transposing reads 8.1, 8.2, 4.3, 4.2 and 4.3, 4.2, 4.3, 4.5.
template <class T, int DP>
struct Tile {
    static constexpr int ROW = DP * sizeof(T), PITCH = ROW + (ROW == 256 ? 48 : 16), CHUNKS = ROW / 32, DB = DP / 32;

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
                __builtin_memcpy(x, __builtin_assume_aligned(p + (8 * (i / 4) + i % 4) * PITCH, 4 * DB), 4 * DB);
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

// the value of lane and of lane ^ 32: their maximum, their sum
__device__ __forceinline__ float max_halves(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float add_halves(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Which keys are admitted, 64 at a time, one bit each: a lane's byte of the mask is on its way with the tile's keys, the bits are taken when both have come
__device__ __forceinline__ uint8_t mask_byte(const Args& a, int b, int n0, int len) {
    const int n = n0 + (threadIdx.x & 63);
    return a.key_mask && n < len ? a.key_mask[b * a.mask_b + n] : 0;
}
__device__ __forceinline__ uint64_t key_bits(const Args& a, uint8_t byte, int n0, int len) {
    if (a.key_mask) return __ballot(byte);
    return len - n0 >= 64 ? ~uint64_t(0) : len > n0 ? (uint64_t(1) << (len - n0)) - 1 : 0;
}

// Tiles of KT rows on their way to LDS: sixteen bytes to a thread, CPR chunks to a row.  The rows' addresses are a base that every lane shares and 32 bits of a lane's own.
template <class T, int DP, int KT, int THREADS>
struct Stage {
    static constexpr int CPR = DP * static_cast<int>(sizeof(T)) / 16, STEP = THREADS / CPR, PASSES = KT / STEP, PITCH = Tile<T, DP>::PITCH;
    static_assert(PASSES >= 1 && KT % STEP == 0, "shape");

    static __device__ __forceinline__ int chunk() { return threadIdx.x % CPR; }
    static __device__ __forceinline__ int row() { return threadIdx.x / CPR; }
    // a chunk behind the head's width reads the row's first, and becomes zeros on the way to LDS
    static __device__ __forceinline__ uint32_t chunk_offset(int d) { return chunk() * 16 < d * static_cast<int>(sizeof(T)) ? chunk() * 16 : 0; }

    // rows [n0, n0 + KT) of x, `step` bytes apart, of which n are there (rows behind them: the last one)
    static __device__ __forceinline__ void fetch(u32x4 (&r)[PASSES], const char* __restrict__ x, int64_t step, int n0, int n, uint32_t chunk_off) {
        const char* tile = x + n0 * step;
        if (n0 + KT <= n) {
            const uint32_t mine = row() * static_cast<uint32_t>(step) + chunk_off;
#pragma unroll
            for (int i = 0; i < PASSES; ++i) r[i] = *reinterpret_cast<const u32x4*>(tile + i * STEP * step + mine);
        } else {
#pragma unroll
            for (int i = 0; i < PASSES; ++i)
                r[i] = *reinterpret_cast<const u32x4*>(tile + (min(row() + i * STEP, n - 1 - n0) * static_cast<uint32_t>(step) + chunk_off));
        }
    }

    // A row whose bit is not set becomes zeros: what stands there may be anything, and 0 x NaN is no 0
    template <int WORDS>
    static __device__ __forceinline__ void put(char* lds, const u32x4 (&r)[PASSES], const uint64_t (&bits)[WORDS], bool full, int d) {
        char* p = lds + row() * PITCH + 16 * chunk();
        if (full && d == DP) {
#pragma unroll
            for (int i = 0; i < PASSES; ++i) *reinterpret_cast<u32x4*>(p + i * STEP * PITCH) = r[i];
        } else {
            const uint32_t there = chunk() * 16 < d * static_cast<int>(sizeof(T)) ? 1 : 0;
#pragma unroll
            for (int i = 0; i < PASSES; ++i) {
                const int n = row() + i * STEP;
                const uint64_t word = bits[WORDS == 1 ? 0 : n >> 6];
                const uint32_t keep = -(static_cast<uint32_t>(word >> (n & 63)) & there);
                *reinterpret_cast<u32x4*>(p + i * STEP * PITCH) = r[i] & keep;
            }
        }
    }
};

// w = 2^(c s - m); -> their sum
__device__ __forceinline__ float weights(f32x16& w, const f32x16& s, float c, float m) {
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        w[i] = __builtin_amdgcn_exp2f(fmaf(s[i], c, -m));
        sum = i ? sum + w[i] : w[i];
    }
    return sum;
}

// A result's start: zeros, or for a lane's sixteen rows 8 (i / 4) + 4 (lane / 32) + i % 4 the values in LDS
__device__ __forceinline__ f32x16 rows_of(const float* lds) {
    f32x16 x;
    lds += 4 * ((threadIdx.x & 63) >> 5);
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
        const float4 v = *reinterpret_cast<const float4*>(lds + 2 * i);
        x[i] = v.x; x[i + 1] = v.y; x[i + 2] = v.z; x[i + 3] = v.w;
    }
    return x;
}

// a lane's column of a result times f to a row of channels in memory: 16-bit four channels at once, fp32 DB.  rest: what the rounding to 16 bits left, in 16 bits again
template <class T, class M>
__device__ __forceinline__ void store_column(T* __restrict__ out, T* __restrict__ rest, const f32x16 (&c)[M::DB], float f, int d) {
    if constexpr (sizeof(T) == 2) {
        typedef T t4 __attribute__((ext_vector_type(4)));
#pragma unroll
        for (int db = 0; db < M::DB; ++db)
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                if (M::channel(db, i) >= d) continue;
                t4 v, w;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float x = c[db][i + e] * f;
                    v[e] = static_cast<T>(x);
                    w[e] = static_cast<T>(x - static_cast<float>(v[e]));
                }
                *reinterpret_cast<t4*>(out + M::channel(db, i)) = v;
                if (rest) *reinterpret_cast<t4*>(rest + M::channel(db, i)) = w;
            }
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            if (M::channel(0, i) >= d) continue;
#pragma unroll
            for (int db = 0; db < M::DB; ++db) out[M::channel(db, i)] = c[db][i] * f;
        }
    }
}
template <class M>
__device__ __forceinline__ void store_part(float* __restrict__ out, const f32x16 (&c)[M::DB], float f, int d) {
    if constexpr (M::ROW == 2 * 32 * M::DB) {
#pragma unroll
        for (int db = 0; db < M::DB; ++db)
#pragma unroll
            for (int i = 0; i < 16; i += 4)
                if (M::channel(db, i) < d) *reinterpret_cast<float4*>(out + M::channel(db, i)) = make_float4(c[db][i] * f, c[db][i + 1] * f, c[db][i + 2] * f, c[db][i + 3] * f);
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            if (M::channel(0, i) >= d) continue;
#pragma unroll
            for (int db = 0; db < M::DB; ++db) out[M::channel(db, i)] = c[db][i] * f;
        }
    }
}
template <class T>
__device__ __forceinline__ void store_one(const ogmm_xattn& a, int64_t at, float x) {
    const T v = static_cast<T>(x);
    static_cast<T*>(a.o)[at] = v;
    if (sizeof(T) == 2 && a.rest) static_cast<T*>(a.rest)[at] = static_cast<T>(x - static_cast<float>(v));
}

// WAVES of 32 query rows each; KEY_WAVES: one tile of 32 rows, and each of the four waves takes its own 32 keys of a tile
template <class T, int DP, int WAVES, bool KEY_WAVES>
struct Fwd {
    // keys of a tile: enough products between two barriers, and so little LDS that two workgroups share a CU
    static constexpr int KT = KEY_WAVES || sizeof(T) * DP * 64 < 1024 * WAVES ? 128 : sizeof(T) == 4 && DP > 64 ? 32 : 64;
    using M = Tile<T, DP>;
    static constexpr int ROWS = KEY_WAVES ? 32 : 32 * WAVES, THREADS = 64 * WAVES;
    static_assert(!KEY_WAVES || WAVES == 4, "shape");
    static constexpr int TILE_BYTES = 2 * KT * M::PITCH + KT * 4;
    // Query waves: two tiles, so that one is written while the other is read, and there is one barrier to a tile; key waves: one, and the four waves' sums side by side at the end
    static constexpr int BUFFERS = KEY_WAVES ? 1 : 2;
    static constexpr int LDS = KEY_WAVES ? std::max(TILE_BYTES, 4 * 32 * (DP + 4) * 4 + 4 * 32 * 8) : BUFFERS * TILE_BYTES;
};

template <class T, int DP, int WAVES, bool KEY_WAVES>
__global__ __launch_bounds__(64 * WAVES, (Fwd<T, DP, WAVES, KEY_WAVES>::LDS > 81920 ? 1 : sizeof(T) * DP <= 128 && !KEY_WAVES ? 4 : 2)) void xattn_fwd_kernel(const Args a) {
    using S = Fwd<T, DP, WAVES, KEY_WAVES>;
    using M = typename S::M;
    using St = Stage<T, DP, S::KT, S::THREADS>;
    constexpr int KT = S::KT, WORDS = KT > 64 ? KT / 64 : 1, BLOCKS = KEY_WAVES ? 1 : KT / 32, DB = M::DB;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    // a tile: keys, values, and 0 or -inf for a key that is not admitted
    uint32_t buffer = 0;          // where in LDS the tile that is read begins; the other: OTHER - buffer
    constexpr uint32_t OTHER = (S::BUFFERS - 1) * S::TILE_BYTES;
    const uint32_t item = item_of(a);
    if (item >= a.items) return;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int split = item % a.splits, tile = item / a.splits % a.tiles, of = item / a.splits / a.tiles, hk = of % a.Hkv, b = batch_of(a, of / a.Hkv), bh = b * a.Hkv + hk;
    const int64_t place = (static_cast<int64_t>(bh) * a.tiles + tile) * a.splits + split;          // of its part
    const int len = clamp_len(a.kv_lens, b, a.Nk), q_rows = clamp_len(a.q_lens, b, a.Nq) * a.G;
    const char *k = reinterpret_cast<const char*>(static_cast<const T*>(a.k) + b * a.k_b + hk * a.k_h);
    const char *v = reinterpret_cast<const char*>(static_cast<const T*>(a.v) + b * a.v_b + hk * a.v_h);
    const int64_t k_step = a.k_n * static_cast<int64_t>(sizeof(T)), v_step = a.v_n * static_cast<int64_t>(sizeof(T));
    const uint32_t chunk_off = St::chunk_offset(a.d);
    // this lane's query row
    const int row = tile * S::ROWS + (KEY_WAVES ? 0 : wave * 32) + (lane & 31), n = row / a.G, g = row - n * a.G;
    const bool row_there = row < q_rows;
    u32x4 q[M::CHUNKS];
    const float c = a.scale == 0.0f ? 1.0f : fabsf(a.scale) * LOG2E;          // (scale = 0: no score, whatever the queries are)
    {
        const char* p = reinterpret_cast<const char*>(static_cast<const T*>(a.q) + b * a.q_b + n * a.q_n + (hk * a.G + g) * a.q_h);
        const uint32_t flip = a.scale < 0.0f ? (sizeof(T) == 4 ? 0x80000000u : 0x80008000u) : 0u;          // a negative scale: the queries' signs
#pragma unroll
        for (int s = 0; s < M::CHUNKS; ++s) {
            q[s] = u32x4{0, 0, 0, 0};
            if (row_there && a.scale != 0.0f && 32 * s + 16 * (lane >> 5) < a.d * static_cast<int>(sizeof(T))) q[s] = *reinterpret_cast<const u32x4*>(p + 32 * s + 16 * (lane >> 5)) ^ flip;
        }
    }
    const int key_tiles = tile * S::ROWS < q_rows ? (len + KT - 1) / KT : 0, per = (key_tiles + a.splits - 1) / a.splits;
    const int end = min(key_tiles, (split + 1) * per);
    float m = -INFINITY, l = 0.0f;          // m: of scale S log2(e), the running maximum or up to WEIGHT_LOG2 below it
    f32x16 o[DB] = {};
    u32x4 rk[St::PASSES], rv[St::PASSES];
    uint8_t bytes[WORDS];
    auto fetch = [&](int t) {
        St::fetch(rk, k, k_step, t * KT, a.Nk, chunk_off);
        St::fetch(rv, v, v_step, t * KT, a.Nk, chunk_off);
#pragma unroll
        for (int w = 0; w < WORDS; ++w) bytes[w] = mask_byte(a, b, t * KT + 64 * w, min(len, (t + 1) * KT));
    };
    bool full = true, any = true;
    auto put = [&](char* to, int t) {
        uint64_t bits[WORDS], all = ~uint64_t(0), one = 0;
#pragma unroll
        for (int w = 0; w < WORDS; ++w) {
            bits[w] = key_bits(a, bytes[w], t * KT + 64 * w, min(len, (t + 1) * KT));
            all &= bits[w];
            one |= bits[w];
        }
        full = all == (KT < 64 ? (uint64_t(1) << (KT & 63)) - 1 : ~uint64_t(0));
        any = one != 0;
        St::put(to, rk, bits, full, a.d);
        St::put(to + KT * M::PITCH, rv, bits, full, a.d);
        if (!full && threadIdx.x < KT)
            reinterpret_cast<float*>(to + 2 * KT * M::PITCH)[threadIdx.x] = bits[WORDS == 1 ? 0 : threadIdx.x >> 6] >> (threadIdx.x & 63) & 1 ? 0.0f : -INFINITY;
    };
    int t = split * per;
    if (t < end) {
        fetch(t);
        put(lds, t);
        __syncthreads();
    }
    for (; t < end; ++t) {
        // (flags are the same in every lane, and known to be: matrix instructions take no notice of lanes that a branch left out)
        const bool all = __builtin_amdgcn_readfirstlane(full), some = __builtin_amdgcn_readfirstlane(any);
        const char *lds_k = lds + buffer, *lds_v = lds_k + KT * M::PITCH;
        const float* lds_bias = reinterpret_cast<const float*>(lds_k + 2 * KT * M::PITCH);
        if (t + 1 < end) fetch(t + 1);
        if (some)
#pragma unroll
        for (int j = 0; j < BLOCKS; ++j) {
            const int key0 = KEY_WAVES ? wave * 32 : 32 * j;
            f32x16 s = {};
            if (all) mma(s, M::row_chunk(lds_k, key0, 0), q[0], T());
            else mma(s = rows_of(lds_bias + key0), M::row_chunk(lds_k, key0, 0), q[0], T());
#pragma unroll
            for (int u = 1; u < M::CHUNKS; ++u) mma(s, M::row_chunk(lds_k, key0, u), q[u], T());
            // Weights against the maximum that the sums stand at.  Where it is too low, their sum tells: only then is the tile's maximum sought and the sums brought to it.
            // A weight up to 2^WEIGHT_LOG2 keeps its relative precision in every type; what falls below the type's range is 2^-WEIGHT_LOG2 of that again.
            f32x16 w;
            float part = weights(w, s, c, m);
            if (__ballot(!(part <= 1 << WEIGHT_LOG2))) {
                float top = s[0];
#pragma unroll
                for (int i = 1; i < 16; ++i) top = fmaxf(top, s[i]);
                const float up = fmaxf(m, max_halves(top) * c), f = up == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - up);
                m = up;
                l *= f;
#pragma unroll
                for (int db = 0; db < DB; ++db)
#pragma unroll
                    for (int i = 0; i < 16; ++i) o[db][i] *= f;
                part = weights(w, s, c, m == -INFINITY ? 0.0f : m);
            }
            l += part;          // (of the weights as they are in 32 bits: lse is what the backward's weights are made of)
            u32x4 p[sizeof(T) == 4 ? 4 : 2];
            as_operand<T>(p, w);
            M::mul_t(o, lds_v, key0, p);
        }
        if constexpr (S::BUFFERS == 1) __syncthreads();
        if (t + 1 < end) put(lds + (OTHER - buffer), t + 1);
        if (t + 1 < end || KEY_WAVES) __syncthreads();
        buffer = OTHER - buffer;
    }
    l = add_halves(l);
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
        const float f = __builtin_amdgcn_exp2f(m - (top == -INFINITY ? 0.0f : top));          // (a wave without a key: 0, also where no wave has one)
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int i = 0; i < 16; ++i) sums[(wave * 32 + (lane & 31)) * (DP + 4) + M::channel(db, i)] = o[db][i] * f;
        __syncthreads();
        const int r = threadIdx.x >> 3;          // eight threads to a row
        const int out_row = tile * 32 + r;
        float2 all = make_float2(-INFINITY, 0.0f);
        for (int w = 0; w < 4; ++w) all.x = fmaxf(all.x, ml[w * 32 + r].x);
        // (a wave whose scores are all NaN has a sum that is NaN, at a maximum of -inf)
        for (int w = 0; w < 4; ++w) all.y += ml[w * 32 + r].y * __builtin_amdgcn_exp2f(ml[w * 32 + r].x - (all.x == -INFINITY ? 0.0f : all.x));
        if (out_row < a.rows) {
            const int on = out_row / a.G, og = out_row - on * a.G;
            const float inv = a.splits > 1 ? 1.0f : all.y > 0.0f ? 1.0f / all.y : all.y;
            float* part = a.splits > 1 ? a.part + (place * 32 + r) * a.d : nullptr;
            const int64_t out = ((static_cast<int64_t>(b) * a.Nq + on) * a.H + hk * a.G + og) * a.d;
            for (int ch = threadIdx.x & 7; ch < a.d; ch += 8) {
                float x = 0.0f;
#pragma unroll
                for (int w = 0; w < 4; ++w) x += sums[(w * 32 + r) * (DP + 4) + ch];
                if (part) part[ch] = x;
                else store_one<T>(a, out + ch, x * inv);
            }
            if ((threadIdx.x & 7) == 0) {
                if (a.splits > 1) reinterpret_cast<float2*>(a.part_ml)[place * 32 + r] = all;
                else if (a.lse) a.lse[(static_cast<int64_t>(b) * a.H + hk * a.G + og) * a.Nq + on] = all.y == 0.0f ? -INFINITY : (all.x + log2f(all.y)) * LN2;
            }
        }
    } else {
        if (row >= a.rows) return;
        if (a.splits > 1) {
            if (lane < 32) reinterpret_cast<float2*>(a.part_ml)[place * S::ROWS + wave * 32 + lane] = make_float2(m, l);
            store_part<M>(a.part + (place * S::ROWS + wave * 32 + (lane & 31)) * a.d, o, 1.0f, a.d);
            return;
        }
        const int64_t out = ((static_cast<int64_t>(b) * a.Nq + n) * a.H + hk * a.G + g) * a.d;
        store_column<T, M>(static_cast<T*>(a.o) + out, a.rest ? static_cast<T*>(a.rest) + out : nullptr, o, l > 0.0f ? 1.0f / l : l, a.d);
        if (a.lse && lane < 32) a.lse[(static_cast<int64_t>(b) * a.H + hk * a.G + g) * a.Nq + n] = l == 0.0f ? -INFINITY : (m + log2f(l)) * LN2;
    }
}

// Joins the parts of the keys: one wave to a query row, the loads of four parts on their way at once (512 rows of 16 parts: 4.8 us, waiting for each part's maximum first 8.4)
template <class T>
__global__ __launch_bounds__(256) void xattn_join_kernel(const Args a, int tile_rows) {
    const int64_t w = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    if (w >= static_cast<int64_t>(a.B) * a.Hkv * a.rows) return;
    const int row = w % a.rows, bh = w / a.rows, hk = bh % a.Hkv, b = bh / a.Hkv, tile = row / tile_rows, n = row / a.G, g = row - n * a.G;
    const int64_t first = (static_cast<int64_t>(bh) * a.tiles + tile) * a.splits;
    const float2* ml = reinterpret_cast<const float2*>(a.part_ml);
    const int64_t at0 = first * tile_rows + row % tile_rows;          // part s: tile_rows rows further on for each
    float top = -INFINITY;
    for (int s = lane; s < a.splits; s += 64) top = fmaxf(top, ml[at0 + s * tile_rows].x);
    top = wave_max(top);
    if (top == -INFINITY) top = 0.0f;          // (no key at all: every part is zero)
    float l = 0.0f, o0 = 0.0f, o1 = 0.0f;
    const int c0 = min(lane, a.d - 1), c1 = min(lane + 64, a.d - 1);
#pragma unroll 4
    for (int s = 0; s < a.splits; ++s) {          // (every part is written, an empty one as zeros: the loads need not wait for each other)
        const int64_t at = at0 + s * tile_rows;
        const float2 x = ml[at];
        const float u0 = a.part[at * a.d + c0], u1 = a.part[at * a.d + c1], f = __builtin_amdgcn_exp2f(x.x - top);
        l = fmaf(x.y, f, l);
        o0 = fmaf(u0, f, o0);
        o1 = fmaf(u1, f, o1);
    }
    const float inv = l > 0.0f ? 1.0f / l : l;
    const int64_t out = ((static_cast<int64_t>(b) * a.Nq + n) * a.H + hk * a.G + g) * a.d;
    if (lane < a.d) store_one<T>(a, out + lane, o0 * inv);
    if (lane + 64 < a.d) store_one<T>(a, out + lane + 64, o1 * inv);
    if (a.lse && lane == 0) a.lse[(static_cast<int64_t>(b) * a.H + hk * a.G + g) * a.Nq + n] = l == 0.0f ? -INFINITY : (top + log2f(l)) * LN2;
}

// ---- backward.  Two kernels form the scores again from lse: one owns query rows and sums dQ over the keys (S^T, dP^T, dQ^T: three products), one owns keys and sums dK, dV over
// the query rows of its G heads (S, dP, dV^T, dK^T: four products); no sum crosses workgroups but where few tiles are cut into parts, which are added in their order.
// fp32: its matrix instructions take eight times as long for the same product, so dS is kept by the kernel that owns keys (up to 1 GB of it) and dQ is one product of it: 16 x 1024 rows
// to 717 keys, 4 heads of 128: dq 300 -> 111 us, dk dv 480 -> 523; 1024 keys, heads of 64: 238 -> 105, 341 -> 379; of 32: 126 -> 67, 163 -> 188.  In 16 bits writing and reading dS would
// take longer than forming it.
struct BwdArgs : Args {
    int row_tiles, row_splits, key_tiles, key_splits;          // dq: tiles of 128 rows, parts of the keys; dk, dv: tiles of 128 keys, parts of the rows
    int delta_blocks;                                          // blocks of 64 rows to a key head
    float *lse2, *delta;                                       // [B Hkv][rows]: lse log2(e) (+inf: the row has no weights), sum of dO O
    // fp16: [B Hkv][rows] |dO| of a row; [B Hkv][delta_blocks] the largest |dO| and |sum of dO O|; [B Hkv][key_tiles][4] the largest |v| of a wave's keys (2-norms)
    float *size, *top_v;
    float2* top;
    float *part_q, *part_k, *part_v;                           // parts in the outputs' own order
    float* ds;                                                 // [B Hkv][key_tiles 128][ds_step] dS as dk, dv's kernel formed it, or null: dq forms it again
    int64_t ds_step;                                           // (rows, up to whole tiles)
};

__device__ __forceinline__ int64_t row_offset(const Args& a, int r, int b, int hk, int64_t sb, int64_t sn, int64_t sh) {
    const int n = a.G == 1 ? r : r / a.G, g = r - n * a.G;
    return b * sb + n * sn + (hk * a.G + g) * sh;
}

template <class T> constexpr bool NARROW = std::is_same_v<T, _Float16>;          // few exponent bits
template <class T> constexpr float P_LOG2 = NARROW<T> ? 14.0f : 0.0f;
template <class T> constexpr float P_POWER = NARROW<T> ? 0x1p14f : 1.0f;

// four threads to a row, each with every fourth sixteen bytes of it (HBM-bound: 16 x 1024 x 4 fp32 rows of 128, 67 MB in 13.4 us = 5.0 TB/s)
template <class T>
__global__ __launch_bounds__(256) void xattn_delta_kernel(const BwdArgs a) {
    __shared__ float2 tops[4];
    constexpr int VEC = 16 / sizeof(T);
    typedef T tv __attribute__((ext_vector_type(VEC)));
    const int block = blockIdx.x % a.delta_blocks, bh = blockIdx.x / a.delta_blocks, hk = bh % a.Hkv, b = bh / a.Hkv;
    const int r = block * 64 + (threadIdx.x >> 2);
    float delta = 0.0f, size = 0.0f;
    if (r < a.rows) {
        const int n = r / a.G, g = r - n * a.G;
        const float lse = a.lse[(static_cast<int64_t>(b) * a.H + hk * a.G + g) * a.Nq + n];
        const bool there = n < clamp_len(a.q_lens, b, a.Nq) && lse != -INFINITY;
        if (there) {
            const int64_t at = ((static_cast<int64_t>(b) * a.Nq + n) * a.H + hk * a.G + g) * a.d;
            const T *o = static_cast<const T*>(a.o) + at, *rest = sizeof(T) == 2 && a.rest ? static_cast<const T*>(a.rest) + at : nullptr;
            const T* go = static_cast<const T*>(a.dout) + b * a.do_b + n * a.do_n + (hk * a.G + g) * a.do_h;
            for (int c = (threadIdx.x & 3) * VEC; c < a.d; c += 4 * VEC) {
                const tv x = *reinterpret_cast<const tv*>(o + c), y = *reinterpret_cast<const tv*>(go + c);
                tv z = {};
                if (rest) z = *reinterpret_cast<const tv*>(rest + c);
#pragma unroll
                for (int k = 0; k < VEC; ++k) {
                    delta = fmaf(static_cast<float>(x[k]) + static_cast<float>(z[k]), static_cast<float>(y[k]), delta);
                    if constexpr (NARROW<T>) size = fmaf(static_cast<float>(y[k]), static_cast<float>(y[k]), size);
                }
            }
        }
        delta += __shfl_xor(delta, 1, 64);
        delta += __shfl_xor(delta, 2, 64);
        if constexpr (NARROW<T>) {
            size += __shfl_xor(size, 1, 64);
            size += __shfl_xor(size, 2, 64);
            size = sqrtf(size);
        }
        if ((threadIdx.x & 3) == 0) {
            const int64_t at = static_cast<int64_t>(bh) * a.rows + r;
            a.lse2[at] = there ? lse * LOG2E : INFINITY;
            a.delta[at] = delta;
            if constexpr (NARROW<T>) a.size[at] = size;
        }
    }
    if constexpr (NARROW<T>) {
        size = wave_max(size);
        const float top = wave_max(fabsf(delta));
        if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = make_float2(size, top);
        __syncthreads();
        if (threadIdx.x == 0)
            a.top[blockIdx.x] = make_float2(fmaxf(fmaxf(tops[0].x, tops[1].x), fmaxf(tops[2].x, tops[3].x)), fmaxf(fmaxf(tops[0].y, tops[1].y), fmaxf(tops[2].y, tops[3].y)));
    }
}

// fp16 ends at 2^-14 and at 65504, so P and dS are operands times powers of two there, which the sums are rid of at the end.  P <= 1 stands at 2^14: half a step is 2^-39 at least, and there is room for
// scores so large that fp32 knows them to within 1.  |dS_ij| = P_ij |dO_i v_j - delta_i| is at most |dO_i| |v_j| + |delta_i| (2-norms): dQ takes that bound for each of its rows, with the longest v,
// dK for each of its keys, with the largest |dO| and |delta|, and brings it to [2^13, 2^14].  Half a step of a small dS is 2^-38 of its bound: with 4096 keys of
// like weights 2^-14 of the dS of a row that lies 2^10 below its head's largest, where fp16's own rounding is 2^-11.  Nothing overflows.  (A power that follows the values as they come would leave
// 2^-21 of each sum's own largest, for 2 to 10 % of the kernels' time.)
__device__ __forceinline__ float power_for(float bound) {
    if (!(bound > 0.0f && bound < INFINITY)) return 1.0f;          // (no gradient at all, or NaN and infinities: so are the sums)
    return __uint_as_float(static_cast<uint32_t>(min(254, 267 - static_cast<int>(__float_as_uint(bound) >> 23))) << 23);
}

template <class T, int DP>
struct Bwd {
    static constexpr int KT = sizeof(T) == 4 && DP > 64 ? 32 : 64;          // keys (dq) or rows (dk, dv) of a tile
    using M = Tile<T, DP>;
    static constexpr int TILE_BYTES = 2 * KT * M::PITCH + 2 * KT * 4, LDS = 2 * TILE_BYTES;
};

// 4 x 4096 rows to 2048 ragged, masked keys, 16 heads of 64 over 4, bf16: 212 us, the matrix pipes busy 44 % of the cycles in which a CU works, 39 % of the time, beside the
// exponentials; the scores' bytes are LDS reads of K and V
template <class T, int DP>
__global__ __launch_bounds__(256, (sizeof(T) * DP > 256 ? 1 : sizeof(T) * DP > 128 ? 2 : 3)) void xattn_dq_kernel(const BwdArgs a) {
    using S = Bwd<T, DP>;
    using M = typename S::M;
    using St = Stage<T, DP, S::KT, 256>;
    constexpr int KT = S::KT, BLOCKS = KT / 32;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    uint32_t buffer = 0;          // where in LDS the tile that is read begins; the other: OTHER - buffer
    constexpr uint32_t OTHER = S::TILE_BYTES;
    const uint32_t item = item_of(a);
    if (item >= a.items) return;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int split = item % a.row_splits, tile = item / a.row_splits % a.row_tiles, of = item / a.row_splits / a.row_tiles, hk = of % a.Hkv, b = batch_of(a, of / a.Hkv), bh = b * a.Hkv + hk;
    const int len = clamp_len(a.kv_lens, b, a.Nk), q_rows = clamp_len(a.q_lens, b, a.Nq) * a.G;
    const char *k = reinterpret_cast<const char*>(static_cast<const T*>(a.k) + b * a.k_b + hk * a.k_h);
    const char *v = reinterpret_cast<const char*>(static_cast<const T*>(a.v) + b * a.v_b + hk * a.v_h);
    const int64_t k_step = a.k_n * static_cast<int64_t>(sizeof(T)), v_step = a.v_n * static_cast<int64_t>(sizeof(T));
    const uint32_t chunk_off = St::chunk_offset(a.d);
    const int row = tile * 128 + wave * 32 + (lane & 31);
    const bool row_there = row < q_rows;
    // (a negative scale turns the queries' signs, so that -inf is below every score; scale = 0: no score)
    const float c = a.scale == 0.0f ? 1.0f : fabsf(a.scale) * LOG2E;
    float up = 1.0f;          // dS's power of two, the same in both halves of a column
    u32x4 q[M::CHUNKS], go[M::CHUNKS];
    float lse2 = INFINITY, delta = 0.0f;
    {
        const int64_t at = static_cast<int64_t>(bh) * a.rows + row;
        if (row_there) { lse2 = a.lse2[at]; delta = a.delta[at]; }
        if constexpr (NARROW<T>) {
            float top = 0.0f;
            for (int i = lane; i < a.key_tiles * 4; i += 64) top = fmaxf(top, a.top_v[static_cast<int64_t>(bh) * a.key_tiles * 4 + i]);
            top = wave_max(top);
            if (row_there) up = power_for(fmaf(a.size[at], top, fabsf(delta)));
        }
        const char* pq = reinterpret_cast<const char*>(static_cast<const T*>(a.q) + row_offset(a, row, b, hk, a.q_b, a.q_n, a.q_h));
        const char* pg = reinterpret_cast<const char*>(static_cast<const T*>(a.dout) + row_offset(a, row, b, hk, a.do_b, a.do_n, a.do_h));
        const uint32_t flip = a.scale < 0.0f ? (sizeof(T) == 4 ? 0x80000000u : 0x80008000u) : 0u;
#pragma unroll
        for (int s = 0; s < M::CHUNKS; ++s) {
            const int at = 32 * s + 16 * (lane >> 5);
            q[s] = go[s] = u32x4{0, 0, 0, 0};
            if (row_there && at < a.d * static_cast<int>(sizeof(T))) {
                if (a.scale != 0.0f) q[s] = *reinterpret_cast<const u32x4*>(pq + at) ^ flip;
                go[s] = *reinterpret_cast<const u32x4*>(pg + at);
            }
        }
    }
    const int tiles = tile * 128 < q_rows ? (len + KT - 1) / KT : 0, per = (tiles + a.row_splits - 1) / a.row_splits, end = min(tiles, (split + 1) * per);
    f32x16 dq[M::DB] = {};
    u32x4 rk[St::PASSES], rv[St::PASSES];
    uint8_t byte;
    auto fetch = [&](int t) {
        St::fetch(rk, k, k_step, t * KT, a.Nk, chunk_off);
        St::fetch(rv, v, v_step, t * KT, a.Nk, chunk_off);
        byte = mask_byte(a, b, t * KT, min(len, (t + 1) * KT));
    };
    bool full = true, any = true;
    auto put = [&](char* to, int t) {
        const uint64_t bits[1] = {key_bits(a, byte, t * KT, min(len, (t + 1) * KT))};
        full = bits[0] == (KT < 64 ? (uint64_t(1) << (KT & 63)) - 1 : ~uint64_t(0));
        any = bits[0] != 0;
        St::put(to, rk, bits, full, a.d);
        St::put(to + KT * M::PITCH, rv, bits, full, a.d);
        if (!full && threadIdx.x < KT) reinterpret_cast<float*>(to + 2 * KT * M::PITCH)[threadIdx.x] = bits[0] >> threadIdx.x & 1 ? 0.0f : -INFINITY;
    };
    f32x16 start;          // dP - delta from the start
#pragma unroll
    for (int i = 0; i < 16; ++i) start[i] = -delta;
    int t = split * per;
    if (t < end) {
        fetch(t);
        put(lds, t);
        __syncthreads();
    }
    for (; t < end; ++t) {
        const bool all = __builtin_amdgcn_readfirstlane(full), some = __builtin_amdgcn_readfirstlane(any);          // (see the forward)
        const char *lds_k = lds + buffer, *lds_v = lds_k + KT * M::PITCH;
        const float* lds_bias = reinterpret_cast<const float*>(lds_k + 2 * KT * M::PITCH);
        if (t + 1 < end) fetch(t + 1);
        if (some)
#pragma unroll
        for (int j = 0; j < BLOCKS; ++j) {
            f32x16 s = {}, dp = start;
            if (all) mma(s, M::row_chunk(lds_k, 32 * j, 0), q[0], T());
            else mma(s = rows_of(lds_bias + 32 * j), M::row_chunk(lds_k, 32 * j, 0), q[0], T());          // (a key that is not admitted: weight 0, and with its zeros for v a finite dP)
#pragma unroll
            for (int u = 1; u < M::CHUNKS; ++u) mma(s, M::row_chunk(lds_k, 32 * j, u), q[u], T());
#pragma unroll
            for (int u = 0; u < M::CHUNKS; ++u) mma(dp, M::row_chunk(lds_v, 32 * j, u), go[u], T());
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] = __builtin_amdgcn_exp2f(fmaf(s[i], c, -lse2)) * dp[i] * up;
            u32x4 ds[sizeof(T) == 4 ? 4 : 2];
            as_operand<T>(ds, s);
            M::mul_t(dq, lds_k, 32 * j, ds);
        }
        if (t + 1 < end) {
            put(lds + (OTHER - buffer), t + 1);
            __syncthreads();
        }
        buffer = OTHER - buffer;
    }
    if (row >= a.rows) return;
    if (!row_there)          // (behind q_lens: a NaN of its neighbours' keys has come to its zeros)
#pragma unroll
        for (int db = 0; db < M::DB; ++db) dq[db] = f32x16{};
    const int n = row / a.G, g = row - n * a.G;
    const int64_t at = ((static_cast<int64_t>(b) * a.Nq + n) * a.H + hk * a.G + g) * a.d;
    const float f = a.scale / up;
    if (a.row_splits > 1) store_part<M>(a.part_q + split * (static_cast<int64_t>(a.B) * a.Nq * a.H * a.d) + at, dq, f, a.d);
    else store_column<T, M>(static_cast<T*>(a.dq) + at, nullptr, dq, f, a.d);
}

// The same case: 305 us, matrix pipes busy 48 % of the cycles in which a CU works, 37 % of the time (two waves to a SIMD hold K, V and both sums in registers).  fp32, 16 x 1024 rows to 717 ragged
// keys, heads of 128: 513 us, 72 % and 57 %.  64 x 1024 rows to 717, heads of 128: bf16 369 us, fp16 405, one wave to a SIMD, whose sums move between register files
template <class T, int DP>
__global__ __launch_bounds__(256, (sizeof(T) * DP > 128 ? 1 : 2)) void xattn_dkv_kernel(const BwdArgs a) {
    using S = Bwd<T, DP>;
    using M = typename S::M;
    using St = Stage<T, DP, S::KT, 256>;
    constexpr int QT = S::KT, BLOCKS = QT / 32;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    // a tile: rows of q, of dout, their -lse, their -delta
    uint32_t buffer = 0;
    constexpr uint32_t OTHER = S::TILE_BYTES;
    const uint32_t item = item_of(a);
    if (item >= a.items) return;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int split = item % a.key_splits, tile = item / a.key_splits % a.key_tiles, bh = item / a.key_splits / a.key_tiles, hk = bh % a.Hkv, b = bh / a.Hkv;
    const int len = clamp_len(a.kv_lens, b, a.Nk), q_rows = clamp_len(a.q_lens, b, a.Nq) * a.G;
    const int key = tile * 128 + wave * 32 + (lane & 31);
    const bool key_there = key < len && (!a.key_mask || a.key_mask[b * a.mask_b + key]);
    // (all four waves take part in the tiles of rows, or none: a tile of keys without one that is admitted)
    const bool any = (key_bits(a, mask_byte(a, b, tile * 128, len), tile * 128, len) | key_bits(a, mask_byte(a, b, tile * 128 + 64, len), tile * 128 + 64, len)) != 0;
    const float c = a.scale * LOG2E;
    float up = 1.0f;          // dS's power of two, the same in both halves of a column
    u32x4 k[M::CHUNKS], v[M::CHUNKS];
    {
        const char* pk = reinterpret_cast<const char*>(static_cast<const T*>(a.k) + b * a.k_b + key * a.k_n + hk * a.k_h);
        const char* pv = reinterpret_cast<const char*>(static_cast<const T*>(a.v) + b * a.v_b + key * a.v_n + hk * a.v_h);
#pragma unroll
        for (int s = 0; s < M::CHUNKS; ++s) {
            const int at = 32 * s + 16 * (lane >> 5);
            k[s] = v[s] = u32x4{0, 0, 0, 0};
            if (key_there && at < a.d * static_cast<int>(sizeof(T))) {
                k[s] = *reinterpret_cast<const u32x4*>(pk + at);
                v[s] = *reinterpret_cast<const u32x4*>(pv + at);
            }
        }
    }
    if constexpr (NARROW<T>) {
        float size = 0.0f, top = 0.0f, top_delta = 0.0f;
        typedef T t8 __attribute__((ext_vector_type(8)));
#pragma unroll
        for (int s = 0; s < M::CHUNKS; ++s) {
            const t8 x = __builtin_bit_cast(t8, v[s]);
#pragma unroll
            for (int i = 0; i < 8; ++i) size = fmaf(static_cast<float>(x[i]), static_cast<float>(x[i]), size);
        }
        size = sqrtf(add_halves(size));
        for (int i = lane; i < a.delta_blocks; i += 64) {
            const float2 t = a.top[static_cast<int64_t>(bh) * a.delta_blocks + i];
            top = fmaxf(top, t.x);
            top_delta = fmaxf(top_delta, t.y);
        }
        up = power_for(fmaf(wave_max(top), size, wave_max(top_delta))) / P_POWER<T>;          // (its dS comes with P's power)
        size = wave_max(size);
        if (split == 0 && lane == 0) a.top_v[(static_cast<int64_t>(bh) * a.key_tiles + tile) * 4 + wave] = size;
    }
    const int tiles = any ? (q_rows + QT - 1) / QT : 0, per = (tiles + a.key_splits - 1) / a.key_splits, end = min(tiles, (split + 1) * per);
    f32x16 dk[M::DB] = {}, dv[M::DB] = {};
    u32x4 rq[St::PASSES], rg[St::PASSES];
    float r_stat = 0.0f;          // threads 0 .. QT: a row's lse, QT .. 2 QT: its delta
    const char *q = reinterpret_cast<const char*>(static_cast<const T*>(a.q) + b * a.q_b + hk * a.G * a.q_h);
    const char *go = reinterpret_cast<const char*>(static_cast<const T*>(a.dout) + b * a.do_b + hk * a.G * a.do_h);
    const int64_t q_step = a.q_n * static_cast<int64_t>(sizeof(T)), go_step = a.do_n * static_cast<int64_t>(sizeof(T));
    const uint32_t q_head = static_cast<uint32_t>(a.q_h * sizeof(T)), go_head = static_cast<uint32_t>(a.do_h * sizeof(T)), chunk_off = St::chunk_offset(a.d);
    // a tile holds whole rows of all G heads: a lane's place in it is the same for every tile
    const bool whole = QT % a.G == 0;
    uint32_t at_q[St::PASSES], at_go[St::PASSES];
#pragma unroll
    for (int i = 0; i < St::PASSES; ++i) {
        const int r = St::row() + i * St::STEP, n = r / a.G, g = r - n * a.G;
        at_q[i] = n * static_cast<uint32_t>(q_step) + g * q_head + chunk_off;
        at_go[i] = n * static_cast<uint32_t>(go_step) + g * go_head + chunk_off;
    }
    auto fetch_tile = [&](int t) {
        const int r0 = t * QT;
        if (whole && r0 + QT <= a.rows) {
            const char *tq = q + r0 / a.G * q_step, *tg = go + r0 / a.G * go_step;
#pragma unroll
            for (int i = 0; i < St::PASSES; ++i) rq[i] = *reinterpret_cast<const u32x4*>(tq + at_q[i]);
#pragma unroll
            for (int i = 0; i < St::PASSES; ++i) rg[i] = *reinterpret_cast<const u32x4*>(tg + at_go[i]);
        } else {
#pragma unroll
            for (int i = 0; i < St::PASSES; ++i) {
                const int r = min(r0 + St::row() + i * St::STEP, a.rows - 1), n = r / a.G, g = r - n * a.G;
                rq[i] = *reinterpret_cast<const u32x4*>(q + n * q_step + (g * q_head + chunk_off));
                rg[i] = *reinterpret_cast<const u32x4*>(go + n * go_step + (g * go_head + chunk_off));
            }
        }
        const int r = r0 + threadIdx.x % QT;
        if (threadIdx.x < 2 * QT) r_stat = r < q_rows ? (threadIdx.x < QT ? a.lse2 : a.delta)[static_cast<int64_t>(bh) * a.rows + r] : threadIdx.x < QT ? INFINITY : 0.0f;
    };
    auto put = [&](char* to, int t) {
        const int left = q_rows - t * QT;
        const uint64_t bits[1] = {left >= 64 ? ~uint64_t(0) : (uint64_t(1) << left) - 1};          // rows behind q_lens become zeros
        St::put(to, rq, bits, left >= QT, a.d);
        St::put(to + QT * M::PITCH, rg, bits, left >= QT, a.d);
        // (P's power comes in here: where the value is fetched, the workgroup would wait for it: 64 x 1024 rows to 717 keys, 4 heads of 128, fp16: 366 us instead of 325)
        if (threadIdx.x < 2 * QT) reinterpret_cast<float*>(to + 2 * QT * M::PITCH)[threadIdx.x] = (threadIdx.x < QT ? P_LOG2<T> : 0.0f) - r_stat;
    };
    int t = split * per;
    if (t < end) {
        fetch_tile(t);
        put(lds, t);
        __syncthreads();
    }
    for (; t < end; ++t) {
        const char *lds_q = lds + buffer, *lds_g = lds_q + QT * M::PITCH;
        const float *lds_lse = reinterpret_cast<const float*>(lds_q + 2 * QT * M::PITCH), *lds_delta = lds_lse + QT;
        if (t + 1 < end) fetch_tile(t + 1);
#pragma unroll
        for (int j = 0; j < BLOCKS; ++j) {
            f32x16 s = {}, dp = rows_of(lds_delta + 32 * j);          // dP - delta from the start
            const f32x16 l = rows_of(lds_lse + 32 * j);
#pragma unroll
            for (int u = 0; u < M::CHUNKS; ++u) mma(s, M::row_chunk(lds_q, 32 * j, u), k[u], T());
#pragma unroll
            for (int u = 0; u < M::CHUNKS; ++u) mma(dp, M::row_chunk(lds_g, 32 * j, u), v[u], T());
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                s[i] = __builtin_amdgcn_exp2f(fmaf(s[i], c, l[i]));
                dp[i] = s[i] * dp[i] * up;
            }
            u32x4 y[sizeof(T) == 4 ? 4 : 2];
            as_operand<T>(y, s);
            M::mul_t(dv, lds_g, 32 * j, y);
            as_operand<T>(y, dp);
            M::mul_t(dk, lds_q, 32 * j, y);
            if constexpr (sizeof(T) == 4)
                if (a.ds) {          // (0 for a key that is not admitted; rows behind q_lens have 0 as it is)
                    float* to = a.ds + (static_cast<int64_t>(bh) * a.key_tiles * 128 + key) * a.ds_step + t * QT + 32 * j + 4 * (lane >> 5);
#pragma unroll
                    for (int i = 0; i < 16; i += 4)
                        *reinterpret_cast<float4*>(to + 2 * i) = key_there ? make_float4(dp[i], dp[i + 1], dp[i + 2], dp[i + 3]) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                }
        }
        if (t + 1 < end) {
            put(lds + (OTHER - buffer), t + 1);
            __syncthreads();
        }
        buffer = OTHER - buffer;
    }
    if (key >= a.Nk) return;
    // (a key that is not admitted has gathered the weights that its zeros gave it: nobody else's sum; its gradient is zero)
    const int64_t at = ((static_cast<int64_t>(b) * a.Nk + key) * a.Hkv + hk) * a.d, all = static_cast<int64_t>(a.B) * a.Nk * a.Hkv * a.d;
    if (!key_there)
#pragma unroll
        for (int db = 0; db < M::DB; ++db) dk[db] = dv[db] = f32x16{};
    const float fk = a.scale / (up * P_POWER<T>), fv = 1.0f / P_POWER<T>;
    if (a.key_splits > 1) {
        store_part<M>(a.part_k + split * all + at, dk, fk, a.d);
        store_part<M>(a.part_v + split * all + at, dv, fv, a.d);
    } else {
        store_column<T, M>(static_cast<T*>(a.dk) + at, nullptr, dk, fk, a.d);
        store_column<T, M>(static_cast<T*>(a.dv) + at, nullptr, dv, fv, a.d);
    }
}

// dQ^T = scale K^T dS^T with the dS that dk, dv's kernel left: a lane reads its row's values of 32 keys, which is the layout of a product's result
template <int DP>
__global__ __launch_bounds__(256, 2) void xattn_dq_of_ds_kernel(const BwdArgs a) {
    using M = Tile<float, DP>;
    constexpr int KT = 32;
    using St = Stage<float, DP, KT, 256>;
    __shared__ __attribute__((aligned(16))) char lds[2 * KT * M::PITCH];
    uint32_t buffer = 0;
    constexpr uint32_t OTHER = KT * M::PITCH;
    const uint32_t item = item_of(a);
    if (item >= a.items) return;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int split = item % a.row_splits, tile = item / a.row_splits % a.row_tiles, of = item / a.row_splits / a.row_tiles, hk = of % a.Hkv, b = batch_of(a, of / a.Hkv), bh = b * a.Hkv + hk;
    const int len = clamp_len(a.kv_lens, b, a.Nk), q_rows = clamp_len(a.q_lens, b, a.Nq) * a.G;
    const char* k = reinterpret_cast<const char*>(static_cast<const float*>(a.k) + b * a.k_b + hk * a.k_h);
    const int64_t k_step = a.k_n * static_cast<int64_t>(sizeof(float));
    const uint32_t chunk_off = St::chunk_offset(a.d);
    const int row = tile * 128 + wave * 32 + (lane & 31);
    const int tiles = tile * 128 < q_rows ? (len + KT - 1) / KT : 0, per = (tiles + a.row_splits - 1) / a.row_splits, end = min(tiles, (split + 1) * per);
    // (a lane behind the last row reads that row's: its column of the result is its own, and becomes zeros)
    const float* ds = a.ds + (static_cast<int64_t>(bh) * a.key_tiles * 128 + 4 * (lane >> 5)) * a.ds_step + max(0, min(row, q_rows - 1));
    f32x16 dq[M::DB] = {};
    u32x4 rk[St::PASSES];
    float next[16];
    uint8_t byte;
    auto fetch = [&](int t) {
        St::fetch(rk, k, k_step, t * KT, a.Nk, chunk_off);
        byte = mask_byte(a, b, t * KT, min(len, (t + 1) * KT));
        const float* p = ds + t * KT * a.ds_step;
#pragma unroll
        for (int i = 0; i < 16; ++i) next[i] = p[(8 * (i / 4) + i % 4) * a.ds_step];
    };
    bool any = true;
    auto put = [&](char* to, int t) {
        const uint64_t bits[1] = {key_bits(a, byte, t * KT, min(len, (t + 1) * KT))};
        any = bits[0] != 0;
        St::put(to, rk, bits, bits[0] == 0xffffffffull, a.d);
    };
    u32x4 y[4];
    auto take = [&] {
#pragma unroll
        for (int i = 0; i < 16; ++i) y[i / 4][i % 4] = __float_as_uint(next[i]);
    };
    int t = split * per;
    if (t < end) {
        fetch(t);
        put(lds, t);
        take();
        __syncthreads();
    }
    for (; t < end; ++t) {
        const bool some = __builtin_amdgcn_readfirstlane(any);          // (see the forward; without an admitted key dS may not have been written)
        if (t + 1 < end) fetch(t + 1);
        if (some) M::mul_t(dq, lds + buffer, 0, y);
        if (t + 1 < end) {
            put(lds + (OTHER - buffer), t + 1);
            take();
            __syncthreads();
        }
        buffer = OTHER - buffer;
    }
    if (row >= a.rows) return;
    if (row >= q_rows)
#pragma unroll
        for (int db = 0; db < M::DB; ++db) dq[db] = f32x16{};
    const int n = row / a.G, g = row - n * a.G;
    const int64_t at = ((static_cast<int64_t>(b) * a.Nq + n) * a.H + hk * a.G + g) * a.d;
    if (a.row_splits > 1) store_part<M>(a.part_q + split * (static_cast<int64_t>(a.B) * a.Nq * a.H * a.d) + at, dq, a.scale, a.d);
    else store_column<float, M>(static_cast<float*>(a.dq) + at, nullptr, dq, a.scale, a.d);
}

// out = the parts' sum, in their order (n: a multiple of 8 values)
template <class T>
__global__ __launch_bounds__(256) void xattn_add_kernel(const float* __restrict__ part, int parts, int64_t n, T* __restrict__ out) {
    typedef T t4 __attribute__((ext_vector_type(4)));
    const int64_t i = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) * 4;
    if (i >= n) return;
    float4 x = *reinterpret_cast<const float4*>(part + i);
    for (int s = 1; s < parts; ++s) {
        const float4 y = *reinterpret_cast<const float4*>(part + s * n + i);
        x.x += y.x; x.y += y.y; x.z += y.z; x.w += y.w;
    }
    *reinterpret_cast<t4*>(out + i) = t4{static_cast<T>(x.x), static_cast<T>(x.y), static_cast<T>(x.z), static_cast<T>(x.w)};
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

// Into how many parts the other sequence's n rows are cut, for `tiles` workgroups on a part that holds `slots` of them at once: parts of least_rows at least, as many as shorten
// the sum of the rounds by more than a part costs in writing and joining (taken as 1/16 of a round of it).
int parts_for(int64_t tiles, int64_t n, int64_t slots, int64_t least_rows = 256) {
    int best = 1;
    double least = 1e30;
    for (int64_t s = 1; s <= std::min<int64_t>((n + least_rows - 1) / least_rows, 512); ++s) {
        const double t = static_cast<double>((tiles * s + slots - 1) / slots) / s + (s > 1 ? s * tiles / (16.0 * slots) : 0.0);
        if (t < least * 0.999) { least = t; best = static_cast<int>(s); }
        if (tiles * s > 4 * slots) break;
    }
    return best;
}

// Rows of a workgroup's tile.  Up to 32 rows of a key head (single tokens): one tile, whose four waves take different keys.  Eight waves share a tile's keys, which halves what each
// does to bring them to LDS, where there are rows enough to fill the CUs with them and heads so narrow that two such workgroups share a CU (bf16, heads of 64: 196 us with four waves,
// 172 with eight; fp16, heads of 128: 155 and 162).
int tile_rows(const ogmm_xattn* a) {
    const int64_t rows = static_cast<int64_t>(a->Nq) * (a->H / a->Hkv);
    const bool narrow = a->d * (a->type == OGMM_F32 ? 2 : 1) <= 64;
    return rows <= 32 ? 32 : narrow && rows * a->Hkv * a->B >= 256 * 256 && rows >= 256 ? 256 : 128;
}

// -> the grid; per_head: the workgroups of one key head
uint32_t deal(Args& a, int64_t items, int64_t per_head) {
    a.items = static_cast<uint32_t>(items);
    a.run = static_cast<uint32_t>(std::max<int64_t>(1, std::min(per_head, items / 64)));
    const uint32_t runs = (a.items + a.run - 1) / a.run;
    return (runs + 7) / 8 * 8 * a.run;
}

Args forward_args(const ogmm_xattn* x, float* ws) {
    Args a{};
    static_cast<ogmm_xattn&>(a) = *x;
    a.G = a.H / a.Hkv;
    a.rows = a.Nq * a.G;
    const int in_tile = tile_rows(x);
    a.tiles = (a.rows + in_tile - 1) / in_tile;
    // Where the row tiles alone do not give every CU two workgroups, the keys are cut
    const int64_t base = static_cast<int64_t>(a.B) * a.Hkv * a.tiles;
    a.splits = parts_for(base, a.Nk, in_tile == 256 ? 256 : 512, in_tile == 32 ? 128 : 256);          // (128 keys: one tile of the key waves)
    a.items = static_cast<uint32_t>(base * a.splits);
    a.part_ml = ws;
    a.part = ws ? ws + static_cast<int64_t>(a.items) * in_tile * 2 : nullptr;
    return a;
}

// More than 64 KB of LDS is asked for once a device.  Noted when it has been granted: a thread that comes while another asks, asks too.
struct Granted { std::atomic<bool> on[64]; };
template <class K>
int allow_lds(K kernel, int bytes, Granted& granted) {
    int device = -1;
    if (bytes <= 65536 || (hipGetDevice(&device) == hipSuccess && device < 64 && granted.on[device])) return 0;
    if (hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, bytes) != hipSuccess)
        return fail("cross attention: %d bytes of LDS are not available", bytes);
    if (device >= 0 && device < 64) granted.on[device] = true;
    return 0;
}

template <class T, int DP, int WAVES, bool KEY_WAVES>
int launch_fwd(Args a, hipStream_t stream) {
    using S = Fwd<T, DP, WAVES, KEY_WAVES>;
    static Granted granted;
    if (allow_lds(&xattn_fwd_kernel<T, DP, WAVES, KEY_WAVES>, S::LDS, granted)) return 1;
    const uint32_t grid = deal(a, a.items, static_cast<int64_t>(a.tiles) * a.splits);
    xattn_fwd_kernel<T, DP, WAVES, KEY_WAVES><<<grid, S::THREADS, S::LDS, stream>>>(a);
    if (a.splits > 1) {
        const int64_t rows = static_cast<int64_t>(a.B) * a.Hkv * a.rows;
        xattn_join_kernel<T><<<static_cast<uint32_t>((rows + 3) / 4), 256, 0, stream>>>(a, S::ROWS);
    }
    return check_launch("ogmm_xattn_fwd");
}

BwdArgs backward_args(const ogmm_xattn* x, float* ws, int64_t* floats) {
    BwdArgs a{};
    static_cast<ogmm_xattn&>(a) = *x;
    a.G = a.H / a.Hkv;
    a.rows = a.Nq * a.G;
    const int64_t heads = static_cast<int64_t>(a.B) * a.Hkv;
    a.row_tiles = (a.rows + 127) / 128;
    a.key_tiles = (a.Nk + 127) / 128;
    a.delta_blocks = (a.rows + 63) / 64;
    const bool wide = a.d * (a.type == OGMM_F32 ? 2 : 1) > 64;          // (the kernel that owns keys has a CU to itself then)
    a.row_splits = parts_for(heads * a.row_tiles, a.Nk, 512);
    a.key_splits = parts_for(heads * a.key_tiles, a.rows, wide ? 256 : 512);
    int64_t n = 0;
    auto take = [&](int64_t count) {
        float* at = ws ? ws + n : nullptr;
        n += (count + 3) / 4 * 4;
        return at;
    };
    a.lse2 = take(heads * a.rows);
    a.delta = take(heads * a.rows);
    if (a.type == OGMM_F16) {
        a.size = take(heads * a.rows);
        a.top = reinterpret_cast<float2*>(take(heads * a.delta_blocks * 2));
        a.top_v = take(heads * a.key_tiles * 4);
    }
    if (a.row_splits > 1) a.part_q = take(a.row_splits * (heads * a.rows * a.d));
    if (a.key_splits > 1) {
        a.part_k = take(a.key_splits * (heads * a.Nk * a.d));
        a.part_v = take(a.key_splits * (heads * a.Nk * a.d));
    }
    a.ds_step = (a.rows + 63) / 64 * 64;
    const int64_t scores = heads * a.key_tiles * 128 * a.ds_step;
    if (a.type == OGMM_F32 && a.Nq && a.Nk && scores <= int64_t(1) << 28) {
        const int64_t at = n;
        n += scores;
        a.ds = ws ? ws + at : reinterpret_cast<float*>(16);          // (for the sizes alone: not null)
    }
    *floats = n;
    return a;
}

template <class T, int DP>
int launch_bwd(BwdArgs a, hipStream_t stream) {
    using S = Bwd<T, DP>;
    static Granted granted_q, granted_k;
    if (allow_lds(&xattn_dq_kernel<T, DP>, S::LDS, granted_q) || allow_lds(&xattn_dkv_kernel<T, DP>, S::LDS, granted_k)) return 1;
    const int64_t heads = static_cast<int64_t>(a.B) * a.Hkv;
    auto add = [&](const float* part, int parts, int64_t n, void* out) {
        xattn_add_kernel<T><<<static_cast<uint32_t>((n / 4 + 255) / 256), 256, 0, stream>>>(part, parts, n, static_cast<T*>(out));
    };
    if (a.Nq) xattn_delta_kernel<T><<<static_cast<uint32_t>(heads * a.delta_blocks), 256, 0, stream>>>(a);
    if (a.Nk) {
        const uint32_t grid = deal(a, heads * a.key_tiles * a.key_splits, static_cast<int64_t>(a.key_tiles) * a.key_splits);
        xattn_dkv_kernel<T, DP><<<grid, 256, S::LDS, stream>>>(a);
        if (a.key_splits > 1) {
            add(a.part_k, a.key_splits, heads * a.Nk * a.d, a.dk);
            add(a.part_v, a.key_splits, heads * a.Nk * a.d, a.dv);
        }
    }
    if (a.Nq) {
        const uint32_t grid = deal(a, heads * a.row_tiles * a.row_splits, static_cast<int64_t>(a.row_tiles) * a.row_splits);
        bool done = false;
        if constexpr (sizeof(T) == 4)
            if (a.ds) {
                xattn_dq_of_ds_kernel<DP><<<grid, 256, 0, stream>>>(a);
                done = true;
            }
        if (!done) xattn_dq_kernel<T, DP><<<grid, 256, S::LDS, stream>>>(a);
        if (a.row_splits > 1) add(a.part_q, a.row_splits, heads * a.rows * a.d, a.dq);
    }
    return check_launch("ogmm_xattn_bwd");
}

bool steps_fit(const ogmm_xattn* a, int64_t n, int64_t h) {
    const int64_t e = a->type == OGMM_F32 ? 4 : 2, most = int64_t(1) << 25;
    return n >= 0 && h >= 0 && n * e < most && h * e < most && 64 * n * e + a->H / a->Hkv * h * e < int64_t(1) << 32;
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
    // (the places of 64 rows and of all heads of a row stay within 32 bits)
    OGMM_REQUIRE(steps_fit(a, a->q_n, a->q_h) && steps_fit(a, a->k_n, 0) && steps_fit(a, a->v_n, 0), "%s: rows or heads are too far apart (32 MB and more)", who);
    OGMM_REQUIRE(aligned16(a->q) && aligned16(a->k) && aligned16(a->v) && aligned16(a->o) && aligned16(a->rest), "%s: addresses must be multiples of 16 bytes", who);
    OGMM_REQUIRE(isfinite(a->scale), "%s: scale must be finite", who);
    // (a workgroup takes 32 rows of a key head at least and up to 512 threads; a grid holds less than 2^32 threads, and rows are counted in 32 bits)
    const int64_t G = a->H / a->Hkv, heads = static_cast<int64_t>(a->B) * a->Hkv, most = int64_t(1) << 23, blocks = std::max((a->Nq * G + 63) / 64, (int64_t(a->Nk) + 127) / 128);
    OGMM_REQUIRE(blocks <= most && heads <= most && heads * blocks <= most, "%s: B = %d, Nq = %d, Nk = %d, H = %d, Hkv = %d are more than 2^23 blocks of 64 query rows or 128 keys of a key head",
                 who, a->B, a->Nq, a->Nk, a->H, a->Hkv);
    const bool rows = a->B && a->Nq, keys = a->B && a->Nk;
    OGMM_REQUIRE(!rows || (a->q && a->o), "%s: missing argument", who);
    OGMM_REQUIRE(!keys || (a->k && a->v), "%s: missing argument", who);
    return 0;
}

}  // namespace

extern "C" int64_t ogmm_xattn_workspace_bytes(const ogmm_xattn* a, int backward) {
    if (!a || a->B < 1 || a->Nq < 0 || a->Nk < 0 || a->H < 1 || a->Hkv < 1 || a->H < a->Hkv) return 0;
    if (backward) {
        int64_t floats;
        backward_args(a, nullptr, &floats);
        return floats * static_cast<int64_t>(sizeof(float));
    }
    const Args f = forward_args(a, nullptr);
    return f.splits > 1 ? static_cast<int64_t>(f.items) * tile_rows(a) * (a->d + 2) * static_cast<int64_t>(sizeof(float)) : 0;
}

extern "C" int ogmm_xattn_fwd(const ogmm_xattn* x, void* stream) {
    if (check("ogmm_xattn_fwd", x)) return 1;
    if (!x->B || !x->Nq) return 0;
    const Args a = forward_args(x, static_cast<float*>(x->workspace));
    OGMM_REQUIRE(a.splits == 1 || (a.workspace && aligned16(a.workspace)), "ogmm_xattn_fwd: missing workspace");
    const int rows = tile_rows(x);
    return with_type(x->type, [&](auto t) {
        return with_width(x->d, [&](auto w) {
            using T = decltype(t);
            constexpr int DP = decltype(w)::value;
            if (rows == 32) return launch_fwd<T, DP, 4, true>(a, as_stream(stream));
            if constexpr (sizeof(T) * DP <= 128)          // (tile_rows gives 256 rows to narrow heads alone)
                if (rows == 256) return launch_fwd<T, DP, 8, false>(a, as_stream(stream));
            return launch_fwd<T, DP, 4, false>(a, as_stream(stream));
        });
    });
}

extern "C" int ogmm_xattn_bwd(const ogmm_xattn* a, void* stream) {
    if (check("ogmm_xattn_bwd", a)) return 1;
    const int64_t e = a->type == OGMM_F32 ? 4 : 2;
    OGMM_REQUIRE(a->do_b * e % 16 == 0 && a->do_n * e % 16 == 0 && a->do_h * e % 16 == 0 && aligned16(a->dout) && steps_fit(a, a->do_n, a->do_h),
                 "ogmm_xattn_bwd: dout's address and strides must be multiples of 16 bytes, rows and heads less than 32 MB apart");
    OGMM_REQUIRE(aligned16(a->dq) && aligned16(a->dk) && aligned16(a->dv), "ogmm_xattn_bwd: addresses must be multiples of 16 bytes");
    const int64_t rows = static_cast<int64_t>(a->B) * a->H * a->Nq, keys = static_cast<int64_t>(a->B) * a->Hkv * a->Nk;
    OGMM_REQUIRE(!rows || (a->dout && a->lse && a->dq), "ogmm_xattn_bwd: missing argument");
    OGMM_REQUIRE(!keys || (a->dk && a->dv), "ogmm_xattn_bwd: missing argument");
    if (!rows && !keys) return 0;
    int64_t floats;
    const BwdArgs args = backward_args(a, static_cast<float*>(a->workspace), &floats);
    OGMM_REQUIRE(!floats || (a->workspace && aligned16(a->workspace)), "ogmm_xattn_bwd: missing workspace");
    return with_type(a->type, [&](auto t) {
        return with_width(a->d, [&](auto w) { return launch_bwd<decltype(t), decltype(w)::value>(args, as_stream(stream)); });
    });
}
