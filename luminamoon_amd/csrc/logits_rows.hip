// Operators over rows of logits: log probabilities of given tokens with entropy and the most likely
// tokens, and distillation from a teacher's top logits, forward and backward.
//
// A wave or a block holds a row in its registers (16-byte vectors, read once): its maximum m is taken,
// then, relative to it, s = sum 2^d and t = sum 2^d d, d = (z - m) log2(e) / temperature. So
//   log sum exp = m / temperature + ln s,   entropy = ln 2 (log2 s - t / s),
// whose two terms are of one sign: nothing cancels. Distillation goes on to the gradient from the
// same registers: the row is read once and its gradient written once. Rows longer than a block holds
// are cut into slices, whose (m, s, t) a second kernel joins: joining to a larger maximum, x higher in
// the units of d, turns s into s 2^-x and t into 2^-x (t - x s).
//
// The most likely tokens. About the count-th largest of the threads' largest logits (bisected by one
// wave; for few alternatives, of the waves' one to three largest) is a bound that at least `count`
// logits reach. The vectors whose largest logit reaches it, few more than count of them, are listed in
// LDS and read again, the logits that reach it listed too, and each one's rank is the number of those
// before it (larger, or equal and of a lower index). Bound and largest logits are compared in full, so
// an offset that a row's logits have in common changes nothing. Where more reach the bound than LDS
// holds (many equal logits, fewer finite ones than alternatives, or large ones crowded into few
// threads), the exact count-th one is found first, by bisection of its value and then of its index.
//
// What bounds it: reading the logits (6.5 TB/s for 8192 rows of 32000 bf16 without alternatives) and,
// with the gradient, writing as much (5.6 TB/s); a large copy runs at 6.15. With alternatives
// instruction issue joins it: 8192 x 50257 bf16 with 8 takes 12.7 vector instructions a logit, 80 to 89% of
// the SIMDs' cycles, 149 us (5.5 TB/s) at a stride of 50304 and 155 packed. Eight vectors a thread fit 64
// registers, so a compute unit holds 256 KiB of rows at once, several rows in different phases: 512 threads
// a row keep the memory busier than 1024 (8192 x 32000: 81 and 112 us). Short rows and few rows are bound
// by the way through the steps: one row of 32000 bf16 with 20 alternatives keeps its block for 7.4 us,
// 257 rows of 32000 f32 with 64 take 16.3. Rows with fewer finite logits than alternatives are read
// thirty times: 8192 x 32000 bf16 with 20 takes 93 us, and 2316 where 5 logits are finite.
#include "ops_common.h"

#include <cfloat>
#include <cmath>

namespace lvops {

constexpr int kThreads = 256;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kFar = -1.0e4f;  // stands for d = -inf where 2^d * d has to be 0

enum Way { kLogProbs, kDistill };

struct Job {
    lv_logits_args a;  // pointers already moved to the launch's first row
    float scale;       // log2(e) / temperature
    float inv_temp;
    int slices;        // blocks per row
    int slice_len;     // logits per block, a multiple of 8
    bool past;         // go past the caches
    float4 *partial;   // [rows][slices]: m, s, t of a slice
    float *part_value; // [rows][slices][count]: a slice's most likely logits, and their tokens
    int *part_token;
};

struct RowStats {
    float m, s, t;  // m -FLT_MAX and s 0 where every logit is -inf
};

static __device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// The same logits relative to a maximum m2 >= a.m.
static __device__ __forceinline__ void raise_max(RowStats &a, float m2, float scale) {
    const float x = fmaxf((a.m - m2) * scale, kFar), f = exp2_fast(x);
    a.t = f * fmaf(x, a.s, a.t);
    a.s *= f;
    a.m = m2;
}

// The block's statistics from its threads', the same in every thread. red: 3 x THREADS / 64 floats.
template <int THREADS>
static __device__ __forceinline__ RowStats block_stats(RowStats a, float scale, float *red) {
    constexpr int kWaves = THREADS / kWave;
    const float m = block_max<THREADS>(a.m, red);
    raise_max(a, m, scale);
    a.s = block_sum<THREADS>(a.s, red + kWaves);
    a.t = block_sum<THREADS>(a.t, red + 2 * kWaves);
    return a;
}

// Whether (v, i) comes before (w, k): the larger logit, the lower index among equals.
static __device__ __forceinline__ bool before(float v, int i, float w, int k) { return v > w || (v == w && i < k); }

// Finite and infinite floats in their order as unsigned integers, -0 as 0, and back.
static __device__ __forceinline__ uint32_t order_of(float v) {
    const uint32_t b = __float_as_uint(v + 0.0f);
    return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}

static __device__ __forceinline__ float of_order(uint32_t k) {
    return __uint_as_float(k ^ ((uint32_t)((int32_t)~k >> 31) | 0x80000000u));
}

// ----------------------------------------------------------------------- a row in a block's registers

// THREADS threads hold a row: the whole block, or one of the four waves of a block of 256.
template <int THREADS>
static constexpr int kBlock = THREADS == kWave ? 256 : THREADS;

template <int THREADS>
static __device__ __forceinline__ int row_thread() {
    return THREADS == kWave ? threadIdx.x % kWave : threadIdx.x;
}

// Orders the row's threads and what they wrote to LDS and memory. A wave's accesses are in order as
// they are: within it this holds the compiler only, and waits for nothing.
template <int THREADS>
static __device__ __forceinline__ void row_sync() {
    if (THREADS == kWave) {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    } else {
        __syncthreads();
    }
}

// LDS of a row: the places of vectors, and the logits, that reach the search's bound. Both lists hold
// at least the most alternatives that rows of these threads are searched for.
template <int THREADS, bool TOP>
struct RowLds {
    static constexpr int kWaves = THREADS / kWave;
    static constexpr int kVectors = !TOP ? 1 : kWaves == 1 ? 128 : 512;
    static constexpr int kLogits = !TOP ? 1 : kWaves == 1 ? 128 : 512;
    uint64_t key[kLogits];
    int first[kVectors];
    float red[5][kWaves];
    float bound[TOP ? THREADS : 1];  // the threads' largest logits, or the waves'
    int vectors, logits;
};
// Alternatives that a single wave's row is searched for: its bound is the less tight the more they are
// of its 64 threads (some 88 logits reach the bound for 48, 177 for 60, more than its list holds).
// 65536 rows of 1000 bf16 with 48: 124 us by single waves, 204 by blocks of 256.
constexpr int kMostOfAWave = 48;

// The sum over the row's threads of each of N values, the same in every thread. Consecutive calls
// with different `red` need no barrier between them.
template <int THREADS, int N>
static __device__ __forceinline__ void row_sums(float (&v)[N], float (*red)[THREADS / kWave]) {
    constexpr int kWaves = THREADS / kWave;
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = wave_sum(v[k]);
    if (kWaves == 1) return;
    if (threadIdx.x % kWave == 0) {
#pragma unroll
        for (int k = 0; k < N; ++k) red[k][threadIdx.x / kWave] = v[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < N; ++k) {
        v[k] = 0.0f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) v[k] += red[k][w];
    }
}

template <int THREADS, int N>
static __device__ __forceinline__ void row_maxes(float (&v)[N], float (*red)[THREADS / kWave]) {
    constexpr int kWaves = THREADS / kWave;
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = wave_max(v[k]);
    if (kWaves == 1) return;
    if (threadIdx.x % kWave == 0) {
#pragma unroll
        for (int k = 0; k < N; ++k) red[k][threadIdx.x / kWave] = v[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < N; ++k) {
        v[k] = red[k][0];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) v[k] = fmaxf(v[k], red[k][w]);
    }
}

// The largest logit of a vector as it is in memory.
static __device__ __forceinline__ float vector_max(const u32x4 &r, F32) {
    return max3(max3(__uint_as_float(r[0]), __uint_as_float(r[1]), __uint_as_float(r[2])), __uint_as_float(r[3]), -INFINITY);
}

static __device__ __forceinline__ float vector_max(const u32x4 &r, BF16) {
    float v[8];
    Type<BF16>::unpack(r, v);
    return max3(max3(max3(v[0], v[1], v[2]), v[3], v[4]), max3(v[5], v[6], v[7]), -INFINITY);
}

static __device__ __forceinline__ float vector_max(const u32x4 &r, F16) {
    auto larger = [](uint32_t a, uint32_t b) {
        uint32_t m;
        asm("v_pk_max_f16 %0, %1, %2" : "=v"(m) : "v"(a), "v"(b));
        return m;
    };
    const uint32_t two = larger(larger(r[0], r[1]), larger(r[2], r[3]));
    const _Float16 lo = __builtin_bit_cast(_Float16, (uint16_t)two), hi = __builtin_bit_cast(_Float16, (uint16_t)(two >> 16));
    return max3((float)lo, (float)hi, -INFINITY);
}

// A row (or slice) z[0, len) over THREADS threads, NV vectors each: thread t holds vectors t,
// t + THREADS, ... A 16-bit row that starts half way into a 4-byte word has its vectors one logit
// earlier (`skew`), on words: 8192 rows of 50257 bf16, every second of them off, take 155 us this way
// and 179 with loads off their words (with 8 alternatives). Logits before the row and past its end are -inf.
template <typename T, int THREADS, int NV>
struct RowRegisters {
    static constexpr int V = Type<T>::kVec;
    u32x4 raw[NV];
    int groups;  // vectors in the row
    int skew;

    __device__ __forceinline__ int first_of(int i) const { return (i * THREADS + row_thread<THREADS>()) * V - skew; }

    __device__ __forceinline__ void load(const store_t<T> *z, int len, bool past) {
        const int t = row_thread<THREADS>();
        skew = sizeof(store_t<T>) == 2 ? (int)((uintptr_t)z >> 1 & 1) : 0;
        int full = (len + skew) / V, rest = (len + skew) % V;  // vectors up to the last whole one
        if (skew && len < V) full = 0, rest = len + skew;
        groups = full + (rest ? 1 : 0);
        // the partial vector at the row's end is asked for first and put in its place last, by its wave
        float tail[V];
        const bool ends = rest && (THREADS == kWave || __builtin_amdgcn_readfirstlane(t / kWave) == full % THREADS / kWave);
        if (ends) {
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const int e = full * V - skew + j;
                tail[j] = t == full % THREADS && j < rest && e >= 0 ? Type<T>::load(z + e) : -INFINITY;
            }
        }
        auto take = [&](bool p) {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                if (i * THREADS >= groups) break;  // the same in every thread
                const int g = i * THREADS + t;
                if (g < full) raw[i] = load16<T>(z + max(g * V - skew, 0), p);
            }
        };
        if (past) take(true);
        else take(false);
        if (skew && t == 0) {  // the first vector was read from logit 0: one place up
            u32x4 &r = raw[0];
#pragma unroll
            for (int k = 3; k > 0; --k) r[k] = r[k] << 16 | r[k - 1] >> 16;
            r[0] = r[0] << 16 | (pack_all<T>(-INFINITY)[0] & 0xffffu);
        }
        u32x4 end = pack_all<T>(-INFINITY);
        if (ends) end = Type<T>::pack(tail);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if (i * THREADS >= groups) break;
            if ((i + 1) * THREADS > full && i * THREADS + t >= full) raw[i] = end;
        }
    }

    // Takes the vectors as changed: the compiler would keep unpacked logits from one pass to the next,
    // which costs more registers than unpacking them again.
    __device__ __forceinline__ void forget() {
#pragma unroll
        for (int i = 0; i < NV; ++i) asm volatile("" : "+v"(raw[i]));
    }

    // f(i, x): every vector as it is in memory
    template <typename F>
    __device__ __forceinline__ void each_raw(F f) const {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if (i * THREADS >= groups) break;
            f(i, raw[i]);
        }
    }

    // f(i, first, v): every vector, unpacked, and its first logit's index
    template <typename F>
    __device__ __forceinline__ void each(F f) const {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if (i * THREADS >= groups) break;
            float v[V];
            Type<T>::unpack(raw[i], v);
            f(i, first_of(i), v);
        }
    }
};

// The largest logit of each of a thread's vectors of a 16-bit type, as it is: two to a register.
template <typename T, int NV>
struct VectorTops {
    uint32_t two[(NV + 1) / 2];
    __device__ __forceinline__ void set(int i, float v) {
        const uint32_t b = __builtin_bit_cast(uint16_t, (store_t<T>)v);
        two[i / 2] = i % 2 ? (two[i / 2] & 0xffffu) | b << 16 : b;
    }
    __device__ __forceinline__ float get(int i, const u32x4 &) const {
        return (float)__builtin_bit_cast(store_t<T>, (uint16_t)(i % 2 ? two[i / 2] >> 16 : two[i / 2]));
    }
};

template <int NV>
struct VectorTops<BF16, NV> {
    uint32_t two[(NV + 1) / 2];
    __device__ __forceinline__ void set(int i, float v) {
        const uint32_t b = __float_as_uint(v);
        two[i / 2] = i % 2 ? (two[i / 2] & 0xffffu) | (b & 0xffff0000u) : b >> 16;
    }
    __device__ __forceinline__ float get(int i, const u32x4 &) const {
        return __uint_as_float(i % 2 ? two[i / 2] & 0xffff0000u : two[i / 2] << 16);
    }
};

// f32: one to a register. From thirteen vectors on that would spill (4096 x 25000 with 8 alternatives: 71
// us, and 67 this way), and the four logits are compared again.
template <int NV>
struct VectorTops<F32, NV> {
    static constexpr bool kKept = NV <= 8;
    float one[kKept ? NV : 1];
    __device__ __forceinline__ void set(int i, float v) {
        if (kKept) one[i] = v;
    }
    __device__ __forceinline__ float get(int i, const u32x4 &x) const { return kKept ? one[i] : vector_max(x, F32()); }
};

// A logit's place in the order of its type, 32 or 16 bits, at least 1, and back.
static __device__ __forceinline__ uint32_t key_of(float v, F32) { return order_of(v); }
static __device__ __forceinline__ uint32_t key_of(float v, BF16) { return order_of(v) >> 16; }
static __device__ __forceinline__ uint32_t key_of(float v, F16) {
    const uint32_t b = __builtin_bit_cast(uint16_t, (_Float16)(v + 0.0f));
    return b & 0x8000u ? b ^ 0xffffu : b | 0x8000u;
}

static __device__ __forceinline__ float of_key(uint32_t k, F32) { return of_order(k); }
static __device__ __forceinline__ float of_key(uint32_t k, BF16) { return of_order(k << 16); }
static __device__ __forceinline__ float of_key(uint32_t k, F16) {
    return (float)__builtin_bit_cast(_Float16, (uint16_t)(k & 0x8000u ? k ^ 0x8000u : k ^ 0xffffu));
}

// A place in a list in LDS for every lane with `in`, or -1; the list's length is *length.
static __device__ __forceinline__ int append(bool in, int *length) {
    const uint64_t all = __ballot(in);
    if (all == 0) return -1;
    int base = 0;
    const int lane = threadIdx.x % kWave, chief = __ffsll((unsigned long long)all) - 1;
    if (lane == chief) base = atomicAdd(length, __popcll(all));
    base = __builtin_amdgcn_readlane(base, chief);
    return in ? base + __builtin_amdgcn_mbcnt_hi((uint32_t)(all >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)all, 0)) : -1;
}

// The sum over the row's threads of small whole numbers (at most 2^24 in all: exact in f32).
template <int THREADS, bool TOP>
static __device__ __forceinline__ int row_count(int n, RowLds<THREADS, TOP> &lds) {
    row_sync<THREADS>();  // red's readers of the call before
    float total[1] = {(float)n};
    row_sums<THREADS>(total, lds.red);
    return (int)total[0];
}

// The exact count-th logit of z[0, len) by value and index, len >= count: at least count logits
// reach `bound`, none is above `most`. The row is read again for every step of the bisection of the
// value, and in order, up to the index, for the index.
template <typename T, int THREADS>
static __device__ __forceinline__ void find_bound(const store_t<T> *z, int len, int count, float most, float &bound, int &last,
                                                  RowLds<THREADS, true> &lds) {
    constexpr int V = Type<T>::kVec;
    const int tid = row_thread<THREADS>();
    uint32_t lo = order_of(bound), hi = order_of(most) + 1;  // count logits reach lo, fewer reach hi
    int above = 0;                                           // those that reach hi
    while (hi - lo > 1) {
        const uint32_t mid = lo + (hi - lo) / 2;
        const float limit = of_order(mid);
        int n = 0;
        for (int e = tid * V; e < len; e += THREADS * V) {
            float v[V];
            load_edge<T>(z, e, len, -INFINITY, v);
#pragma unroll
            for (int j = 0; j < V; ++j) n += v[j] >= limit && e + j < len ? 1 : 0;
        }
        n = row_count(n, lds);
        if (n >= count) lo = mid;
        else hi = mid, above = n;
    }
    bound = of_order(lo);
    int need = count - above;  // of those equal to the bound, from the lowest index on
    last = len - 1;
    for (int begin = 0; begin < len; begin += THREADS * V) {
        float v[V];
        const int e = begin + tid * V;
        load_edge<T>(z, e, len, INFINITY, v);
        int n = 0;
#pragma unroll
        for (int j = 0; j < V; ++j) n += v[j] == bound ? 1 : 0;
        n = row_count(n, lds);
        if (n < need) {
            need -= n;
            continue;
        }
        int none = begin - 1, all = begin + THREADS * V - 1;
        while (all - none > 1) {
            const int mid = none + (all - none) / 2;
            n = 0;
#pragma unroll
            for (int j = 0; j < V; ++j) n += v[j] == bound && e + j <= mid ? 1 : 0;
            (row_count(n, lds) >= need ? all : none) = mid;
        }
        last = all;
        break;
    }
}

// The `count` best of the row z[0, len), no logit of which is NaN: put(rank, logit, index) is called
// once for every rank below min(count, len). tops and best: the calling thread's vectors' largest
// logits and the largest of all of them, most: the row's. The lists' order depends on the waves'
// timing, the ranks do not.
template <typename T, int THREADS, int NV, typename Put>
static __device__ __forceinline__ void find_top(RowRegisters<T, THREADS, NV> &r, const VectorTops<T, NV> &tops, const store_t<T> *z,
                                                int len, int count, float best, float most, RowLds<THREADS, true> &lds, Put put) {
    using Lds = RowLds<THREADS, true>;
    constexpr int V = Type<T>::kVec, kWaves = THREADS / kWave;
    const int skew = r.skew, tid = row_thread<THREADS>(), lane = tid % kWave, wave = tid / kWave;
    float bound = -INFINITY;
    if (tid == 0) lds.vectors = lds.logits = 0;
    const int j = (count + kWaves - 1) / kWaves, n = j * kWaves;
    if (kWaves > 1 && j <= 3) {
        float rest = best;
        for (int k = 0; k < j; ++k) {
            const float first = wave_max(rest);
            if (lane == 0) lds.bound[wave * j + k] = first;
            const uint64_t at = __ballot(rest == first);
            if (lane == __ffsll((unsigned long long)at) - 1) rest = -INFINITY;
        }
        row_sync<THREADS>();
        // the count-th largest of the n, by every wave for itself
        float pick = INFINITY;
        if (lane < n) {
            const float v = lds.bound[lane];
            int ahead = 0;
#pragma unroll 8
            for (int k = 0; k < n; ++k) ahead += lds.bound[k] > v;
            if (ahead < count) pick = v;
        }
        bound = -wave_max(-pick);
    } else {
        // A short row gives too few threads' bests for a bound: there every logit stands for itself, for
        // twice the time (65536 rows of 1000 bf16 with 64 alternatives take 240 us, 424 this way; with
        // 128 they take 484 us this way, 1106 with the exact search that a loose bound leads to).
        constexpr bool kWide = sizeof(store_t<T>) == 4;  // a key fills a word, or half of one
        constexpr int kWords = Lds::kLogits * 2;         // of the keys where the list will be
        constexpr int kShort = kWaves == 4 && NV <= 8 ? kWords * (kWide ? 1 : 2) : 0;
        const bool each = kShort > 0 && len <= kShort && 2 * len < 3 * V * count;
        if (each) {
            for (int e = tid; e < kShort; e += THREADS) {
                const uint32_t key = e < len ? key_of(Type<T>::load(z + e), T()) : 0;
                if (kWide) reinterpret_cast<uint32_t *>(lds.key)[e] = key;
                else reinterpret_cast<uint16_t *>(lds.key)[e] = (uint16_t)key;
            }
        } else if (kWaves > 1) {
            lds.bound[tid] = best;
        }
        row_sync<THREADS>();
        if (wave == 0) {
            // the highest key that `count` reach; of f32 its upper half, and its lower half only where the
            // upper one lets half as many again through, as it does if the logits have an offset in common
            constexpr int kHalf = kWide ? 16 : 0;
            auto search = [&](uint32_t lo, uint32_t hi, auto reach) {  // count reach lo, fewer hi
                while (hi - lo > 1) {
                    const uint32_t mid = lo + (hi - lo) / 2;
                    (reach(mid) >= count ? lo : hi) = mid;
                }
                return lo;
            };
            const uint32_t least = key_of(-INFINITY, T());
            const uint32_t top = (key_of(most, T()) >> kHalf) + 1;
            uint32_t key;
            if (each) {
                const uint32_t *keys = reinterpret_cast<const uint32_t *>(lds.key);
                uint32_t word[kWords / kWave];
#pragma unroll
                for (int k = 0; k < kWords / kWave; ++k) word[k] = keys[k * kWave + lane] >> kHalf;
                auto reach = [&](uint32_t limit) {
                    int n = 0;
#pragma unroll
                    for (int k = 0; k < kWords / kWave; ++k) {
                        n += __popcll(__ballot((kWide ? word[k] : word[k] >> 16) >= limit));
                        if (!kWide) n += __popcll(__ballot((word[k] & 0xffffu) >= limit));
                    }
                    return n;
                };
                key = search(least >> kHalf, top, reach);
                if (kWide && reach(key) > count + count / 2 + 8) {
#pragma unroll
                    for (int k = 0; k < kWords / kWave; ++k) word[k] = keys[k * kWave + lane];
                    key = search(key << 16, (key + 1) << 16, reach);
                } else {
                    key <<= kHalf;
                }
            } else {
                uint32_t own[kWaves];
#pragma unroll
                for (int k = 0; k < kWaves; ++k) own[k] = key_of(kWaves > 1 ? lds.bound[k * kWave + lane] : best, T()) >> kHalf;
                auto reach = [&](uint32_t limit) {
                    int n = 0;
#pragma unroll
                    for (int k = 0; k < kWaves; ++k) n += __popcll(__ballot(own[k] >= limit));
                    return n;
                };
                key = search(least >> kHalf, top, reach);
                if (kWide && reach(key) > count + count / 2 + 8) {
#pragma unroll
                    for (int k = 0; k < kWaves; ++k) own[k] = key_of(kWaves > 1 ? lds.bound[k * kWave + lane] : best, T());
                    key = search(key << 16, (key + 1) << 16, reach);
                } else {
                    key <<= kHalf;
                }
            }
            bound = key <= least ? -INFINITY : of_key(key, T());
            if (kWaves > 1 && lane == 0) lds.bound[THREADS - 1] = bound;  // read by this wave already
        }
        row_sync<THREADS>();
        if (kWaves > 1) bound = lds.bound[THREADS - 1];
    }
    if (__ballot(best >= bound) != 0) {
        uint32_t left = 0;  // the thread's vectors that may hold a logit that reaches the bound
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (i * THREADS * V - skew < len) left |= (tops.get(i, r.raw[i]) >= bound ? 1u : 0u) << i;
        while (__ballot(left != 0) != 0) {
            const int first = ((__ffs(left) - 1) * THREADS + tid) * V - skew;
            const int at = append(left != 0 && first < len, &lds.vectors);
            if (at >= 0 && at < Lds::kVectors) lds.first[at] = first;
            left &= left - 1;
        }
    }
    row_sync<THREADS>();
    auto take = [&](bool in, float v, int index) {
        const int at = append(in, &lds.logits);
        if (at >= 0 && at < Lds::kLogits) lds.key[at] = (uint64_t)order_of(v) << 32 | (uint32_t)~index;
    };
    const int vectors = lds.vectors;
    if (vectors <= Lds::kVectors) {
        for (int e = tid; e < (vectors * V + kWave - 1) / kWave * kWave; e += THREADS) {  // whole waves
            const int at = e / V, index = at < vectors ? lds.first[at] + e % V : len;
            const bool there = index >= 0 && index < len;
            const float v = there ? Type<T>::load(z + index) : -INFINITY;
            take(there && v >= bound, v, index);
        }
        row_sync<THREADS>();
    }
    if (vectors > Lds::kVectors || lds.logits > Lds::kLogits) {
        int last;
        find_bound<T, THREADS>(z, len, count, most, bound, last, lds);  // its barriers come after the reads above
        if (tid == 0) lds.logits = 0;
        row_sync<THREADS>();
        for (int begin = 0; begin < len; begin += THREADS * V) {  // exactly `count` logits now
            float v[V];
            const int first = begin + tid * V;
            load_edge<T>(z, first, len, -INFINITY, v);
#pragma unroll
            for (int j = 0; j < V; ++j) take(first + j < len && !before(bound, last, v[j], first + j), v[j], first + j);
        }
        row_sync<THREADS>();
    }
    const int held = min(lds.logits, Lds::kLogits);
    for (int i = tid; i < held; i += THREADS) {
        const uint64_t key = lds.key[i];
        int rank = 0;
#pragma unroll 8
        for (int k = 0; k < held; ++k) rank += lds.key[k] > key;
        if (rank < count) put(rank, of_order((uint32_t)(key >> 32)), (int)~(uint32_t)key);
    }
}

// ------------------------------------------------------------------------------ a row's results

static __device__ __forceinline__ float stats_log_sum(const RowStats &a) { return a.s > 0.0f ? kLn2 * log2f(a.s) : a.s == 0.0f ? -INFINITY : a.s; }

static __device__ __forceinline__ void write_stats(const Job &job, int64_t row, const RowStats &a, float log_sum) {
    if (job.a.stats == nullptr) return;
    job.a.stats[2 * row] = a.s == 0.0f ? -INFINITY : a.m;
    job.a.stats[2 * row + 1] = log_sum;
}

// The row's token and its logit, asked for early: the row's own loads hide their way.
struct Named {
    bool there;
    float logit;
};

template <typename T>
static __device__ __forceinline__ Named load_named(const Job &job, int64_t row) {
    const int64_t token = job.a.tokens[row];
    Named n = {token >= 0 && token < (int64_t)job.a.vocab, 0.0f};
    if (n.there) n.logit = Type<T>::load(static_cast<const store_t<T> *>(job.a.logits) + row * job.a.stride + token);
    return n;
}

// By one thread: log_probs, entropy, stats of a row.
static __device__ __forceinline__ void write_log_probs(const Job &job, int64_t row, const RowStats &a, const Named &named) {
    const float log_sum = stats_log_sum(a);
    float lp = 0.0f;
    if (named.there) lp = a.s == 0.0f ? -INFINITY : (named.logit - a.m) * job.inv_temp - log_sum;
    job.a.out[row] = lp;
    job.a.entropy[row] = a.s == 0.0f ? 0.0f : log_sum - kLn2 * (a.t / a.s);
    write_stats(job, row, a, log_sum);
}

// The teacher's entries of a row in LDS, by the row's threads: the tokens (-1: names nothing), the
// student's logits of them, and the teacher's own, which become e = 2^((u - max u) scale), that is q
// times their sum.
struct Teacher {
    float *q, *student;
    int *token;
};

static __device__ __forceinline__ Teacher teacher_lds(float *base, int count) {
    return {base, base + count, (int *)(base + 2 * count)};
}

static __device__ __forceinline__ float load_any(const void *p, int64_t i, int dtype) {
    if (dtype == LV_DTYPE_F32) return static_cast<const float *>(p)[i];
    if (dtype == LV_DTYPE_BF16) return (float)static_cast<const __bf16 *>(p)[i];
    return (float)static_cast<const _Float16 *>(p)[i];
}

// The row's tokens into LDS, -1 for those that name nothing; whether any names something.
template <int THREADS>
static __device__ __forceinline__ bool load_teacher_tokens(const Job &job, int64_t row, const Teacher &q) {
    const int count = job.a.count;
    bool any = false;
    for (int k = row_thread<THREADS>(); k < count; k += THREADS) {
        const int64_t token = job.a.teacher_tokens[row * count + k];
        const bool there = token >= 0 && token < (int64_t)job.a.vocab;
        q.token[k] = there ? (int)token : -1;
        any |= there;
    }
    if (THREADS == kWave) {
        row_sync<THREADS>();
        return __ballot(any) != 0;
    }
    return __syncthreads_or(any);
}

// Both sides' logits of the tokens; the largest of the calling thread's own.
template <typename T, int THREADS>
static __device__ __forceinline__ float load_teacher_logits(const Job &job, int64_t row, const Teacher &q) {
    const store_t<T> *z = static_cast<const store_t<T> *>(job.a.logits) + row * job.a.stride;
    const int count = job.a.count;
    float m = -INFINITY;
    for (int k = row_thread<THREADS>(); k < count; k += THREADS) {
        const int token = q.token[k];
        q.student[k] = token >= 0 ? Type<T>::load(z + token) : 0.0f;
        const float u = token >= 0 ? load_any(job.a.teacher_logits, row * count + k, job.a.teacher_dtype) : -INFINITY;
        q.q[k] = u;
        m = fmaxf(m, u);
    }
    return m;
}

// e of the calling thread's entries and their sums, of e and of e (teacher's - student's distance from
// the largest logit) / kShares: with S and L these sums over the row and s the student's,
// T^2 KL(q || p) = T kShares L / S + T^2 ln 2 (log2 s - log2 S). Shares of logits, rather than sums of
// multiples in units of d, keep every step below f32's range where the loss is.
constexpr float kShares = 2.0f * LV_OPS_MAX_TEACHER;
static_assert((LV_OPS_MAX_TEACHER & (LV_OPS_MAX_TEACHER - 1)) == 0, "shares cost no rounding");

template <int THREADS>
static __device__ __forceinline__ void teacher_sums(const Job &job, const Teacher &q, float u_max, float m, float &sum, float &cross) {
    sum = cross = 0.0f;
    for (int k = row_thread<THREADS>(); k < job.a.count; k += THREADS) {
        const float u = q.q[k], below = u - u_max;
        const float e = u == -INFINITY ? 0.0f : exp2_fast(below * job.scale);  // no mass, nor in a row of -inf alone
        q.q[k] = e;
        sum += e;
        if (e != 0.0f) cross = fmaf(e * (1.0f / kShares), below - (q.student[k] - m), cross);
    }
}

static __device__ __forceinline__ float distill_loss(const Job &job, const RowStats &a, float sum, float cross) {
    if (sum == 0.0f) return 0.0f;
    if (a.s == 0.0f) return INFINITY;
    const float t = job.a.temperature;
    return t * (cross / sum * kShares + (log2f(a.s) - log2f(sum)) * (kLn2 * t));
}

// The weight of a row's gradient.
static __device__ __forceinline__ float grad_weight(const Job &job, int64_t row) {
    const float w = job.a.weight * job.a.temperature;
    return job.a.row_weight != nullptr ? w * job.a.row_weight[row] : w;
}

// The teacher's tokens in [begin, end) of a row's gradient, by the row's threads: w (p - q) over the
// w p that they wrote there before their last meeting. sum: of the entries' e. Every entry is compared
// with all of them for doubled tokens, quadratic in their number: the step of 4096 x 32000 bf16 takes 94
// us with 1, 99 with 32, 115 with 128, 219 with 512 and 630 with 1024.
template <typename T, int THREADS>
static __device__ __forceinline__ void grad_of_teacher(const Job &job, int64_t row, const RowStats &a, const Teacher &q, float sum,
                                                       float w, int begin, int end) {
    store_t<T> *grad = static_cast<store_t<T> *>(job.a.grad) + row * job.a.grad_stride;
    const int count = job.a.count;
    const float inv_s = 1.0f / a.s, inv_sum = 1.0f / sum;
    for (int k = row_thread<THREADS>(); k < count; k += THREADS) {
        const int token = q.token[k];
        if (token < begin || token >= end) continue;
        float e = 0.0f;
        bool first = true;
        for (int i = 0; i < count; ++i) {
            if (q.token[i] != token) continue;
            first = first && i >= k;
            e += q.q[i];
        }
        if (!first) continue;  // the first entry of a token writes for all of them
        const float p = exp2_fast((q.student[k] - a.m) * job.scale) * inv_s;
        Type<T>::store(grad + token, w * (p - e * inv_sum));
    }
}

// ----------------------------------------------------------------------------------- the kernels

// d = (z - m) scale as one product and sum, fma(z, scale, -base), base = m scale rounded: every d is
// then too large by the same `slip`, at most half a unit in the last place of base, which probabilities
// and entropy do not see and the log sum gives back. Above 2^24 (`far`) the slip could pass 1, and from
// 2^31 on f32's exponents: there d is a difference and a product.
struct Centre {
    float m, scale, base, slip;
    bool far;
};

static __device__ __forceinline__ Centre centre_of(float m, float scale) {
    Centre c = {m, scale, m * scale, 0.0f, false};
    c.far = __builtin_amdgcn_readfirstlane(!(fabsf(c.base) <= 16777216.0f));  // m is the same in the row's threads
    if (!c.far) c.slip = fmaf(m, scale, -c.base);
    return c;
}

// f(first, d): every vector's d and its first logit's index.
template <typename R, typename F>
static __device__ __forceinline__ void each_d(const R &r, const Centre &c, F f) {
    if (c.far) {
        r.each([&](int, int first, float(&v)[R::V]) {
#pragma unroll
            for (int j = 0; j < R::V; ++j) v[j] = (v[j] - c.m) * c.scale;
            f(first, v);
        });
    } else {
        r.each([&](int, int first, float(&v)[R::V]) {
#pragma unroll
            for (int j = 0; j < R::V; ++j) v[j] = fmaf(v[j], c.scale, -c.base);
            f(first, v);
        });
    }
}

// Waves per SIMD that a shape's registers leave: NV vectors of 4 registers and some 25 others; 1024
// threads come four waves to a SIMD.
template <int THREADS, int NV>
static constexpr int kWavesPerSimd = NV <= 8 ? 8 : NV <= 13 ? 6 : THREADS < 1024 ? 5 : 4;

// Row (or slice) blockIdx.x, or one of four for a wave each: its statistics from registers. A whole
// row goes on to its results, and with GRAD to its gradient.
template <typename T, int THREADS, int NV, Way WAY, bool TOP, bool GRAD>
__global__ void __launch_bounds__(kBlock<THREADS>, (kWavesPerSimd<THREADS, NV>)) rows_kernel(Job job) {
    constexpr int V = Type<T>::kVec, kRows = kBlock<THREADS> / THREADS;
    constexpr bool kEntropy = WAY == kLogProbs;
    extern __shared__ float dynamic[];
    __shared__ RowLds<THREADS, TOP> row_lds[kRows];
    const int own = kRows > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x / kWave) : 0;
    const int64_t unit = (int64_t)blockIdx.x * kRows + own;
    if (kRows > 1 && unit >= (int64_t)job.a.rows) return;  // one slice a row there
    RowLds<THREADS, TOP> &lds = row_lds[own];
    const int64_t row = kRows > 1 ? unit : blockIdx.x / job.slices;
    const int slice = kRows > 1 ? 0 : blockIdx.x % job.slices;
    const int tid = row_thread<THREADS>();
    const int vocab = (int)job.a.vocab;
    const int begin = slice * job.slice_len, len = min(job.slice_len, vocab - begin);
    const store_t<T> *z = static_cast<const store_t<T> *>(job.a.logits) + row * job.a.stride + begin;
    const Teacher q = teacher_lds(dynamic + own * 3 * job.a.count, job.a.count);
    const bool whole = kRows > 1 || job.slices == 1;

    bool mass = true;
    if (WAY == kDistill && whole) mass = load_teacher_tokens<THREADS>(job, row, q);
    Named named = {false, 0.0f};
    if (WAY == kLogProbs && whole) named = load_named<T>(job, row);
    RowRegisters<T, THREADS, NV> r;
    r.groups = r.skew = 0;
    if (!GRAD || mass) r.load(z, len, job.past);  // a row without a teacher has a gradient of 0 and no use for its logits
    float u_max = -INFINITY;
    const bool teach = WAY == kDistill && whole && mass;
    if (teach) u_max = load_teacher_logits<T, THREADS>(job, row, q);

    float best = -INFINITY;
    VectorTops<T, NV> tops;
    r.each_raw([&](int i, const u32x4 &x) {
        const float top = vector_max(x, T());
        if (TOP) tops.set(i, top);
        best = max3(best, top, best);
    });
    float maxes[WAY == kDistill ? 2 : 1];
    maxes[0] = fmaxf(best, -FLT_MAX);
    if constexpr (WAY == kDistill) maxes[1] = u_max;
    row_maxes<THREADS>(maxes, lds.red);
    RowStats a = {maxes[0], 0.0f, 0.0f};
    const Centre c = centre_of(a.m, job.scale);
    r.forget();
    each_d(r, c, [&](int, const float(&d)[V]) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const float e = exp2_fast(d[j]);
            a.s += e;
            if (kEntropy) a.t = fmaf(e, fmaxf(d[j], kFar), a.t);
        }
    });
    float sum = 0.0f, cross = 0.0f;  // the teacher's
    if constexpr (WAY == kDistill) {
        if (teach) teacher_sums<THREADS>(job, q, maxes[1], a.m, sum, cross);
        float sums[3] = {a.s, sum, cross};
        row_sums<THREADS>(sums, lds.red + 2);
        a.s = sums[0], sum = sums[1], cross = sums[2];
    } else {
        float sums[2] = {a.s, a.t};
        row_sums<THREADS>(sums, lds.red + 2);
        a.s = sums[0], a.t = sums[1];
    }
    const float grad_scale = 1.0f / a.s;  // of 2^d as computed
    if (c.slip != 0.0f) {
        a.t = exp2_fast(-c.slip) * fmaf(-c.slip, a.s, a.t);
        a.s *= exp2_fast(-c.slip);
    }
    const bool regular = a.s == a.s;  // no NaN, no +inf

    if (!whole) {
        const int64_t part = row * job.slices + slice;
        if (threadIdx.x == 0) job.partial[part] = make_float4(a.m, a.s, a.t, 0.0f);
        if constexpr (TOP) {
            if (regular) {
                float *value = job.part_value + part * job.a.count;
                int *token = job.part_token + part * job.a.count;
                find_top<T, THREADS, NV>(r, tops, z, len, job.a.count, best, a.m, lds, [&](int rank, float v, int at) {
                    value[rank] = v;
                    token[rank] = begin + at;
                });
            }
        }
        return;
    }
    if (WAY == kLogProbs) {
        if (tid == 0) write_log_probs(job, row, a, named);
        if constexpr (TOP) {
            float *value = job.a.top_log_probs + row * job.a.count;
            int64_t *token = job.a.top_tokens + row * job.a.count;
            if (regular) {
                const float log_sum = stats_log_sum(a), inv_temp = job.inv_temp, m = a.m;
                const bool some = a.s != 0.0f;
                find_top<T, THREADS, NV>(r, tops, z, len, job.a.count, best, a.m, lds, [&](int rank, float v, int at) {
                    value[rank] = some ? (v - m) * inv_temp - log_sum : -INFINITY;
                    token[rank] = at;
                });
            } else {
                for (int k = tid; k < job.a.count; k += THREADS) {
                    value[k] = a.s;
                    token[k] = k;
                }
            }
        }
    } else {
        if (tid == 0) {
            job.a.out[row] = distill_loss(job, a, sum, cross);
            write_stats(job, row, a, stats_log_sum(a));
        }
        if (GRAD) {
            store_t<T> *grad = static_cast<store_t<T> *>(job.a.grad) + row * job.a.grad_stride;
            if (sum != 0.0f && a.s != 0.0f) {  // NaN goes on
                const float w = grad_weight(job, row), ws = w * grad_scale;
                r.forget();
                each_d(r, c, [&](int first, const float(&d)[V]) {
                    float g[V];
#pragma unroll
                    for (int j = 0; j < V; ++j) g[j] = ws * exp2_fast(d[j]);
                    if (first >= 0 && first + V <= vocab) {
                        store16<T>(grad + first, Type<T>::pack(g), job.past);
                    } else if (first < vocab) {
#pragma unroll
                        for (int j = 0; j < V; ++j)
                            if (first + j >= 0 && first + j < vocab) Type<T>::store(grad + first + j, g[j]);
                    }
                });
                row_sync<THREADS>();
                grad_of_teacher<T, THREADS>(job, row, a, q, sum, w, 0, vocab);
            } else {
                float zero[V];
#pragma unroll
                for (int j = 0; j < V; ++j) zero[j] = 0.0f;
                for (int e = tid * V; e < vocab; e += THREADS * V) store_edge<T>(grad, e, vocab, zero);
            }
        }
    }
}

constexpr int kJoined = 4096;  // alternatives of a row's slices that join_kernel keeps in LDS

// One block a row: its slices' statistics put together, in their order, and the row's results. The
// slices' most likely tokens are sorted and the slices in order of their tokens, so the place of each
// among all is its place in its own slice plus, for every other slice, the number before it there.
template <typename T, Way WAY, bool TOP>
__global__ void __launch_bounds__(kThreads) join_kernel(Job job) {
    extern __shared__ float dynamic[];
    __shared__ float red[12];
    const int64_t row = blockIdx.x;
    const int slices = job.slices, count = job.a.count;
    const float4 *part = job.partial + row * slices;
    RowStats a = {-FLT_MAX, 0.0f, 0.0f};
    for (int i = threadIdx.x; i < slices; i += kThreads) {
        RowStats b = {part[i].x, part[i].y, part[i].z};
        const float m = fmaxf(a.m, b.m);
        raise_max(a, m, job.scale);
        raise_max(b, m, job.scale);
        a.s += b.s;
        a.t += b.t;
    }
    a = block_stats<kThreads>(a, job.scale, red);
    if (WAY == kDistill) {
        const Teacher q = teacher_lds(dynamic, count);
        float sum = 0.0f, cross = 0.0f;
        if (load_teacher_tokens<kThreads>(job, row, q)) {
            const float u_max = block_max<kThreads>(load_teacher_logits<T, kThreads>(job, row, q), red);
            teacher_sums<kThreads>(job, q, u_max, a.m, sum, cross);
            sum = block_sum<kThreads>(sum, red + 4);
            cross = block_sum<kThreads>(cross, red + 8);
        }
        if (threadIdx.x == 0) {
            job.a.out[row] = distill_loss(job, a, sum, cross);
            write_stats(job, row, a, stats_log_sum(a));
        }
        return;
    }
    if (threadIdx.x == 0) write_log_probs(job, row, a, load_named<T>(job, row));
    if (!TOP) return;
    float *value = job.a.top_log_probs + row * count;
    int64_t *token = job.a.top_tokens + row * count;
    if (!(a.s == a.s)) {
        for (int k = threadIdx.x; k < count; k += kThreads) {
            value[k] = a.s;
            token[k] = k;
        }
        return;
    }
    const float log_sum = stats_log_sum(a);
    const float *pv = job.part_value + row * slices * count;
    const int *pt = job.part_token + row * slices * count;
    const int last = min(count, (int)job.a.vocab - (slices - 1) * job.slice_len);  // entries of the last slice
    // each value is compared with log2(count) of every other slice: from LDS where they fit
    __shared__ float near[kJoined];
    const bool fits = slices * count <= kJoined;
    if (fits) {
        for (int i = threadIdx.x; i < slices * count; i += kThreads)
            if (i < (slices - 1) * count + last) near[i] = pv[i];
        __syncthreads();
    }
    auto value_at = [&](int i) { return fits ? near[i] : pv[i]; };
    for (int i = threadIdx.x; i < slices * count; i += kThreads) {
        const int own = i / count;
        int rank = i % count;
        if (own == slices - 1 && rank >= last) continue;
        const float v = value_at(i);
        for (int b = 0; b < slices && rank < count; ++b) {
            if (b == own) continue;
            int lo = 0, hi = b == slices - 1 ? last : count;  // how many of slice b come before v
            while (lo < hi) {
                const int mid = (lo + hi) / 2;
                const float w = value_at(b * count + mid);
                if (w > v || (w == v && b < own)) lo = mid + 1;
                else hi = mid;
            }
            rank += lo;
        }
        if (rank < count) {
            value[rank] = a.s != 0.0f ? (v - a.m) * job.inv_temp - log_sum : -INFINITY;
            token[rank] = pt[i];
        }
    }
}

// A row's statistics as the forward pass left them.
static __device__ __forceinline__ RowStats saved_stats(const Job &job, int64_t row) {
    const float m = job.a.stats[2 * row], log_sum = job.a.stats[2 * row + 1];
    RowStats a;
    a.m = m;
    a.s = m == -INFINITY ? 0.0f : exp2f(log_sum * kLog2e);
    a.t = 0.0f;
    return a;
}

// Block (row, slice): distillation's gradient from saved statistics.
template <typename T>
__global__ void __launch_bounds__(kThreads) distill_grad_kernel(Job job) {
    constexpr int V = Type<T>::kVec;
    extern __shared__ float dynamic[];
    __shared__ float red[12];
    const int64_t row = blockIdx.x / job.slices;
    const int begin = (int)(blockIdx.x % job.slices) * job.slice_len;
    const int end = min(begin + job.slice_len, (int)job.a.vocab);
    const store_t<T> *z = static_cast<const store_t<T> *>(job.a.logits) + row * job.a.stride;
    store_t<T> *grad = static_cast<store_t<T> *>(job.a.grad) + row * job.a.grad_stride;
    const Teacher q = teacher_lds(dynamic, job.a.count);
    const RowStats a = saved_stats(job, row);
    float sum = 0.0f, cross = 0.0f;
    if (load_teacher_tokens<kThreads>(job, row, q)) {
        const float u_max = block_max<kThreads>(load_teacher_logits<T, kThreads>(job, row, q), red);
        teacher_sums<kThreads>(job, q, u_max, a.m, sum, cross);
        sum = block_sum<kThreads>(sum, red + 4);
    }
    const bool some = sum != 0.0f && a.s != 0.0f;
    const float w = grad_weight(job, row), ws = w / a.s;
    for (int e = begin + threadIdx.x * V; e < end; e += kThreads * V) {
        float v[V];
        if (some) load_edge<T>(z, e, end, 0.0f, v, job.past);
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = some ? ws * exp2_fast((v[j] - a.m) * job.scale) : 0.0f;
        store_edge<T>(grad, e, end, v, job.past);
    }
    if (!some) return;
    __syncthreads();
    grad_of_teacher<T, kThreads>(job, row, a, q, sum, w, begin, end);
}

// The gradient of log probabilities and entropy: TPR threads to a row (or a slice of one), as many
// rows to a block as it has room for.
template <typename T, int TPR>
__global__ void __launch_bounds__(kThreads) log_probs_grad_kernel(Job job) {
    constexpr int V = Type<T>::kVec, kRows = kThreads / TPR;
    const int64_t row = kRows > 1 ? (int64_t)blockIdx.x * kRows + threadIdx.x / TPR : blockIdx.x / job.slices;
    if (kRows > 1 && row >= (int64_t)job.a.rows) return;
    const int begin = kRows > 1 ? 0 : (int)(blockIdx.x % job.slices) * job.slice_len;
    const int end = min(begin + job.slice_len, (int)job.a.vocab);
    const store_t<T> *z = static_cast<const store_t<T> *>(job.a.logits) + row * job.a.stride;
    store_t<T> *grad = static_cast<store_t<T> *>(job.a.grad) + row * job.a.grad_stride;
    const float m = job.a.stats[2 * row], log2_s = job.a.stats[2 * row + 1] * kLog2e;
    const int64_t named = job.a.tokens[row];
    const int token = named >= 0 && named < (int64_t)job.a.vocab ? (int)named : -1;
    const float g = token >= 0 && job.a.d_log_probs != nullptr ? job.a.d_log_probs[row] * job.inv_temp : 0.0f;
    const float h = job.a.d_entropy != nullptr ? job.a.d_entropy[row] * job.inv_temp : 0.0f;
    // -p (g + h (ln p + H)) = -p (c0 + c1 log2 p)
    const float c0 = h == 0.0f ? g : fmaf(h, job.a.entropy[row], g), c1 = h * kLn2;
    const bool none = m == -INFINITY;
    for (int e = begin + (int)(threadIdx.x % TPR) * V; e < end; e += TPR * V) {
        float v[V];
        load_edge<T>(z, e, end, 0.0f, v, job.past);
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const float d = (v[j] - m) * job.scale - log2_s;
            v[j] = none ? 0.0f : -exp2_fast(d) * fmaf(c1, fmaxf(d, kFar), c0);
            if (e + j == token && !none) v[j] += g;
        }
        store_edge<T>(grad, e, end, v, job.past);
    }
}

// ------------------------------------------------------------------------------------- host side

constexpr int64_t kLaunchBlocks = 1 << 22;  // blocks of one launch; more rows take several
constexpr uint64_t kLargestVocab = 1ull << 30, kMostRows = 1ull << 40;

static int check(const lv_logits_args *a, Way way, bool forward, bool backward) {
    const char *what = way == kLogProbs ? "token log probs" : "distill";
    if (a == nullptr) return fail(LV_STATUS_NULL_POINTER, "%s: null arguments", what);
    if (a->dtype < 0 || a->dtype > 2) return fail(LV_STATUS_INVALID_CONFIG, "%s: invalid dtype code %d", what, a->dtype);
    if (a->vocab < 1 || a->vocab > kLargestVocab || a->rows > kMostRows)
        return fail(LV_STATUS_INVALID_CONFIG, "%s: invalid size %llu x %llu", what, (unsigned long long)a->rows,
                    (unsigned long long)a->vocab);
    if (!(a->temperature > 0.0f) || !std::isfinite(a->temperature) || !std::isfinite(kLog2e / a->temperature))
        return fail(LV_STATUS_INVALID_CONFIG, "%s: invalid temperature: %g", what, a->temperature);
    if (way == kLogProbs && (a->count < 0 || a->count > LV_OPS_MAX_TOP || (uint64_t)a->count > a->vocab))
        return fail(LV_STATUS_INVALID_CONFIG, "%s: invalid number of alternatives: %d (0 to %d, at most the vocabulary)", what,
                    a->count, LV_OPS_MAX_TOP);
    if (way == kDistill && (a->count < 1 || a->count > LV_OPS_MAX_TEACHER))
        return fail(LV_STATUS_INVALID_CONFIG, "%s: invalid number of teacher logits: %d (1 to %d)", what, a->count,
                    LV_OPS_MAX_TEACHER);
    if (way == kDistill && (a->teacher_dtype < 0 || a->teacher_dtype > 2))
        return fail(LV_STATUS_INVALID_CONFIG, "%s: invalid teacher dtype code %d", what, a->teacher_dtype);
    if (a->rows == 0) return LV_STATUS_SUCCESS;
    bool null = a->logits == nullptr;
    if (way == kLogProbs) null |= a->tokens == nullptr || a->entropy == nullptr;
    if (way == kDistill) null |= a->teacher_tokens == nullptr || a->teacher_logits == nullptr;
    if (forward) null |= a->out == nullptr || (!backward && a->stats == nullptr);
    if (way == kLogProbs && forward && a->count > 0) null |= a->top_log_probs == nullptr || a->top_tokens == nullptr;
    if (backward) null |= a->grad == nullptr || (!forward && a->stats == nullptr);
    if (null) return fail(LV_STATUS_NULL_POINTER, "%s: null pointer", what);
    if (a->rows > 1 && (a->stride < 0 || (backward && a->grad_stride < (int64_t)a->vocab)))
        return fail(LV_STATUS_INVALID_CONFIG, "%s: invalid row stride", what);
    return LV_STATUS_SUCCESS;
}

struct Cut {
    int threads, vectors;  // of the block that holds a slice
    int slices, slice_len;
};

static int round_up(int64_t n, int m) { return (int)((n + m - 1) / m * m); }

// What holds a row: threads and 16-byte vectors of each, smallest first. In us, without and with 8
// alternatives and the distillation step, bf16:
//   32768 x 4000   64 x 8: 42, 55, 115     256 x 4: 61, 106, 138
//   16384 x 12000  256 x 8: 62, 82, 156    512 x 4: 80, 128, 168
//   8192 x 32000   512 x 8: 81, 100, 188   256 x 16: 80, 90, 197    1024 x 4: 112, 151, 231
//   8192 x 50257   512 x 13: 136, 155, 327 1024 x 8: 160, 206, 344  256 x 25: 130, 152, 340
static const int kShapes[][2] = {{64, 4}, {64, 8}, {256, 8}, {512, 8}, {512, 13}, {1024, 8}, {1024, 16}};
constexpr int kShapeCount = sizeof kShapes / sizeof kShapes[0];
constexpr int kSliced = 3;  // the shape of slices: 512 threads, 8 vectors

// 1 if a row may start half way into a word: its vectors then reach one logit further back.
static int row_skew(const lv_logits_args *a) {
    if (a->dtype == LV_DTYPE_F32) return 0;
    return ((uintptr_t)a->logits & 2) != 0 || (a->rows > 1 && a->stride % 2 != 0);
}

// The smallest block that holds a whole row. Longer rows are cut into slices of the largest block's,
// or of the smallest one's that still give every compute unit a block. Without a gradient, which
// would have to read the row again, rows are cut to slices of 512 threads where they would take 1024
// threads and 16 vectors (2048 x 50257 f32: 86 us whole, 62 cut), or 8 and there are many rows
// (4096 x 65536 bf16 with 8 alternatives: 116 us whole and 105 as slices of 512 threads, which cut_rows
// makes 256, 98 us; 512 rows: 20 whole and 22).
static Cut smallest_block(const lv_logits_args *a, int top, int skew, bool grad) {
    const int64_t vocab = (int64_t)a->vocab, rows = (int64_t)a->rows;
    const int v = a->dtype == LV_DTYPE_F32 ? 4 : 8;
    Cut c = {0, 0, 1, round_up(vocab, 8)};
    int k = 0;
    for (; k < kShapeCount; ++k) {
        c.threads = kShapes[k][0], c.vectors = kShapes[k][1];
        if (c.threads == kWave && top > kMostOfAWave) continue;
        if (!grad && c.threads > 512 && (c.vectors > 8 || rows >= 4 * compute_units())) break;
        if (vocab + skew <= (int64_t)c.threads * c.vectors * v) return c;
    }
    int64_t len = 0;
    for (k = grad ? kShapeCount - 1 : kSliced; kShapes[k][0] >= 256; --k) {
        c.threads = kShapes[k][0], c.vectors = kShapes[k][1];
        const int64_t most = (int64_t)c.threads * c.vectors * v - (skew ? 8 : 0);  // a multiple of 8
        c.slices = (int)((vocab + most - 1) / most);
        len = (vocab + c.slices - 1) / c.slices;
        if (rows * c.slices >= compute_units()) break;
    }
    c.slice_len = round_up(len, 8);
    c.slices = (int)((vocab + c.slice_len - 1) / c.slice_len);
    return c;
}

// Half the threads with twice the vectors hold as much as 512 with 8. Without a gradient and with eight
// blocks or more for every compute unit they are quicker, as the threads meet and search in half the
// waves, but for slices without alternatives. In us, 512 x 8 and 256 x 16, with 8 alternatives (without):
//   8192 x 32000 bf16 100, 90 (81, 80)   8192 x 18000 bf16 77, 62 (54, 46)   2048 x 32000 bf16 30, 28 (23, 24)
//   1024 x 32000 bf16 17.6, 18.4 (14.2, 15.0)   8192 x 12000 f32 70, 61 (60, 60)
//   slices: 4096 x 60000 f16 100, 88 (80, 81)   2048 x 131072 bf16 102, 94 (85, 89)
// The distillation step of 8192 x 32000 takes 188 and 197.
static Cut cut_rows(const lv_logits_args *a, int top, int skew, bool grad) {
    Cut c = smallest_block(a, top, skew, grad);
    if (!grad && c.threads == 512 && c.vectors == 8 && (top > 0 || c.slices == 1) && (int64_t)a->rows * c.slices >= 8 * compute_units())
        c.threads = 256, c.vectors = 16;
    return c;
}

// Slices of the gradient kernels, which need nothing of the rest of the row.
static Cut cut_grad(const lv_logits_args *a) {
    Cut c = {kThreads, 0, 1, 8192};
    c.slices = (int)((a->vocab + c.slice_len - 1) / c.slice_len);
    return c;
}

static int64_t piece_rows(const lv_logits_args *a, const Cut &c) {
    int64_t n = kLaunchBlocks / c.slices;
    if (n < 1) n = 1;
    return n < (int64_t)a->rows ? n : (int64_t)a->rows;
}

static size_t align256(size_t n) { return (n + 255) / 256 * 256; }

static size_t workspace_bytes(const lv_logits_args *a, Way way) {
    // nothing for a call that its entry point refuses
    if (a == nullptr || a->rows == 0 || a->vocab < 1 || a->vocab > kLargestVocab || a->count < 0 || a->rows > kMostRows ||
        a->count > (way == kLogProbs ? LV_OPS_MAX_TOP : LV_OPS_MAX_TEACHER))
        return 0;
    const bool top = way == kLogProbs && a->count > 0;
    size_t most = 0;
    for (int k = 0; k < 4; ++k) {  // the size does not depend on where the rows are, nor on the gradient
        const Cut c = cut_rows(a, top ? a->count : 0, k % 2, k / 2 != 0 && way == kDistill);
        if (c.slices == 1) continue;
        const size_t parts = (size_t)piece_rows(a, c) * c.slices;
        size_t n = align256(parts * sizeof(float4));
        if (top) n += 2 * align256(parts * a->count * sizeof(float));
        if (way == kDistill) n += align256((size_t)piece_rows(a, c) * 2 * sizeof(float));  // stats of loss_and_grad
        if (n > most) most = n;
    }
    return most;
}

static Job make_job(const lv_logits_args *a, const Cut &c, int64_t first) {
    Job j;
    j.a = *a;
    auto skip = [&](auto *&p, int64_t n) {
        if (p != nullptr) p += n;
    };
    const int64_t size = a->dtype == LV_DTYPE_F32 ? 4 : 2, tsize = a->teacher_dtype == LV_DTYPE_F32 ? 4 : 2;
    const char *z = static_cast<const char *>(a->logits);
    skip(z, first * a->stride * size);
    j.a.logits = z;
    char *g = static_cast<char *>(a->grad);
    skip(g, first * a->grad_stride * size);
    j.a.grad = g;
    const char *t = static_cast<const char *>(a->teacher_logits);
    skip(t, first * a->count * tsize);
    j.a.teacher_logits = t;
    skip(j.a.tokens, first);
    skip(j.a.teacher_tokens, first * a->count);
    skip(j.a.row_weight, first);
    skip(j.a.d_log_probs, first);
    skip(j.a.d_entropy, first);
    skip(j.a.out, first);
    skip(j.a.entropy, first);
    skip(j.a.stats, 2 * first);
    skip(j.a.top_log_probs, first * a->count);
    skip(j.a.top_tokens, first * a->count);
    j.scale = kLog2e / a->temperature;
    j.inv_temp = 1.0f / a->temperature;
    j.slices = c.slices, j.slice_len = c.slice_len;
    j.past = a->rows * a->vocab * (uint64_t)size >= kPastCaches;
    j.partial = nullptr, j.part_value = nullptr, j.part_token = nullptr;
    return j;
}

typedef void (*RowsKernel)(Job);

#define LV_BY_TYPE(dtype, KERNEL, ...) \
    ((dtype) == LV_DTYPE_F32 ? (RowsKernel)KERNEL<F32, ##__VA_ARGS__> \
     : (dtype) == LV_DTYPE_BF16 ? (RowsKernel)KERNEL<BF16, ##__VA_ARGS__> : (RowsKernel)KERNEL<F16, ##__VA_ARGS__>)

// The kernel of a cut, of those that cuts of such a call can have: 256 threads with sixteen vectors come
// without a gradient only, 1024 with sixteen with one (or on the way to one).
template <typename T, Way WAY, bool TOP, bool GRAD>
static RowsKernel pick_rows(const Cut &c) {
    if constexpr (!GRAD) {
        if (c.threads == 256 && c.vectors == 16) return rows_kernel<T, 256, 16, WAY, TOP, GRAD>;
    }
    if constexpr (WAY == kDistill) {
        if (c.threads == 1024 && c.vectors == 16) return rows_kernel<T, 1024, 16, WAY, TOP, GRAD>;
    }
    switch (c.threads * 100 + c.vectors) {
    case 6404: return rows_kernel<T, 64, 4, WAY, TOP, GRAD>;
    case 6408: return rows_kernel<T, 64, 8, WAY, TOP, GRAD>;
    case 25608: return rows_kernel<T, 256, 8, WAY, TOP, GRAD>;
    case 51208: return rows_kernel<T, 512, 8, WAY, TOP, GRAD>;
    case 51213: return rows_kernel<T, 512, 13, WAY, TOP, GRAD>;
    case 102408: return rows_kernel<T, 1024, 8, WAY, TOP, GRAD>;
    default: return nullptr;
    }
}

template <Way WAY, bool TOP, bool GRAD>
static RowsKernel pick_rows(int dtype, const Cut &c) {
    return dtype == LV_DTYPE_F32    ? pick_rows<F32, WAY, TOP, GRAD>(c)
           : dtype == LV_DTYPE_BF16 ? pick_rows<BF16, WAY, TOP, GRAD>(c)
                                    : pick_rows<F16, WAY, TOP, GRAD>(c);
}

static int run(RowsKernel k, int64_t blocks, int threads, size_t lds, const Job &job, hipStream_t s, const char *what) {
    if (k == nullptr) return fail(LV_STATUS_EXECUTION_FAILED, "%s: no kernel of %d threads a row for this cut", what, threads);
    k<<<dim3((unsigned)blocks), dim3((unsigned)threads), lds, s>>>(job);
    return launched(what);
}

// LDS for the teacher's entries of the rows that a block of `threads` per row holds.
static size_t teacher_bytes(const lv_logits_args *a, int threads = kThreads) { return (size_t)a->count * 12 * (threads == kWave ? 4 : 1); }

static int forward(const lv_logits_args *a, Way way, bool grad, void *ws, size_t ws_bytes, hipStream_t s) {
    int rc = check(a, way, true, grad);
    if (rc != LV_STATUS_SUCCESS || a->rows == 0) return rc;
    const char *what = way == kLogProbs ? "token log probs" : "distill";
    const bool top = way == kLogProbs && a->count > 0;
    const Cut c = cut_rows(a, top ? a->count : 0, row_skew(a), grad);
    const size_t need = workspace_bytes(a, way);
    if (need > 0 && (uintptr_t)ws % 256 != 0) return fail(LV_STATUS_INVALID_CONFIG, "%s: misaligned workspace", what);
    if (need > 0 && ws == nullptr) return fail(LV_STATUS_NULL_POINTER, "%s: null workspace", what);
    if (ws_bytes < need)
        return fail(LV_STATUS_INVALID_CONFIG, "%s: workspace too small: %zu bytes, %zu needed", what, ws_bytes, need);
    const int64_t step = piece_rows(a, c);
    for (int64_t first = 0; first < (int64_t)a->rows; first += step) {
        const int64_t n = (int64_t)a->rows - first < step ? (int64_t)a->rows - first : step;
        Job job = make_job(a, c, first);
        float *stats = nullptr;
        if (c.slices > 1) {
            char *p = static_cast<char *>(ws);
            const size_t parts = (size_t)step * c.slices;
            job.partial = reinterpret_cast<float4 *>(p);
            p += align256(parts * sizeof(float4));
            if (top) {
                job.part_value = reinterpret_cast<float *>(p);
                p += align256(parts * a->count * sizeof(float));
                job.part_token = reinterpret_cast<int *>(p);
            }
            stats = reinterpret_cast<float *>(p);
        }
        const size_t lds = way == kDistill ? teacher_bytes(a, c.threads) : 0;
        const bool one = grad && c.slices == 1;
        RowsKernel k = way == kDistill ? (one ? pick_rows<kDistill, false, true>(a->dtype, c) : pick_rows<kDistill, false, false>(a->dtype, c))
                                       : (top ? pick_rows<kLogProbs, true, false>(a->dtype, c) : pick_rows<kLogProbs, false, false>(a->dtype, c));
        if (one) job.a.stats = nullptr;  // not returned, and of no meaning in rows without a teacher
        job.a.rows = (uint64_t)n;
        if (c.threads == kWave) rc = run(k, (n + 3) / 4, 256, lds, job, s, what);
        else rc = run(k, n * c.slices, c.threads, lds, job, s, what);
        if (rc != LV_STATUS_SUCCESS) return rc;
        if (c.slices == 1) continue;
        if (way == kDistill && grad) job.a.stats = stats;
        k = way == kDistill ? LV_BY_TYPE(a->dtype, join_kernel, kDistill, false)
            : top           ? LV_BY_TYPE(a->dtype, join_kernel, kLogProbs, true)
                            : LV_BY_TYPE(a->dtype, join_kernel, kLogProbs, false);
        rc = run(k, n, kThreads, lds, job, s, what);
        if (rc == LV_STATUS_SUCCESS && way == kDistill && grad) {
            const Cut g = cut_grad(a);
            job.slices = g.slices, job.slice_len = g.slice_len;
            rc = run(LV_BY_TYPE(a->dtype, distill_grad_kernel), n * g.slices, kThreads, teacher_bytes(a), job, s, what);
        }
        if (rc != LV_STATUS_SUCCESS) return rc;
    }
    return LV_STATUS_SUCCESS;
}

static int backward(const lv_logits_args *a, Way way, hipStream_t s) {
    int rc = check(a, way, false, true);
    if (rc != LV_STATUS_SUCCESS || a->rows == 0) return rc;
    const Cut c = cut_grad(a);
    const int64_t step = piece_rows(a, c);
    for (int64_t first = 0; first < (int64_t)a->rows && rc == LV_STATUS_SUCCESS; first += step) {
        const int64_t n = (int64_t)a->rows - first < step ? (int64_t)a->rows - first : step;
        Job job = make_job(a, c, first);
        if (way == kDistill)
            rc = run(LV_BY_TYPE(a->dtype, distill_grad_kernel), n * c.slices, kThreads, teacher_bytes(a), job, s, "distill backward");
        else {
            // about two vectors a thread at least; slices only where a block has one row
            job.a.rows = (uint64_t)n;
            const char *what = "token log probs backward";
            const int64_t vectors = ((int64_t)a->vocab * (a->dtype == LV_DTYPE_F32 ? 4 : 2) + 15) / 16;
            if (vectors <= 32) rc = run(LV_BY_TYPE(a->dtype, log_probs_grad_kernel, 16), (n + 15) / 16, kThreads, 0, job, s, what);
            else if (vectors <= 256) rc = run(LV_BY_TYPE(a->dtype, log_probs_grad_kernel, 64), (n + 3) / 4, kThreads, 0, job, s, what);
            else rc = run(LV_BY_TYPE(a->dtype, log_probs_grad_kernel, kThreads), n * c.slices, kThreads, 0, job, s, what);
        }
    }
    return rc;
}

}  // namespace lvops

using namespace lvops;

extern "C" {

size_t lv_token_log_probs_workspace_bytes(const lv_logits_args *a) { return workspace_bytes(a, kLogProbs); }

int lv_token_log_probs_forward(const lv_logits_args *a, void *ws, size_t ws_bytes, void *stream) {
    clear_error();
    return forward(a, kLogProbs, false, ws, ws_bytes, (hipStream_t)stream);
}

int lv_token_log_probs_backward(const lv_logits_args *a, void *stream) {
    clear_error();
    return backward(a, kLogProbs, (hipStream_t)stream);
}

size_t lv_distill_workspace_bytes(const lv_logits_args *a) { return workspace_bytes(a, kDistill); }

int lv_distill_forward(const lv_logits_args *a, void *ws, size_t ws_bytes, void *stream) {
    clear_error();
    return forward(a, kDistill, false, ws, ws_bytes, (hipStream_t)stream);
}

int lv_distill_backward(const lv_logits_args *a, void *stream) {
    clear_error();
    return backward(a, kDistill, (hipStream_t)stream);
}

int lv_distill_loss_and_grad(const lv_logits_args *a, void *ws, size_t ws_bytes, void *stream) {
    clear_error();
    return forward(a, kDistill, true, ws, ws_bytes, (hipStream_t)stream);
}

}  // extern "C"
