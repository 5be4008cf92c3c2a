// Layer norm over the rows of a matrix, forward and backward.
//
// A row of up to 16384 elements lives in the registers of 8 to 1024 threads, at most 16 elements in
// each: it is read once, its mean is taken, then the mean of the squared differences from it (two
// passes over registers, so a large mean costs no digits), and the result is written. Wider rows
// are read again for each pass, by one block.
//
// The backward pass keeps the columns' sums for the weight's and the bias's gradients in registers
// while a group of threads walks its rows; a block's groups join theirs in LDS, every block leaves one
// partial row of each, and a second kernel adds those in a fixed order. Where a group has four rows at
// most, one block takes them all and writes the sums itself.
//
// What bounds it: memory, once there are rows enough. 32768 x 4096 bf16 takes 84 us forward, back to back,
// where the last of its output is still in the 256 MiB cache as a call ends (95 us, 5.7 TB/s, with stores
// past that cache), and 145 us backward (5.5 TB/s, 7.5 us of it the second kernel; 17 MB of partial
// rows); a large copy runs at 6.15. 174762 x 768 bf16: 88 us (94 past the cache) and 154 (5.2). Blocks
// therefore walk many rows, so that weights are read once a block and the next row is under way while one
// is worked on. Small calls are bound by the launches: 8192 x 768 f32 takes 9.7 us, 16384 x 768 bf16
// backward 21.4 with 3.9 of them the second kernel, one row 3.4 and the host's part of the call 6.4. Rows
// of odd 16-bit widths start half way into a word and take a fifth to a quarter longer (131200 x 1023:
// 110 us, 131072 x 1024: 85).
// Rows above 16384 elements: 3.1 TB/s forward, 1.9 backward (6710 x 20000 bf16).
#include "ops_common.h"

namespace lvops {

struct LnJob {
    const void *x, *dy;
    void *out;
    const void *weight, *bias;
    float *mean, *rstd;
    void *dweight, *dbias;
    float *partial;  // [blocks][2][width]
    int64_t rows, width, x_stride, dy_stride, out_stride;
    float eps;
    bool past;       // go past the caches
    int blocks;      // partial rows; 1: the block writes the results itself, 0: no columns wanted
};

// VEC elements of the weight or bias (type W, T itself or f32) from column e; `absent` without one.
template <typename W, int VEC>
static __device__ __forceinline__ void load_columns(const void *p, int64_t e, int64_t width, float absent, float (&v)[VEC]) {
    const store_t<W> *w = static_cast<const store_t<W> *>(p);
    constexpr int WV = Type<W>::kVec;
    static_assert(VEC % WV == 0, "the weight is of the rows' type or wider");
    if (w != nullptr && e + VEC <= width) {
#pragma unroll
        for (int c = 0; c < VEC / WV; ++c) {
            float t[WV];
            Type<W>::unpack(load16<W>(w + e + c * WV), t);
#pragma unroll
            for (int j = 0; j < WV; ++j) v[c * WV + j] = t[j];
        }
    } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[j] = w != nullptr && e + j < width ? Type<W>::load(w + e + j) : absent;
    }
}

// A vector of a row as it is in memory; what lies past the row's end reads as 0.
template <typename T>
static __device__ __forceinline__ u32x4 load_raw(const store_t<T> *row, int64_t e, int64_t width, bool past) {
    if (e + Type<T>::kVec <= width) return load16<T>(row + e, past);
    float v[Type<T>::kVec];
#pragma unroll
    for (int j = 0; j < Type<T>::kVec; ++j) v[j] = e + j < width ? Type<T>::load(row + e + j) : 0.0f;
    return Type<T>::pack(v);
}

// Groups of TPR threads (8 to 1024: part of a wave, or several) walk the rows, each thread its NV vectors
// of every row and its columns' weight and bias; the next row's vectors are under way while one is
// worked on. Each wave takes its own mean and squared differences from it; with several waves to a row
// these meet in LDS, where the differences of the waves' means from the row's are added (one barrier).
template <typename T, typename W, int TPR, int NV, int THREADS>
__global__ void __launch_bounds__(THREADS, NV * Type<T>::kVec <= 8 ? 8 : TPR < 256 ? 5 : 4) ln_forward(LnJob job) {
    constexpr int V = Type<T>::kVec, kGroups = THREADS / TPR, kWaves = TPR / kWave, kLanes = TPR < kWave ? TPR : kWave;
    __shared__ float red[2][2][THREADS / kWave];
    const int lane = threadIdx.x % TPR, group = threadIdx.x / TPR, wave = threadIdx.x / kWave;
    const float inv = 1.0f / (float)job.width;
    float w[NV][V], b[NV][V];
    float share[kWaves > 1 ? kWaves : 1];  // of the row's elements that each of its waves holds
    float inv_n = inv;                     // 1 / those of this wave
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int64_t e = (int64_t)(i * TPR + lane) * V;
        load_columns<W>(job.weight, e, job.width, 1.0f, w[i]);
        load_columns<W>(job.bias, e, job.width, 0.0f, b[i]);
    }
    if (kWaves > 1) {
#pragma unroll
        for (int k = 0; k < kWaves; ++k) {
            int n = 0;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int64_t left = job.width - (int64_t)(i * TPR + k * kWave) * V;
                n += left <= 0 ? 0 : left < kWave * V ? (int)left : kWave * V;
            }
            share[k] = (float)n * inv;
            if (k == wave % kWaves) inv_n = n > 0 ? 1.0f / (float)n : 0.0f;
        }
    }
    u32x4 next[NV];
    auto fetch = [&](int64_t r) {
        const store_t<T> *x = static_cast<const store_t<T> *>(job.x) + r * job.x_stride;
#pragma unroll
        for (int i = 0; i < NV; ++i) next[i] = load_raw<T>(x, (int64_t)(i * TPR + lane) * V, job.width, job.past);
    };
    const int64_t step = (int64_t)gridDim.x * kGroups;
    int64_t r = (int64_t)blockIdx.x * kGroups + group;
    if (r < job.rows) fetch(r);
    int turn = 0;
    // the groups of a block meet at barriers: all stay until the block's first row is past the end
    for (int64_t first = (int64_t)blockIdx.x * kGroups; first < job.rows; first += step, r += step) {
        float v[NV][V];
#pragma unroll
        for (int i = 0; i < NV; ++i) Type<T>::unpack(next[i], v[i]);
        if (r + step < job.rows) fetch(r + step);
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < V; ++j) sum += v[i][j];  // 0 past the row's end
        float mean = lanes_sum<kLanes>(sum) * inv_n;
        float sq = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int64_t e = (int64_t)(i * TPR + lane) * V;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float d = e + j < job.width ? v[i][j] - mean : 0.0f;
                sq = fmaf(d, d, sq);
            }
        }
        sq = lanes_sum<kLanes>(sq);
        if (kWaves > 1) {
            // two sets of slots in turn: a wave may be one row ahead of the slowest reader
            if (threadIdx.x % kWave == 0) {
                red[turn][0][wave] = mean;
                red[turn][1][wave] = sq;
            }
            __syncthreads();
            mean = sq = 0.0f;
#pragma unroll
            for (int k = 0; k < kWaves; ++k) mean = fmaf(red[turn][0][group * kWaves + k], share[k], mean);
#pragma unroll
            for (int k = 0; k < kWaves; ++k) {
                const float d = red[turn][0][group * kWaves + k] - mean;
                sq += fmaf(d * d, share[k] * (float)job.width, red[turn][1][group * kWaves + k]);
            }
            turn ^= 1;
        }
        const float rstd = 1.0f / sqrtf(sq * inv + job.eps);
        if (r >= job.rows) continue;
        store_t<T> *y = static_cast<store_t<T> *>(job.out) + r * job.out_stride;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int64_t e = (int64_t)(i * TPR + lane) * V;
            if (e >= job.width) continue;
#pragma unroll
            for (int j = 0; j < V; ++j) v[i][j] = fmaf((v[i][j] - mean) * rstd, w[i][j], b[i][j]);
            store_edge<T>(y, e, job.width, v[i]);
        }
        if (lane == 0) {
            job.mean[r] = mean;
            job.rstd[r] = rstd;
        }
    }
}

// Rows wider than a block's registers: three passes over memory.
template <typename T, typename W>
__global__ void __launch_bounds__(256) ln_forward_wide(LnJob job) {
    constexpr int V = Type<T>::kVec;
    __shared__ float red[2][4];
    const float inv = 1.0f / (float)job.width;
    for (int64_t r = blockIdx.x; r < job.rows; r += gridDim.x) {
        const store_t<T> *x = static_cast<const store_t<T> *>(job.x) + r * job.x_stride;
        store_t<T> *y = static_cast<store_t<T> *>(job.out) + r * job.out_stride;
        float v[V], sum = 0.0f, sq = 0.0f;
        for (int64_t e = (int64_t)threadIdx.x * V; e < job.width; e += 256 * V) {
            load_edge<T>(x, e, job.width, 0.0f, v);
#pragma unroll
            for (int j = 0; j < V; ++j) sum += v[j];
        }
        const float mean = block_sum<256>(sum, red[0]) * inv;
        for (int64_t e = (int64_t)threadIdx.x * V; e < job.width; e += 256 * V) {
            load_edge<T>(x, e, job.width, mean, v);
#pragma unroll
            for (int j = 0; j < V; ++j) sq = fmaf(v[j] - mean, v[j] - mean, sq);
        }
        const float rstd = 1.0f / sqrtf(block_sum<256>(sq, red[1]) * inv + job.eps);
        for (int64_t e = (int64_t)threadIdx.x * V; e < job.width; e += 256 * V) {
            float w[V], b[V];
            load_edge<T>(x, e, job.width, mean, v);
            load_columns<W>(job.weight, e, job.width, 1.0f, w);
            load_columns<W>(job.bias, e, job.width, 0.0f, b);
#pragma unroll
            for (int j = 0; j < V; ++j) w[j] = fmaf((v[j] - mean) * rstd, w[j], b[j]);
            store_edge<T>(y, e, job.width, w);
        }
        if (threadIdx.x == 0) {
            job.mean[r] = mean;
            job.rstd[r] = rstd;
        }
        __syncthreads();  // red is written again in the next row
    }
}

// Groups of TPR threads (8 to 1024) walk the rows, each thread its NV vectors of every row; the next row's vectors
// are under way while one is worked on. Per row the group's two sums cost one barrier (none for a
// wave), and x and dy are unpacked twice rather than kept unpacked across it. Four waves a SIMD leave 128
// registers: f32 rows above 512 columns and 16-bit rows above 4096 spill 4 to 20 of them (32768 x 4096 f32
// 286 us, 5.6 TB/s; 16384 x 768 f32 31.8, 4.7; 16384 x 8192 bf16 161, 5.0).
template <typename T, typename W, int TPR, int NV, int THREADS>
__global__ void __launch_bounds__(THREADS, 4) ln_backward(LnJob job) {
    constexpr int V = Type<T>::kVec, kGroups = THREADS / TPR, kWaves = TPR / kWave, kLanes = TPR < kWave ? TPR : kWave;
    constexpr int kCols = NV * V * TPR;                              // columns that a group covers
    constexpr int kParts = TPR < kWave ? THREADS / kWave : kGroups;  // sums of the columns, a wave's groups as one
    // 16 f32 elements a thread fill the registers without a second row, and so do sixteen waves' sums
    constexpr bool kAhead = NV * 4 * 4 <= 32 && TPR <= 512;
    __shared__ float red[2][2][THREADS / kWave];
    __shared__ float4 cols[kParts > 1 ? kParts : 1][kParts > 1 ? kCols / 4 : 1];
    const int lane = threadIdx.x % TPR, group = threadIdx.x / TPR, wave = threadIdx.x / kWave;
    const float inv = 1.0f / (float)job.width;
    float w[NV][V], dw[NV][V], db[NV][V];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        load_columns<W>(job.weight, (int64_t)(i * TPR + lane) * V, job.width, 1.0f, w[i]);
#pragma unroll
        for (int j = 0; j < V; ++j) dw[i][j] = db[i][j] = 0.0f;
    }
    u32x4 next_x[NV], next_dy[NV];
    float next_mean = 0.0f, next_rstd = 0.0f;
    auto fetch = [&](int64_t r) {
        const store_t<T> *x = static_cast<const store_t<T> *>(job.x) + r * job.x_stride;
        const store_t<T> *dy = static_cast<const store_t<T> *>(job.dy) + r * job.dy_stride;
        next_mean = job.mean[r], next_rstd = job.rstd[r];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int64_t e = (int64_t)(i * TPR + lane) * V;
            next_x[i] = load_raw<T>(x, e, job.width, job.past);
            next_dy[i] = load_raw<T>(dy, e, job.width, job.past);
        }
    };
    const int64_t step = (int64_t)gridDim.x * kGroups;
    int64_t r = (int64_t)blockIdx.x * kGroups + group;
    if (kAhead && r < job.rows) fetch(r);
    int turn = 0;
    // the groups of a block meet at barriers: all stay until the block's first row is past the end
    for (int64_t first = (int64_t)blockIdx.x * kGroups; first < job.rows; first += step, r += step) {
        const bool here = r < job.rows;
        u32x4 x[NV], dy[NV];
        if (!kAhead && here) fetch(r);
        const float mean = next_mean, rstd = next_rstd;
        float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i) x[i] = next_x[i], dy[i] = next_dy[i];
        if (kAhead && r + step < job.rows) fetch(r + step);
        if (here) {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                float xv[V], g[V];
                Type<T>::unpack(x[i], xv);
                Type<T>::unpack(dy[i], g);
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float xh = (xv[j] - mean) * rstd;
                    dw[i][j] = fmaf(g[j], xh, dw[i][j]);
                    db[i][j] += g[j];
                    g[j] *= w[i][j];
                    s1 += g[j];
                    s2 = fmaf(g[j], xh, s2);
                }
            }
        }
        s1 = lanes_sum<kLanes>(s1);
        s2 = lanes_sum<kLanes>(s2);
        if (kWaves > 1) {
            // two sets of slots in turn: a wave may be one row ahead of the slowest reader
            if (threadIdx.x % kWave == 0) {
                red[turn][0][wave] = s1;
                red[turn][1][wave] = s2;
            }
            __syncthreads();
            s1 = s2 = 0.0f;
#pragma unroll
            for (int k = 0; k < kWaves; ++k) {
                s1 += red[turn][0][group * kWaves + k];
                s2 += red[turn][1][group * kWaves + k];
            }
            turn ^= 1;
        }
        if (here && job.out != nullptr) {
            store_t<T> *out = static_cast<store_t<T> *>(job.out) + r * job.out_stride;
            const float a = -rstd * (s1 * inv), b = -rstd * (s2 * inv);
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int64_t e = (int64_t)(i * TPR + lane) * V;
                if (e >= job.width) continue;
                float xv[V], g[V];
                asm volatile("" : "+v"(x[i]), "+v"(dy[i]));  // or the compiler keeps both unpacked from above
                Type<T>::unpack(x[i], xv);
                Type<T>::unpack(dy[i], g);
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float xh = (xv[j] - mean) * rstd;
                    g[j] = fmaf(xh, b, fmaf(g[j] * w[i][j], rstd, a));
                }
                store_edge<T>(out, e, job.width, g, job.past);
            }
        }
    }
    if (job.blocks == 0) return;  // no columns wanted
    const bool alone = job.blocks == 1;  // these sums are the results
    float *pw = alone ? nullptr : job.partial + (int64_t)blockIdx.x * 2 * job.width, *pb = pw + job.width;
    // column c's sums: of the weight's gradient, then of the bias's
    auto put = [&](bool second, int64_t c, float sum) {
        void *out = second ? job.dbias : job.dweight;
        if (!alone) (second ? pb : pw)[c] = sum;
        else if (out != nullptr) Type<W>::store(static_cast<store_t<W> *>(out) + c, sum);
    };
    if (TPR < kWave) {  // a wave's groups first
#pragma unroll
        for (int o = TPR; o < kWave; o *= 2)
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    dw[i][j] += __shfl_xor(dw[i][j], o, kWave);
                    db[i][j] += __shfl_xor(db[i][j], o, kWave);
                }
    }
    const int part = TPR < kWave ? wave : group;
#pragma unroll
    for (int second = 0; second < 2; ++second) {
        const float(&sum)[NV][V] = second ? db : dw;
        if (kParts > 1) {  // through LDS, in the parts' order
            if (second) __syncthreads();
            if (threadIdx.x % (TPR < kWave ? kWave : TPR) < TPR) {
#pragma unroll
                for (int i = 0; i < NV; ++i)
#pragma unroll
                    for (int j = 0; j < V; j += 4)
                        cols[part][((i * TPR + lane) * V + j) / 4] =
                            make_float4(sum[i][j], sum[i][j + 1], sum[i][j + 2], sum[i][j + 3]);
            }
            __syncthreads();
            for (int c = threadIdx.x; c < job.width; c += THREADS) {
                float total = 0.0f;
#pragma unroll
                for (int k = 0; k < kParts; ++k) total += reinterpret_cast<const float *>(cols[k])[c];
                put(second, c, total);
            }
        } else {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int64_t e = (int64_t)(i * TPR + lane) * V;
#pragma unroll
                for (int j = 0; j < V; ++j)
                    if (e + j < job.width) put(second, e + j, sum[i][j]);
            }
        }
    }
}

template <typename T, typename W>
__global__ void __launch_bounds__(256) ln_backward_wide(LnJob job) {
    constexpr int V = Type<T>::kVec;
    __shared__ float red[2][4];
    const float inv = 1.0f / (float)job.width;
    for (int64_t r = blockIdx.x; r < job.rows; r += gridDim.x) {
        const store_t<T> *x = static_cast<const store_t<T> *>(job.x) + r * job.x_stride;
        const store_t<T> *dy = static_cast<const store_t<T> *>(job.dy) + r * job.dy_stride;
        store_t<T> *out = static_cast<store_t<T> *>(job.out) + r * job.out_stride;
        const float mean = job.mean[r], rstd = job.rstd[r];
        float xv[V], g[V], w[V], s1 = 0.0f, s2 = 0.0f;
        for (int64_t e = (int64_t)threadIdx.x * V; e < job.width; e += 256 * V) {
            load_edge<T>(x, e, job.width, mean, xv);
            load_edge<T>(dy, e, job.width, 0.0f, g);
            load_columns<W>(job.weight, e, job.width, 1.0f, w);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                s1 = fmaf(g[j], w[j], s1);
                s2 = fmaf(g[j] * w[j], (xv[j] - mean) * rstd, s2);
            }
        }
        const float m1 = block_sum<256>(s1, red[0]) * inv, m2 = block_sum<256>(s2, red[1]) * inv;
        for (int64_t e = (int64_t)threadIdx.x * V; e < job.width; e += 256 * V) {
            load_edge<T>(x, e, job.width, mean, xv);
            load_edge<T>(dy, e, job.width, 0.0f, g);
            load_columns<W>(job.weight, e, job.width, 1.0f, w);
#pragma unroll
            for (int j = 0; j < V; ++j) g[j] = rstd * (g[j] * w[j] - m1 - (xv[j] - mean) * rstd * m2);
            store_edge<T>(out, e, job.width, g);
        }
        __syncthreads();  // red is written again in the next row
    }
}

// Partial sums of the weight's and bias's gradients of wide rows: one thread a column, block row
// blockIdx.y takes every gridDim.y-th row.
template <typename T>
__global__ void __launch_bounds__(256) ln_columns_wide(LnJob job) {
    const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (c >= job.width) return;
    float dw = 0.0f, db = 0.0f;
    for (int64_t r = blockIdx.y; r < job.rows; r += gridDim.y) {
        const float x = Type<T>::load(static_cast<const store_t<T> *>(job.x) + r * job.x_stride + c);
        const float dy = Type<T>::load(static_cast<const store_t<T> *>(job.dy) + r * job.dy_stride + c);
        dw = fmaf(dy, (x - job.mean[r]) * job.rstd[r], dw);
        db += dy;
    }
    float *p = job.partial + (int64_t)blockIdx.y * 2 * job.width;
    p[c] = dw;
    p[job.width + c] = db;
}

// The blocks' partial rows, added up: 16 columns a block, 64 threads to a column, each of which takes
// every 64th partial row. blockIdx.y 0 is the weight's gradient, 1 the bias's.
template <typename W>
__global__ void __launch_bounds__(1024) ln_reduce_columns(LnJob job) {
    constexpr int kCols = 16, kLanes = 64, kAhead = 8;
    __shared__ float part[kLanes][kCols + 1];
    void *out = blockIdx.y ? job.dbias : job.dweight;
    if (out == nullptr) return;
    const int col = threadIdx.x % kCols, k = threadIdx.x / kCols;
    const int64_t c = (int64_t)blockIdx.x * kCols + col;
    float s = 0.0f;
    if (c < job.width) {
        const float *p = job.partial + (int64_t)blockIdx.y * job.width + c;
        for (int b = k; b < job.blocks; b += kAhead * kLanes) {
            float v[kAhead];
#pragma unroll
            for (int i = 0; i < kAhead; ++i) {
                const int at = b + i * kLanes;
                v[i] = at < job.blocks ? p[(int64_t)at * 2 * job.width] : 0.0f;
            }
#pragma unroll
            for (int i = 0; i < kAhead; ++i) s += v[i];
        }
    }
    part[k][col] = s;
#pragma unroll
    for (int h = kLanes / 2; h; h /= 2) {
        __syncthreads();
        if (k < h) part[k][col] += part[k + h][col];
    }
    if (k == 0 && c < job.width) Type<W>::store(static_cast<store_t<W> *>(out) + c, part[0][col]);
}

// ------------------------------------------------------------------------------------- host side

static int check(const lv_layer_norm_args *a, bool backward) {
    if (a == nullptr) return fail(LV_STATUS_NULL_POINTER, "layer norm: null arguments");
    if (a->dtype < 0 || a->dtype > 2) return fail(LV_STATUS_INVALID_CONFIG, "layer norm: invalid dtype code %d", a->dtype);
    if (a->weight_dtype != LV_DTYPE_F32 && a->weight_dtype != a->dtype)
        return fail(LV_STATUS_INVALID_CONFIG, "layer norm: the weight is f32 or of x's dtype, not code %d", a->weight_dtype);
    if (a->width < 1 || a->width > (1ull << 30) || a->rows > (1ull << 40))
        return fail(LV_STATUS_INVALID_CONFIG, "layer norm: invalid size %llu x %llu", (unsigned long long)a->rows,
                    (unsigned long long)a->width);
    if (!backward && !(a->eps >= 0.0f)) return fail(LV_STATUS_INVALID_CONFIG, "layer norm: invalid eps: %g", a->eps);
    if (a->rows == 0) return LV_STATUS_SUCCESS;
    if (a->x == nullptr || a->mean == nullptr || a->rstd == nullptr || (backward ? a->dy == nullptr : a->out == nullptr))
        return fail(LV_STATUS_NULL_POINTER, "layer norm: null pointer");
    const int64_t w = (int64_t)a->width;
    if (a->rows > 1 && (a->x_stride < 0 || (a->out != nullptr && a->out_stride < w) || (backward && a->dy_stride < 0)))
        return fail(LV_STATUS_INVALID_CONFIG, "layer norm: invalid row stride");
    return LV_STATUS_SUCCESS;
}

static LnJob make_job(const lv_layer_norm_args *a) {
    LnJob j;
    j.x = a->x, j.dy = a->dy, j.out = a->out, j.weight = a->weight, j.bias = a->bias;
    j.mean = a->mean, j.rstd = a->rstd, j.dweight = a->dweight, j.dbias = a->dbias;
    j.partial = nullptr;
    j.rows = (int64_t)a->rows, j.width = (int64_t)a->width;
    j.x_stride = a->x_stride, j.dy_stride = a->dy_stride, j.out_stride = a->out_stride;
    j.eps = a->eps;
    j.past = a->rows * a->width * (a->dtype == LV_DTYPE_F32 ? 4 : 2) * (a->dy != nullptr ? 2 : 1) >= kPastCaches;
    j.blocks = 0;
    return j;
}

typedef void (*LnKernel)(LnJob);
struct Pick {
    LnKernel kernel;
    int rows_per_block, threads;
};

// Widest row that a block's registers hold.
constexpr int64_t kWidest = 16384;
// Most rows for each group of a block that does without partial rows.
constexpr int64_t kAlone = 4;

// The register kernel of a width: the fewest threads to a row that hold it with at most 16 elements
// each, so that columns' weights or sums fit beside the row.
template <typename T, typename W, bool BACK>
static Pick pick_registers(int64_t width) {
    constexpr int V = Type<T>::kVec, S = 8 / V;  // S: vectors per eight elements
    if constexpr (BACK) {
#define LV_PICK(TPR, N, THREADS) \
    if (width <= (int64_t)(TPR) * 8 * (N)) return {ln_backward<T, W, TPR, (N) * S, THREADS>, (THREADS) / (TPR), THREADS};
        LV_PICK(8, 1, 512)
        LV_PICK(16, 1, 512)
        LV_PICK(32, 1, 512)
        LV_PICK(64, 1, 512)
        LV_PICK(64, 2, 512)
        LV_PICK(128, 2, 512)
        LV_PICK(256, 2, 512)
        LV_PICK(512, 2, 512)
        LV_PICK(1024, 2, 1024)
#undef LV_PICK
        return {ln_backward_wide<T, W>, 1, 256};
    } else {
#define LV_PICK(TPR, N, THREADS) \
    if (width <= (int64_t)(TPR) * 8 * (N)) return {ln_forward<T, W, TPR, (N) * S, THREADS>, (THREADS) / (TPR), THREADS};
        LV_PICK(8, 1, 256)
        LV_PICK(16, 1, 256)
        LV_PICK(32, 1, 256)
        LV_PICK(64, 1, 256)
        LV_PICK(64, 2, 256)
        LV_PICK(128, 2, 256)
        LV_PICK(256, 2, 256)
        LV_PICK(512, 2, 512)
        LV_PICK(1024, 2, 1024)
#undef LV_PICK
        return {ln_forward_wide<T, W>, 1, 256};
    }
}

template <bool BACK>
static Pick pick(int dtype, int wdtype, int64_t width) {
    if (dtype == LV_DTYPE_F32) return pick_registers<F32, F32, BACK>(width);
    if (dtype == LV_DTYPE_BF16)
        return wdtype == LV_DTYPE_F32 ? pick_registers<BF16, F32, BACK>(width) : pick_registers<BF16, BF16, BACK>(width);
    return wdtype == LV_DTYPE_F32 ? pick_registers<F16, F32, BACK>(width) : pick_registers<F16, F16, BACK>(width);
}

static LnKernel pick_columns(int dtype) {
    return dtype == LV_DTYPE_F32 ? ln_columns_wide<F32> : dtype == LV_DTYPE_BF16 ? ln_columns_wide<BF16> : ln_columns_wide<F16>;
}

static LnKernel pick_reduce(int wdtype) {
    return wdtype == LV_DTYPE_F32 ? ln_reduce_columns<F32> : wdtype == LV_DTYPE_BF16 ? ln_reduce_columns<BF16>
                                                                                      : ln_reduce_columns<F16>;
}

static bool wants_columns(const lv_layer_norm_args *a) { return a->dweight != nullptr || a->dbias != nullptr; }

// Blocks of the backward launch, and so partial rows: two blocks a compute unit walk all rows. Where
// columns are wanted, one alone does if it has four rows or fewer for each of its groups, which saves
// the second launch; the gradient of x by itself has none to save (32 rows of 768 bf16 take 4.2 us in
// four blocks and 8.8 in one, 4 of 16384 f32 5.3 and 11.7).
static int backward_blocks(const lv_layer_norm_args *a) {
    const int64_t width = (int64_t)a->width, rows = (int64_t)a->rows;
    if (width > kWidest) return (int)(rows < 2 * compute_units() ? rows : 2 * compute_units());
    const int64_t per = pick<true>(a->dtype, a->weight_dtype, width).rows_per_block;
    const int64_t need = (rows + per - 1) / per, most = 2 * compute_units();
    return need <= kAlone && wants_columns(a) ? 1 : (int)(need < most ? need : most);
}

}  // namespace lvops

using namespace lvops;

extern "C" int lv_layer_norm_forward(const lv_layer_norm_args *a, void *stream) {
    clear_error();
    int rc = check(a, false);
    if (rc != LV_STATUS_SUCCESS || a->rows == 0) return rc;
    LnJob job = make_job(a);
    Pick p = pick<false>(a->dtype, a->weight_dtype, job.width);
    int64_t blocks = (job.rows + p.rows_per_block - 1) / p.rows_per_block;
    const int64_t most = (job.width <= kWidest ? (job.width <= 512 ? 8 : job.width <= 2048 ? 5 : 4) * 256 / p.threads : 64) * (int64_t)compute_units();
    if (blocks > most) blocks = most;
    p.kernel<<<dim3((unsigned)blocks), dim3((unsigned)p.threads), 0, (hipStream_t)stream>>>(job);
    return launched("layer norm");
}

extern "C" size_t lv_layer_norm_workspace_bytes(const lv_layer_norm_args *a) {
    if (a == nullptr || a->rows == 0 || a->width == 0 || a->dtype < 0 || a->dtype > 2 || !wants_columns(a)) return 0;
    const int blocks = backward_blocks(a);
    return blocks == 1 && a->width <= kWidest ? 0 : (size_t)blocks * 2 * a->width * sizeof(float);
}

extern "C" int lv_layer_norm_backward(const lv_layer_norm_args *a, void *workspace, size_t workspace_bytes, void *stream) {
    clear_error();
    int rc = check(a, true);
    if (rc != LV_STATUS_SUCCESS) return rc;
    LnJob job = make_job(a);
    const bool columns = wants_columns(a);
    const size_t need = lv_layer_norm_workspace_bytes(a);
    if (need > 0 && workspace == nullptr) return fail(LV_STATUS_NULL_POINTER, "layer norm: null workspace");
    if (workspace_bytes < need)
        return fail(LV_STATUS_INVALID_CONFIG, "layer norm: workspace too small: %zu bytes, %zu needed", workspace_bytes, need);
    job.partial = static_cast<float *>(workspace);
    job.blocks = columns && a->rows != 0 ? backward_blocks(a) : 0;
    const bool alone = job.blocks == 1 && job.width <= kWidest;
    const hipStream_t s = (hipStream_t)stream;
    if (a->rows != 0 && (columns || job.out != nullptr)) {
        if (job.width <= kWidest) {
            Pick p = pick<true>(a->dtype, a->weight_dtype, job.width);
            const int blocks = job.blocks != 0 ? job.blocks : backward_blocks(a);
            p.kernel<<<dim3((unsigned)blocks), dim3((unsigned)p.threads), 0, s>>>(job);
            rc = launched("layer norm backward");
        } else {
            if (job.out != nullptr) {
                Pick p = pick<true>(a->dtype, a->weight_dtype, job.width);
                int64_t blocks = job.rows < (1 << 20) ? job.rows : 1 << 20;
                p.kernel<<<dim3((unsigned)blocks), dim3(256), 0, s>>>(job);
                rc = launched("layer norm backward");
            }
            if (rc == LV_STATUS_SUCCESS && columns) {
                pick_columns(a->dtype)<<<dim3((unsigned)((job.width + 255) / 256), (unsigned)job.blocks), dim3(256), 0, s>>>(job);
                rc = launched("layer norm backward, columns");
            }
        }
        if (rc != LV_STATUS_SUCCESS) return rc;
    }
    if (columns && !alone) {  // without rows: zeros
        pick_reduce(a->weight_dtype)<<<dim3((unsigned)((job.width + 15) / 16), 2), dim3(1024), 0, s>>>(job);
        rc = launched("layer norm backward, weights");
    }
    return rc;
}
