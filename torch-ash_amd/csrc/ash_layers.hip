// The layers that read a grid's features: the C ABI of the dense layer (its kernels are
// in ash_linear.hip) and the root-mean-square norm with the residual's addition, its
// gradients, and its output in 8 bits.
//
// Norm: s = x + residual, i = (mean s^2 + eps)^-1/2, y = s i w.  One pass: a row is
// held in the registers of the lanes that share it (kLanes, eight consecutive values of
// the row each, kChunks times), whose sums go by lane exchanges, of a whole workgroup
// through LDS.  All arithmetic is float32; y is made of s before it is rounded for the
// caller, the gradients of s as it was rounded, which is what the caller keeps (half a
// step of the type in s i, as much as y itself is rounded by).
//
// Bound by memory: 65 536 rows of 1024 bf16 with a residual read and write 537 MB forward in
// 113 us and as much backward in 112 (4.8 TB/s, what a copy reaches); 262 144 rows of 256
// bf16 with a residual to 8 bits and the sum 92 us (470 MB, 5.1 TB/s).  A few rows are bound by the launch, 4 us.
#include "ash_linear.h"

namespace ash {
namespace {

constexpr int kThreads = 256;

template <typename T, int N> struct Values { T v[N]; };

// Eight consecutive values, those at `left` and beyond zeros and not read; memory need
// not be aligned to more than a value.
template <typename T> __device__ inline void read8(const T* p, int64_t left, float (&out)[8]) {
    Values<T, 8> r;
    if (left >= 8) {
        __builtin_memcpy(&r, p, sizeof(r));
    } else {
        __builtin_memset(&r, 0, sizeof(r));
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (i < left) r.v[i] = p[i];
        }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) out[i] = static_cast<float>(r.v[i]);
}

template <typename T> __device__ inline void write8(T* p, int64_t left, const float (&v)[8]) {
    Values<T, 8> r;
#pragma unroll
    for (int i = 0; i < 8; ++i) r.v[i] = static_cast<T>(v[i]);
    if (left >= 8) {
        __builtin_memcpy(p, &r, sizeof(r));
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (i < left) p[i] = r.v[i];
        }
    }
}

constexpr float kE4m3Max = 448.0f;

__device__ inline void write8_e4m3(uint8_t* p, int64_t left, const float (&v)[8]) {
    uint32_t w[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        int r = 0;
        r = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * h], v[4 * h + 1], r, false);
        r = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * h + 2], v[4 * h + 3], r, true);
        w[h] = static_cast<uint32_t>(r);
    }
    if (left >= 8) {
        __builtin_memcpy(p, w, 8);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (i < left) p[i] = static_cast<uint8_t>(w[i >> 2] >> (8 * (i & 3)));
        }
    }
}

struct Sum { static __device__ float of(float a, float b) { return a + b; } };
struct Max { static __device__ float of(float a, float b) { return fmaxf(a, b); } };

// N values joined over the kLanes lanes that share a row; every lane gets them.  A whole
// workgroup joins through `space` (every thread has to take part).
template <int kLanes, typename Op, int N>
__device__ inline void join(float (&v)[N], float (*space)[N]) {
    constexpr int kIn = kLanes < 64 ? kLanes : 64;
#pragma unroll
    for (int step = 1; step < kIn; step <<= 1) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = Op::of(v[i], __shfl_xor(v[i], step));
    }
    if constexpr (kLanes > 64) {
        __syncthreads();   // the space's last use is over
        if ((threadIdx.x & 63) == 0) {
#pragma unroll
            for (int i = 0; i < N; ++i) space[threadIdx.x >> 6][i] = v[i];
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; ++i) {
            v[i] = space[0][i];
#pragma unroll
            for (int w = 1; w < kLanes / 64; ++w) v[i] = Op::of(v[i], space[w][i]);
        }
    }
}

struct NormDev {
    ash_norm_args a;
    float inverse_cols;
    int64_t first;   // forward: row of the launch's first workgroup
};

// A grid holds fewer than 2^32 threads: longer work takes several launches of this many
// workgroups.
constexpr int64_t kMaxGroups = 1 << 23;

// Where a thread stands: row of the workgroup's, lane of the row's, first value of chunk i.
template <int kLanes> struct Lane {
    static constexpr int kRows = kThreads / kLanes;
    int row, lane;
    __device__ Lane() : row(threadIdx.x / kLanes), lane(threadIdx.x % kLanes) {}
    __device__ int64_t at(int chunk) const { return (static_cast<int64_t>(chunk) * kLanes + lane) * 8; }
};

template <typename T, int kLanes, int kChunks>
__global__ __launch_bounds__(kThreads) void norm_forward_kernel(const NormDev d) {
    const Lane<kLanes> me;
    const ash_norm_args& a = d.a;
    __shared__ float space[kThreads / 64][1];
    const int64_t row = d.first + static_cast<int64_t>(blockIdx.x) * Lane<kLanes>::kRows + me.row;
    const bool there = row < a.rows;
    if (kLanes <= 64 && !there) return;
    float s[kChunks][8];
    float sum[1] = {0.0f};
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
        const int64_t at = me.at(c), left = there ? a.cols - at : 0;
        read8(static_cast<const T*>(a.input) + row * a.input_stride + at, left, s[c]);
        if (a.residual != nullptr) {
            float more[8];
            read8(static_cast<const T*>(a.residual) + row * a.residual_stride + at, left, more);
#pragma unroll
            for (int i = 0; i < 8; ++i) s[c][i] += more[i];
        }
    }
    if (a.sum_out != nullptr) {
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
            const int64_t at = me.at(c);
            write8(static_cast<T*>(a.sum_out) + row * a.cols + at, there ? a.cols - at : 0, s[c]);
        }
    }
    if (a.normalise) {
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
#pragma unroll
            for (int i = 0; i < 8; ++i) sum[0] += s[c][i] * s[c][i];
        }
        join<kLanes, Sum>(sum, space);
        const float inverse = 1.0f / sqrtf(sum[0] * d.inverse_cols + a.eps);
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
            float w[8] = {1.0f, 1.0f, 1.0f, 1.0f, 1.0f, 1.0f, 1.0f, 1.0f};
            const int64_t at = me.at(c);
            if (a.weight != nullptr) read8(static_cast<const T*>(a.weight) + at, a.cols - at, w);
#pragma unroll
            for (int i = 0; i < 8; ++i) s[c][i] *= inverse * w[i];
        }
    }
    if (a.scales == nullptr) {
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
            const int64_t at = me.at(c);
            write8(static_cast<T*>(a.output) + row * a.cols + at, there ? a.cols - at : 0, s[c]);
        }
        return;
    }
    // 8 bits: the row's largest magnitude becomes the largest number of the type.  A row
    // that holds an infinity or NaN has the scale NaN; one of zeros has one.
    float most[1] = {0.0f};
    bool finite = true;
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
        const int64_t left = a.cols - me.at(c);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float v = i < left ? fabsf(s[c][i]) : 0.0f;
            most[0] = fmaxf(most[0], v);
            finite = finite && v <= 3.4028235e38f;
        }
    }
    if (!finite) most[0] = __builtin_inff();
    join<kLanes, Max>(most, space);
    float scale = most[0] > 0.0f ? fmaxf(most[0] * (1.0f / kE4m3Max), 1.17549435e-38f) : 1.0f;
    const bool broken = most[0] > 3.4028235e38f;
    const float inverse = broken ? 0.0f : 1.0f / scale;
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
        const int64_t at = me.at(c);
        float q[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) q[i] = broken ? 0.0f : fminf(fmaxf(s[c][i] * inverse, -kE4m3Max), kE4m3Max);
        write8_e4m3(static_cast<uint8_t*>(a.output) + row * a.cols + at, there ? a.cols - at : 0, q);
    }
    if (there && me.lane == 0) a.scales[row] = broken ? __builtin_nanf("") : scale;
}

// The columns' sums of a workgroup's rows: over the lanes of a wavefront that stand at
// the same columns, then over the wavefronts, into the workgroup's row of `parts`.
template <int kLanes, int kChunks>
__device__ inline void sum_columns(float (&w)[kChunks][8], float* parts, int64_t cols) {
    constexpr int kWaves = kThreads / 64;
    const Lane<kLanes> me;
    if constexpr (kLanes < 64) {
#pragma unroll
        for (int step = kLanes; step < 64; step <<= 1) {
#pragma unroll
            for (int c = 0; c < kChunks; ++c) {
#pragma unroll
                for (int i = 0; i < 8; ++i) w[c][i] += __shfl_xor(w[c][i], step);
            }
        }
    }
    if constexpr (kLanes <= 64) {
        constexpr int kWidth = kLanes * kChunks * 8;
        __shared__ float space[kWaves][kWidth];
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
        __syncthreads();
        if (lane < kLanes) {
#pragma unroll
            for (int c = 0; c < kChunks; ++c) {
#pragma unroll
                for (int i = 0; i < 8; ++i) space[wave][me.at(c) + i] = w[c][i];
            }
        }
        __syncthreads();
        for (int i = threadIdx.x; i < kWidth; i += kThreads) {
            if (i < cols) parts[blockIdx.x * cols + i] = space[0][i] + space[1][i] + space[2][i] + space[3][i];
        }
    } else {
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
            const int64_t at = me.at(c);
            write8(parts + blockIdx.x * cols + at, cols - at, w[c]);
        }
    }
}

template <typename T, int kLanes, int kChunks>
__global__ __launch_bounds__(kThreads) void norm_backward_kernel(const NormDev d) {
    const Lane<kLanes> me;
    const ash_norm_args& a = d.a;
    __shared__ float space[kThreads / 64][2];
    constexpr int kRows = Lane<kLanes>::kRows;
    float w[kChunks][8], gw[kChunks][8];
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            w[c][i] = 1.0f;
            gw[c][i] = 0.0f;
        }
        if (a.weight != nullptr) read8(static_cast<const T*>(a.weight) + me.at(c), a.cols - me.at(c), w[c]);
    }
    for (int64_t row0 = static_cast<int64_t>(blockIdx.x) * kRows; row0 < a.rows;
         row0 += static_cast<int64_t>(gridDim.x) * kRows) {
        const int64_t row = row0 + me.row;
        const bool there = row < a.rows;
        float s[kChunks][8], g[kChunks][8];
        float sums[2] = {0.0f, 0.0f};   // s . s, s . (g w)
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
            const int64_t at = me.at(c), left = there ? a.cols - at : 0;
            read8(static_cast<const T*>(a.input) + row * a.input_stride + at, left, s[c]);
            read8(static_cast<const T*>(a.grad) + row * a.cols + at, left, g[c]);
        }
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                sums[0] += s[c][i] * s[c][i];
                sums[1] += s[c][i] * (g[c][i] * w[c][i]);
            }
        }
        join<kLanes, Sum>(sums, space);
        const float inverse = 1.0f / sqrtf(sums[0] * d.inverse_cols + a.eps);
        const float along = inverse * inverse * inverse * sums[1] * d.inverse_cols;
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
            const int64_t at = me.at(c), left = there ? a.cols - at : 0;
            float out[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
            if (a.grad_sum != nullptr) read8(static_cast<const T*>(a.grad_sum) + row * a.cols + at, left, out);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                gw[c][i] += g[c][i] * s[c][i] * inverse;
                out[i] += inverse * g[c][i] * w[c][i] - along * s[c][i];
            }
            if (a.output != nullptr) write8(static_cast<T*>(a.output) + row * a.cols + at, left, out);
        }
    }
    if (a.parts != nullptr) sum_columns<kLanes, kChunks>(gw, a.parts, a.cols);
}

// Second order: u of the gradient of s (a.second), v of the gradient of the weight
// (a.second_weight).  With t = g w and the row's sums a = u.t, b = u.s, c = t.s,
// e = (g v).s, q = s.s, and n values a row:
//   of g       w (i u - i^3 s b / n) + i s v
//   of weight  sum over rows of g (i u - i^3 s b / n)
//   of s       -i^3 (s a + t b + u c) / n + 3 i^5 s b c / n^2 + i g v - i^3 s e / n
template <typename T, int kLanes, int kChunks>
__global__ __launch_bounds__(kThreads) void norm_second_kernel(const NormDev d) {
    const Lane<kLanes> me;
    const ash_norm_args& a = d.a;
    __shared__ float space[kThreads / 64][5];
    constexpr int kRows = Lane<kLanes>::kRows;
    float gw[kChunks][8];
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
#pragma unroll
        for (int i = 0; i < 8; ++i) gw[c][i] = 0.0f;
    }
    for (int64_t row0 = static_cast<int64_t>(blockIdx.x) * kRows; row0 < a.rows;
         row0 += static_cast<int64_t>(gridDim.x) * kRows) {
        const int64_t row = row0 + me.row;
        const bool there = row < a.rows;
        float s[kChunks][8], g[kChunks][8], u[kChunks][8];
        float sums[5] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
            const int64_t at = me.at(c), left = there ? a.cols - at : 0;
            read8(static_cast<const T*>(a.input) + row * a.input_stride + at, left, s[c]);
            read8(static_cast<const T*>(a.grad) + row * a.cols + at, left, g[c]);
            read8(static_cast<const T*>(a.second) + row * a.cols + at, a.second != nullptr ? left : 0, u[c]);
            float w[8] = {1.0f, 1.0f, 1.0f, 1.0f, 1.0f, 1.0f, 1.0f, 1.0f}, v[8];
            if (a.weight != nullptr) read8(static_cast<const T*>(a.weight) + at, left, w);
            read8(static_cast<const T*>(a.second_weight) + at, a.second_weight != nullptr ? left : 0, v);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float t = g[c][i] * w[i];
                sums[0] += s[c][i] * s[c][i];
                sums[1] += u[c][i] * t;
                sums[2] += u[c][i] * s[c][i];
                sums[3] += t * s[c][i];
                sums[4] += g[c][i] * v[i] * s[c][i];
            }
        }
        join<kLanes, Sum>(sums, space);
        const float i1 = 1.0f / sqrtf(sums[0] * d.inverse_cols + a.eps), i3 = i1 * i1 * i1;
        const float per = i3 * d.inverse_cols;
        const float of_s = -per * (sums[1] + sums[4]) +
                           3.0f * i3 * i1 * i1 * sums[2] * sums[3] * d.inverse_cols * d.inverse_cols;
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
            const int64_t at = me.at(c), left = there ? a.cols - at : 0;
            float w[8] = {1.0f, 1.0f, 1.0f, 1.0f, 1.0f, 1.0f, 1.0f, 1.0f}, v[8], of_g[8], out[8];
            if (a.weight != nullptr) read8(static_cast<const T*>(a.weight) + at, left, w);
            read8(static_cast<const T*>(a.second_weight) + at, a.second_weight != nullptr ? left : 0, v);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float p = i1 * u[c][i] - per * sums[2] * s[c][i];
                of_g[i] = w[i] * p + i1 * s[c][i] * v[i];
                gw[c][i] += g[c][i] * p;
                out[i] = of_s * s[c][i] - per * (g[c][i] * w[i] * sums[2] + u[c][i] * sums[3]) + i1 * g[c][i] * v[i];
            }
            if (a.output != nullptr) write8(static_cast<T*>(a.output) + row * a.cols + at, left, out);
            if (a.grad_out != nullptr) write8(static_cast<T*>(a.grad_out) + row * a.cols + at, left, of_g);
        }
    }
    if (a.parts != nullptr) sum_columns<kLanes, kChunks>(gw, a.parts, a.cols);
}

// Joins the workgroups' column sums, in their order: 32 columns a workgroup, eight
// threads each.
constexpr int kJoin = 32;
template <typename T>
__global__ __launch_bounds__(kThreads) void join_columns_kernel(const float* parts, int64_t cols, int64_t n, T* out) {
    constexpr int kGroups = kThreads / kJoin;
    __shared__ float sums[kGroups][kJoin];
    const int64_t at = static_cast<int64_t>(blockIdx.x) * kJoin + threadIdx.x % kJoin;
    const int group = threadIdx.x / kJoin;
    float sum = 0.0f;
    if (at < cols) {
        const int64_t each = (n + kGroups - 1) / kGroups;
        const int64_t to = (group + 1) * each < n ? (group + 1) * each : n;
#pragma unroll 8
        for (int64_t part = group * each; part < to; ++part) sum += parts[part * cols + at];
    }
    sums[group][threadIdx.x % kJoin] = sum;
    __syncthreads();
    if (group != 0 || at >= cols) return;
#pragma unroll
    for (int i = 1; i < kGroups; ++i) sum += sums[i][threadIdx.x % kJoin];
    out[at] = static_cast<T>(sum);
}

constexpr int64_t kMaxColumns = 16384;
constexpr int kMaxParts = 1024;   // workgroups of the gradients: four a CU

int lanes_of(int64_t cols) {
    int lanes = 4;
    while (lanes < 64 && lanes * 8 < cols) lanes *= 2;
    return cols > 64 * 8 * 4 ? kThreads : lanes;
}

int64_t parts_of(int64_t rows, int64_t cols) {
    const int64_t each = kThreads / lanes_of(cols), groups = (rows + each - 1) / each;
    return groups < kMaxParts ? groups : kMaxParts;
}

enum NormKind { kNormForward, kNormBackward, kNormSecond };

template <typename T, int kLanes, int kChunks>
int launch_norm(NormKind kind, NormDev d, hipStream_t s) {
    if (kind == kNormForward) {
        constexpr int64_t kEach = kThreads / kLanes;
        for (; d.first < d.a.rows; d.first += kMaxGroups * kEach) {
            const int64_t groups = (d.a.rows - d.first + kEach - 1) / kEach;
            norm_forward_kernel<T, kLanes, kChunks>
                    <<<static_cast<unsigned>(groups < kMaxGroups ? groups : kMaxGroups), kThreads, 0, s>>>(d);
            ASH_LAUNCH_CHECK();
        }
        return 0;
    } else {
        const unsigned grid = static_cast<unsigned>(parts_of(d.a.rows, d.a.cols));
        if (kind == kNormBackward) norm_backward_kernel<T, kLanes, kChunks><<<grid, kThreads, 0, s>>>(d);
        else norm_second_kernel<T, kLanes, kChunks><<<grid, kThreads, 0, s>>>(d);
    }
    ASH_LAUNCH_CHECK();
    return 0;
}

template <typename T>
int norm_of(NormKind kind, const NormDev& d, hipStream_t s) {
    const int64_t cols = d.a.cols;
    if (d.a.rows > 0) {
        int status;
        switch (lanes_of(cols)) {
            case 4: status = launch_norm<T, 4, 1>(kind, d, s); break;
            case 8: status = launch_norm<T, 8, 1>(kind, d, s); break;
            case 16: status = launch_norm<T, 16, 1>(kind, d, s); break;
            case 32: status = launch_norm<T, 32, 1>(kind, d, s); break;
            case 64:
                if (cols <= 512) status = launch_norm<T, 64, 1>(kind, d, s);
                else if (cols <= 1024) status = launch_norm<T, 64, 2>(kind, d, s);
                else status = launch_norm<T, 64, 4>(kind, d, s);
                break;
            default:
                if (cols <= 4096) status = launch_norm<T, 256, 2>(kind, d, s);
                else if (cols <= 8192) status = launch_norm<T, 256, 4>(kind, d, s);
                else status = launch_norm<T, 256, 8>(kind, d, s);
        }
        if (status != 0) return status;
    }
    if (kind != kNormForward && d.a.weight_out != nullptr) {
        join_columns_kernel<T><<<static_cast<unsigned>((cols + kJoin - 1) / kJoin), kThreads, 0, s>>>(
                d.a.parts, cols, d.a.rows > 0 ? parts_of(d.a.rows, cols) : 0, static_cast<T*>(d.a.weight_out));
        ASH_LAUNCH_CHECK();
    }
    return 0;
}

int run_norm(NormKind kind, const ash_norm_args* args, void* stream, const char* what) {
    if (args == nullptr) ASH_FAIL(std::string("null pointer in ") + what);
    const ash_norm_args& a = *args;
    if (a.rows < 0 || a.rows > 0x7FFFFFFFll || a.cols < 1 || a.cols > kMaxColumns) {
        ASH_FAIL(std::string(what) + " takes up to 2^31 - 1 rows of 1 to 16384 values");
    }
    if (a.dtype != ASH_F32 && a.dtype != ASH_BF16 && a.dtype != ASH_F16) {
        ASH_FAIL(std::string(what) + ": float32, bfloat16 or float16 values");
    }
    if (a.rows > 0 && (a.input == nullptr || (kind == kNormForward && a.output == nullptr) ||
                       (kind != kNormForward && a.grad == nullptr))) {
        ASH_FAIL(std::string("null pointer in ") + what);
    }
    if (kind != kNormForward && a.weight_out != nullptr && a.parts == nullptr) {
        ASH_FAIL(std::string(what) + ": the weight's gradient needs scratch");
    }
    if ((a.rows > 1 && a.input_stride < 0) || a.residual_stride < 0) ASH_FAIL(std::string(what) + ": bad strides");
    PointerGuard guard;
    ASH_HIP(guard.enter_for(a.rows > 0 ? a.input : a.weight_out));
    const NormDev d = {a, 1.0f / static_cast<float>(a.cols), 0};
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (a.dtype == ASH_F32) return norm_of<float>(kind, d, s);
    if (a.dtype == ASH_BF16) return norm_of<__bf16>(kind, d, s);
    return norm_of<_Float16>(kind, d, s);
}

// ------------------------------------------------------------------- dense layers
constexpr int64_t kMaxFeatures = 65536;

// grad * slope, rounded to the operands' type as the products round it.
template <typename T, typename S>
__global__ __launch_bounds__(kThreads) void scale_kernel(const T* grad, const S* slope, float factor, T* out, int64_t n) {
    const int64_t at = (static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x) * 8;
    float g[8], d[8];
    read8(grad + at, n - at, g);
    read8(slope + at, n - at, d);
#pragma unroll
    for (int i = 0; i < 8; ++i) g[i] *= factor * d[i];
    write8(out + at, n - at, g);
}

template <typename T, typename S>
int launch_scale(const void* grad, const void* slope, float factor, void* out, int64_t n, hipStream_t s) {
    constexpr int64_t kMost = kMaxGroups * kThreads * 8;
    for (int64_t at = 0; at < n; at += kMost) {
        const int64_t left = n - at < kMost ? n - at : kMost;
        scale_kernel<<<static_cast<unsigned>((left + kThreads * 8 - 1) / (kThreads * 8)), kThreads, 0, s>>>(
                static_cast<const T*>(grad) + at, static_cast<const S*>(slope) + at, factor, static_cast<T*>(out) + at, left);
        ASH_LAUNCH_CHECK();
    }
    return 0;
}

int run_linear(LinearKind kind, const LinearJob& j, int32_t dtype, hipStream_t s) {
    switch (dtype) {
        case ASH_F32: return linear_run<ASH_F32>(kind, j, s);
        case ASH_BF16: return linear_run<ASH_BF16>(kind, j, s);
        case ASH_F16: return linear_run<ASH_F16>(kind, j, s);
        default: return linear_run<ASH_E4M3>(kind, j, s);
    }
}

int check_linear(const ash_linear_args* a, bool eight_bits, const char* what) {
    if (a == nullptr) ASH_FAIL(std::string("null pointer in ") + what);
    if (a->rows < 0 || a->rows > 0x7FFFFFFFll || a->in_features < 1 || a->in_features > kMaxFeatures ||
        a->out_features < 1 || a->out_features > kMaxFeatures) {
        ASH_FAIL(std::string(what) + " takes up to 2^31 - 1 rows, 1 to 65536 features in and out");
    }
    const bool floats = a->dtype == ASH_F32 || a->dtype == ASH_BF16 || a->dtype == ASH_F16;
    if (!floats && !(eight_bits && a->dtype == ASH_E4M3)) {
        ASH_FAIL(std::string(what) + ": float32, bfloat16 or float16 operands" + (eight_bits ? ", or e4m3" : ""));
    }
    if (floats ? a->out_dtype != a->dtype
               : a->out_dtype != ASH_F32 && a->out_dtype != ASH_BF16 && a->out_dtype != ASH_F16) {
        ASH_FAIL(std::string(what) + ": bad type of the output");
    }
    if (a->activation < ASH_ACT_NONE || a->activation > ASH_ACT_SINE) ASH_FAIL("linear: unknown activation");
    if (!(a->activation_scale > 0.0f) || a->activation_scale > 3.4028235e38f) {
        ASH_FAIL("linear: the activation's scale must be positive and finite");
    }
    if (a->slope_is_output && !ash_linear_slope_by_output(a->dtype, a->activation)) {
        ASH_FAIL(std::string(what) + ": the output does not tell the slope");
    }
    if (a->rows > 0 && (a->input == nullptr || a->weight == nullptr ||
                        (a->dtype == ASH_E4M3 && (a->input_scales == nullptr || a->weight_scales == nullptr)))) {
        ASH_FAIL(std::string("null pointer in ") + what);
    }
    if ((a->rows > 1 && a->input_stride < 0) || a->residual_stride < 0) ASH_FAIL(std::string(what) + ": bad strides");
    return 0;
}

LinearJob job_of(const ash_linear_args& a) {
    LinearJob j{};
    j.input = a.input;
    j.weight = a.weight;
    j.bias = a.bias;
    j.residual = a.residual;
    j.input_scales = a.input_scales;
    j.weight_scales = a.weight_scales;
    j.rows = a.rows;
    j.in = a.in_features;
    j.cols = a.out_features;
    j.input_stride = a.input_stride;
    j.residual_stride = a.residual_stride;
    j.out_dtype = a.out_dtype;
    j.activation = a.activation;
    j.act_scale = a.activation_scale;
    j.splits = 1;
    j.slope_factor = a.activation == ASH_ACT_SINE ? a.activation_scale : 1.0f;
    if (a.slope_is_output) {
        j.slope_kind = a.activation == ASH_ACT_RELU ? 1 : 2;
        if (a.activation == ASH_ACT_SOFTPLUS) j.slope_factor = a.activation_scale;
    }
    return j;
}

}  // namespace

// Enough workgroups for two a CU (one of the largest tiles, four of the smallest where their
// parts are not too many to join: 40 000 rows of 333 fp16 to 515 136 us for 161, of 67 to 129
// 29 for 26), parts of four steps of k at least.
int32_t linear_splits(int64_t rows, int64_t in, int64_t out, int32_t dtype, int pairs) {
    const WeightTile t = weight_tile(in, out, dtype);
    const int64_t tiles = ((out + t.rows - 1) / t.rows) * ((in + t.cols - 1) / t.cols) * pairs;
    const int64_t step = dtype == ASH_F32 ? 32 : 64, steps = (rows + step - 1) / step;
    const int64_t groups = t.rows == 256 ? 256 : t.rows == 64 && tiles > 4 ? 1024 : 512;
    const int64_t wanted = (groups + tiles - 1) / tiles, most = steps / 4 > 0 ? steps / 4 : 1;
    return static_cast<int32_t>(wanted < most ? wanted : most);
}

}  // namespace ash

using namespace ash;

extern "C" {

int ash_linear_forward(const ash_linear_args* args, void* output, void* slope, void* stream) {
    if (check_linear(args, true, "linear") != 0) return 1;
    if (args->rows == 0) return 0;
    if (output == nullptr) ASH_FAIL("null pointer in linear");
    if (slope != nullptr && args->dtype == ASH_E4M3) ASH_FAIL("linear: 8-bit rows have no gradients");
    LinearJob j = job_of(*args);
    j.out = output;
    j.slope_out = slope;
    PointerGuard guard;
    ASH_HIP(guard.enter_for(args->input));
    return run_linear(kLinearForward, j, args->dtype, static_cast<hipStream_t>(stream));
}

int ash_linear_backward_input(const ash_linear_args* args, const void* grad, const void* slope, const void* addend,
                              void* grad_input, void* stream) {
    if (check_linear(args, false, "linear_backward_input") != 0) return 1;
    if (args->rows == 0) return 0;
    if (grad == nullptr || grad_input == nullptr) ASH_FAIL("null pointer in linear_backward_input");
    LinearJob j = job_of(*args);
    j.bias = nullptr;
    j.grad = grad;
    j.slope = slope;
    j.residual = addend;
    j.residual_stride = args->in_features;
    j.activation = ASH_ACT_NONE;
    j.out = grad_input;
    PointerGuard guard;
    ASH_HIP(guard.enter_for(grad));
    return run_linear(kLinearGradInput, j, args->dtype, static_cast<hipStream_t>(stream));
}

int ash_linear_slope_by_output(int32_t dtype, int32_t activation) {
    return dtype == ASH_F32 && (activation == ASH_ACT_RELU || activation == ASH_ACT_SOFTPLUS);
}

// One pass more over the gradient, for two products of direct loads: 65 536 rows of 256 bf16
// to 256 21 + 44 us for 123, 4096 of 128 to 128 3 + 17 for 26.
int ash_linear_wants_scaled_gradient(int64_t rows, int64_t in_features, int64_t out_features, int32_t dtype) {
    return (dtype == ASH_BF16 || dtype == ASH_F16) && rows >= 512 &&
           weight_tile(in_features, out_features, dtype).cols >= 128;
}

int ash_linear_scale_gradient(const ash_linear_args* args, const void* grad, const void* slope, void* scaled,
                              void* stream) {
    if (check_linear(args, false, "linear_scale_gradient") != 0) return 1;
    if (args->rows == 0) return 0;
    if (grad == nullptr || slope == nullptr || scaled == nullptr) ASH_FAIL("null pointer in linear_scale_gradient");
    if (args->slope_is_output) ASH_FAIL("linear_scale_gradient takes slopes, not what tells them");
    const int64_t n = args->rows * args->out_features;
    const float factor = job_of(*args).slope_factor;
    PointerGuard guard;
    ASH_HIP(guard.enter_for(grad));
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (args->dtype == ASH_F32) return launch_scale<float, float>(grad, slope, factor, scaled, n, s);
    if (args->dtype == ASH_BF16) return launch_scale<__bf16, _Float16>(grad, slope, factor, scaled, n, s);
    return launch_scale<_Float16, float>(grad, slope, factor, scaled, n, s);
}

int64_t ash_linear_backward_weight_scratch_bytes(int64_t rows, int64_t in_features, int64_t out_features,
                                                 int32_t dtype, int pairs) {
    if (rows <= 0 || in_features < 1 || out_features < 1 || pairs < 1) return 0;
    const int64_t parts = static_cast<int64_t>(linear_splits(rows, in_features, out_features, dtype, pairs)) * pairs;
    return parts * (in_features * out_features + out_features) * 4;
}

int ash_linear_backward_weight(const ash_linear_args* args, const void* grad, const void* slope,
                               const void* second_grad, const void* second_slope, const void* second_input,
                               int64_t second_input_stride, int second_has_bias, void* grad_weight, void* grad_bias,
                               void* scratch, int64_t scratch_bytes, void* stream) {
    if (check_linear(args, false, "linear_backward_weight") != 0) return 1;
    const int pairs = second_grad != nullptr ? 2 : 1;
    if (grad_weight == nullptr && grad_bias == nullptr) return 0;
    if (args->rows > 0 && (grad == nullptr || (pairs == 2 && second_input == nullptr))) {
        ASH_FAIL("null pointer in linear_backward_weight");
    }
    if (second_input_stride < 0 || (second_has_bias && pairs == 1)) ASH_FAIL("linear_backward_weight: bad second pair");
    const int64_t bytes = ash_linear_backward_weight_scratch_bytes(args->rows, args->in_features, args->out_features,
                                                                   args->dtype, pairs);
    if (scratch_bytes < bytes || (bytes > 0 && scratch == nullptr)) {
        ASH_FAIL("linear_backward_weight: the scratch is too small");
    }
    LinearJob j = job_of(*args);
    j.grad = grad;
    j.slope = slope;
    j.second_grad = second_grad;
    j.second_slope = second_slope;
    j.second_factor = second_input;
    j.second_stride = second_input_stride;
    j.second_has_bias = second_has_bias != 0;
    j.weight_out = grad_weight;
    j.bias_out = grad_bias;
    j.scratch = scratch;
    j.splits = args->rows > 0 ? linear_splits(args->rows, args->in_features, args->out_features, args->dtype, pairs) : 1;
    PointerGuard guard;
    ASH_HIP(guard.enter_for(grad_weight != nullptr ? grad_weight : grad_bias));
    return run_linear(kLinearGradWeight, j, args->dtype, static_cast<hipStream_t>(stream));
}

int64_t ash_linear_backward_both_scratch_bytes(int64_t rows, int64_t in_features, int64_t out_features, int32_t dtype,
                                               int pairs) {
    if (rows <= 0 || in_features < 1 || out_features < 1 || in_features > kNarrowFeatures ||
        out_features > kNarrowFeatures || pairs < 1 || (dtype != ASH_F32 && dtype != ASH_BF16 && dtype != ASH_F16)) {
        return 0;
    }
    return narrow_backward_parts(rows, pairs) * (in_features * out_features + out_features) * 4;
}

int ash_linear_backward_both(const ash_linear_args* args, const void* grad, const void* slope, const void* second_grad,
                             const void* second_slope, const void* second_input, int64_t second_input_stride,
                             void* grad_input, void* grad_weight, void* grad_bias, void* scratch, int64_t scratch_bytes,
                             void* stream) {
    if (check_linear(args, false, "linear_backward_both") != 0) return 1;
    const int pairs = second_grad != nullptr ? 2 : 1;
    const int64_t bytes = ash_linear_backward_both_scratch_bytes(args->rows, args->in_features, args->out_features,
                                                                 args->dtype, pairs);
    if (bytes == 0) ASH_FAIL("linear_backward_both takes rows of up to 64 features in and out");
    if (grad == nullptr || grad_input == nullptr || grad_weight == nullptr || scratch == nullptr ||
        (pairs == 2 && second_input == nullptr) || second_input_stride < 0) {
        ASH_FAIL("null pointer in linear_backward_both");
    }
    if (scratch_bytes < bytes) ASH_FAIL("linear_backward_both: the scratch is too small");
    LinearJob j = job_of(*args);
    j.grad = grad;
    j.slope = slope;
    j.second_grad = second_grad;
    j.second_slope = second_slope;
    j.second_factor = second_input;
    j.second_stride = second_input_stride;
    j.out = grad_input;
    j.weight_out = grad_weight;
    j.bias_out = grad_bias;
    j.scratch = scratch;
    PointerGuard guard;
    ASH_HIP(guard.enter_for(grad));
    return run_linear(kLinearGradBoth, j, args->dtype, static_cast<hipStream_t>(stream));
}

int ash_linear_second(const ash_linear_args* args, const void* grad, const void* second_input,
                      int64_t second_input_stride, const void* addend, int64_t addend_stride, void* grad_grad,
                      void* curvature, void* stream) {
    if (check_linear(args, false, "linear_second") != 0) return 1;
    if (args->rows == 0) return 0;
    if (grad == nullptr || second_input_stride < 0 || addend_stride < 0 || (grad_grad == nullptr && curvature == nullptr)) {
        ASH_FAIL("null pointer in linear_second");
    }
    LinearJob j = job_of(*args);
    j.residual = nullptr;
    j.grad = grad;
    j.second_input = second_input;
    j.second_stride = second_input_stride;
    j.addend = addend;
    j.addend_stride = addend_stride;
    j.out = grad_grad;
    j.curvature_out = curvature;
    PointerGuard guard;
    ASH_HIP(guard.enter_for(args->input));
    return run_linear(kLinearSecond, j, args->dtype, static_cast<hipStream_t>(stream));
}

int ash_norm_forward(const ash_norm_args* args, void* stream) {
    return run_norm(kNormForward, args, stream, "rms_norm");
}

int64_t ash_norm_backward_scratch_bytes(int64_t rows, int64_t cols) {
    return rows <= 0 || cols < 1 || cols > kMaxColumns ? 0 : parts_of(rows, cols) * cols * 4;
}

int ash_norm_backward(const ash_norm_args* args, void* stream) {
    return run_norm(kNormBackward, args, stream, "rms_norm_backward");
}

int ash_norm_second(const ash_norm_args* args, void* stream) {
    return run_norm(kNormSecond, args, stream, "rms_norm_second");
}

}  // extern "C"
