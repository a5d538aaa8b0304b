// Dense layers: activation(x W^T + b) + residual, its gradients and theirs.
//
// Compiled once for every type of operands, -DASH_LINEAR_DTYPE=<ASH_F32 / ASH_BF16 /
// ASH_F16 / ASH_E4M3>, each into device code of its own, which the runtime loads where
// it is used.
//
// Everything is one product, out[r, c] = sum_k P[r, k] Q[c, k] (ash_linear.h).  A
// workgroup computes a tile of it.  Both operands pass through LDS as 16-byte chunks of
// consecutive k, whichever way they lie in memory, so that a lane's operand of a matrix
// instruction is one or two reads of 16 bytes: operands that lie across k are turned in
// registers, eight values of k at a time.  The next step's operands are on their way
// into registers while this step's are multiplied.
//
// Matrix instructions take Q as their first operand and P as their second, so that a
// lane holds four consecutive columns of a row of the result.
//
// float32 goes through the bf16 matrix units, which have sixteen times the rate of the
// float32 ones: a value is the sum of three bf16 numbers (8 bits each, 24 together), and
// of the nine products of two such sums six are formed; the other three are below 2^-24
// of the largest.  All sums are float32.  (An infinite operand gives NaN, for infinity
// times the second number of the other operand, which may be zero.)
#include "ash_linear.h"

#include <type_traits>

#ifndef ASH_LINEAR_DTYPE
#error "ASH_LINEAR_DTYPE: the type of operands to compile for"
#endif

namespace ash {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// 8-bit rows for the 8-bit units, and for the bf16 ones, which hold their values exactly.
// The 8-bit units add the products of eight consecutive k to the last bit that is 2^-13 of
// the largest of them (and those sums in float32): 2^-19 of the sum of magnitudes, or 2^-16
// of the result's, for rows of normal numbers.  An output of 16 bits is rounded to 2^-9 or
// 2^-12 and takes them; one of float32 takes the bf16 units, at half the rate.
struct E4M3 { uint8_t bits; };
struct WideE4M3 { uint8_t bits; };

template <int DTYPE> struct TypeOf;
template <> struct TypeOf<ASH_F32> { using T = float; };
template <> struct TypeOf<ASH_BF16> { using T = __bf16; };
template <> struct TypeOf<ASH_F16> { using T = _Float16; };
template <> struct TypeOf<ASH_E4M3> { using T = E4M3; };

// How a type goes through LDS and the matrix units.
template <typename T> struct Form {
    static constexpr bool kIsFloat = sizeof(T) == 4, kIsByte = std::is_same<T, E4M3>::value;
    static constexpr bool kScaled = sizeof(T) == 1;                 // rows have scales
    static constexpr int kParts = kIsFloat ? 3 : 1;                 // numbers a value is made of
    static constexpr int kStep = kIsFloat ? 32 : kIsByte ? 128 : 64;   // values of k a step
    static constexpr int kChunk = kIsByte ? 16 : 8;                 // values of k a chunk of 16 bytes
    static constexpr int kLane = kIsByte ? 32 : 8;                  // values of k a lane gives to one instruction
    static constexpr int kInner = kStep / (4 * kLane);              // instructions along k a step
    using Unit = std::conditional_t<kScaled, __bf16, T>;            // what two bytes of a chunk hold
    using Slope = std::conditional_t<std::is_same<T, __bf16>::value, _Float16, float>;   // see activate
};


// Byte at which chunk `c` of row `row` lies in a plane whose rows are RB bytes.  Chunks
// are exchanged within a line of 128 bytes such that eight lanes that read one chunk of
// eight consecutive rows meet eight different sets of banks, and so do eight lanes that
// write one chunk of rows four apart (operands that are turned).
template <int RB>
__device__ inline int place(int row, int c) {
    if constexpr (RB == 128) {
        const int f = ((row >> 2) & 1) | (((row ^ (row >> 3)) & 1) << 1) | ((((row >> 1) ^ (row >> 4)) & 1) << 2);
        return row * 128 + ((c ^ f) << 4);
    } else {
        static_assert(RB == 64, "");
        const int line = row >> 1;
        const int f = ((line >> 1) & 1) | (((line ^ (line >> 2)) & 1) << 1) | (((line >> 3) & 1) << 2);
        return line * 128 + (((((row & 1) << 2) | c) ^ f) << 4);
    }
}

// The same for rows of k of ROWS values of two bytes, such that the 32 lanes that are served
// together by a turning read (rows k to k + 3 and k + 8 to k + 11, 32 bytes of each) meet
// different banks of the 64.
template <int ROWS>
__device__ inline int stacked_place(int k, int c) {
    int f;
    if constexpr (ROWS >= 128) f = ((k & 3) << 1) | (k & 8);
    else if constexpr (ROWS == 64) f = (k & 2) | ((k & 8) >> 1);
    else f = (k & 8) >> 2;
    return k * ROWS * 2 + ((c ^ f) << 4);
}

template <typename T> __device__ inline float as_float(T v) { return static_cast<float>(v); }
template <> __device__ inline float as_float(WideE4M3 v) { return __builtin_amdgcn_cvt_f32_fp8(v.bits, 0); }

// N consecutive values from memory that need not be aligned to more than a value; those
// at `left` and beyond are zeros and not read.
template <typename T, int N>
struct Values {
    T v[N];
};
template <typename T, int N>
__device__ inline Values<T, N> read(const T* p, int64_t left) {
    Values<T, N> r;
    if (left >= N) {
        __builtin_memcpy(&r, p, sizeof(r));
    } else {
        __builtin_memset(&r, 0, sizeof(r));
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if (i < left) r.v[i] = p[i];
        }
    }
    return r;
}
template <typename T, int N> __device__ inline Values<T, N> read(const T* p) {
    Values<T, N> r;
    __builtin_memcpy(&r, p, sizeof(r));
    return r;
}

// ---------------------------------------------------------------- three bf16 numbers
struct Three {
    bf16x8 part[3];
};
__device__ inline Three split(const float (&v)[8]) {
    Three t;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const __bf16 h = static_cast<__bf16>(v[i]);
        const float rest = v[i] - static_cast<float>(h);
        const __bf16 m = static_cast<__bf16>(rest);
        t.part[0][i] = h;
        t.part[1][i] = m;
        t.part[2][i] = static_cast<__bf16>(rest - static_cast<float>(m));
    }
    return t;
}

// One operand as a kernel gets it.
struct Side {
    const void* p;
    const void* mul;    // of the same layout (in the type of slopes), or null
    int64_t stride;     // values between rows (lying along k) or between values of k
    int64_t rows;
    float factor;       // of mul
    int32_t kind;       // SlopeKind
};

template <typename T> __device__ inline uint4 packed(const float (&v)[8]) {
    Values<T, 8> r;
#pragma unroll
    for (int i = 0; i < 8; ++i) r.v[i] = static_cast<T>(v[i]);
    uint4 u;
    __builtin_memcpy(&u, &r, 16);
    return u;
}

// exp(x) by the unit's exp2.  FULL: the argument's product with log2(e) in two parts, of which
// the second, below a step of the first, is applied as a factor; without, the error is 2^-24
// of the argument, which results of 16 bits do not show.
template <bool FULL> __device__ inline float exp_of(float x) {
    const float t = x * 1.44269504f;
    if constexpr (!FULL) return __builtin_amdgcn_exp2f(t);
    const float rest = fmaf(x, 1.44269504f, -t) + x * 1.92596299e-8f;
    const float e = __builtin_amdgcn_exp2f(t);
    // (beyond the range of float the first part says all there is)
    return fabsf(rest) < 1.0f ? fmaf(e, rest * 0.69314718f, e) : e;
}

// f'(z) / factor by what was kept: itself, or (float32 alone) the output of an activation that
// tells it, without a residual: 0 or more of relu, log(1 + exp(a z)) / a of softplus, whose
// slope is 1 - exp(-a y).
enum SlopeKind { kSlopeKept, kSlopeRelu, kSlopeSoftplus };
template <typename T> __device__ inline float slope_of(float kept, int kind, float factor) {
    if constexpr (sizeof(T) == 4) {
        if (kind == kSlopeRelu) return kept > 0.0f ? 1.0f : 0.0f;
        if (kind == kSlopeSoftplus) {
            const float t = factor * kept;   // (the factor is a)
            // (the series leaves off 2^-24 of the value at 1/4, the difference 2^-22)
            const float near = t * fmaf(t, fmaf(t, fmaf(t, fmaf(t, fmaf(t, -1.3888889e-3f, 8.3333333e-3f), -0.041666668f),
                                                        0.16666667f), -0.5f), 1.0f);
            return t < 0.25f ? near : 1.0f - exp_of<true>(-t);
        }
    }
    return factor * kept;
}

// Eight consecutive values of k of one row into LDS.
template <typename T, int ROWS>
__device__ inline void put(char* plane, int row, int chunk, const float (&v)[8]) {
    constexpr int RB = Form<T>::kStep / Form<T>::kChunk * 16;
    char* at = plane + place<RB>(row, chunk);
    if constexpr (Form<T>::kParts == 3) {
        const Three t = split(v);
#pragma unroll
        for (int part = 0; part < 3; ++part) {
            uint4 u;
            __builtin_memcpy(&u, &t.part[part], 16);
            *reinterpret_cast<uint4*>(at + part * ROWS * RB) = u;
        }
    } else {
        *reinterpret_cast<uint4*>(at) = packed<typename Form<T>::Unit>(v);
    }
}

// Operand that lies along k: row r at p + r * stride.
template <typename T, int ROWS, bool MUL, int THREADS>
struct Along {
    using M = typename Form<T>::Slope;
    static constexpr int kChunks = Form<T>::kStep / Form<T>::kChunk;
    static constexpr int kEach = (ROWS * kChunks + THREADS - 1) / THREADS;
    static constexpr int N = Form<T>::kChunk;
    static_assert(ROWS * kChunks % THREADS == 0 || kEach == 1, "");
    const T* p[kEach];
    const M* m[kEach];
    int row[kEach], chunk;
    bool mul;
    float factor;
    int kind;
    Values<T, N> v[kEach];
    Values<M, N> w[kEach];

    // kTwo: every other sixteen rows are rows of another operand of the same shape, zeros
    // where there is none (second order)
    template <bool kTwo>
    __device__ void start(const Side& a, int64_t row0, const void* other, int64_t other_stride) {
        chunk = threadIdx.x % kChunks;
        mul = MUL && a.mul != nullptr;
        factor = a.factor;
        kind = a.kind;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            row[i] = (threadIdx.x + i * THREADS) / kChunks;
            int r = row[i];
            const T* base = static_cast<const T*>(a.p);
            int64_t stride = a.stride;
            if (kTwo) {
                if (r & 16) {
                    base = static_cast<const T*>(other);
                    stride = other_stride;
                }
                r = r / 32 * 16 + r % 16;
            }
            const bool there = base != nullptr && row[i] < ROWS && row0 + r < a.rows;
            p[i] = there ? base + (row0 + r) * stride : nullptr;
            if constexpr (MUL) m[i] = there && mul ? static_cast<const M*>(a.mul) + (row0 + r) * stride : nullptr;
        }
    }
    __device__ void load(int64_t k0, int64_t k_end) {
        const int64_t k = k0 + chunk * N;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const int64_t left = p[i] != nullptr ? k_end - k : 0;
            v[i] = read<T, N>(p[i] + k, left);
            if constexpr (MUL) {
                if (mul) w[i] = read<M, N>(m[i] + k, left);
            }
        }
    }
    __device__ void store(char* plane) {
        constexpr int RB = kChunks * 16;
        if (ROWS * kChunks < THREADS && row[0] >= ROWS) return;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            if constexpr (Form<T>::kParts == 3 || MUL || (Form<T>::kScaled && !Form<T>::kIsByte)) {
                float f[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) f[j] = as_float(v[i].v[j]);
                if constexpr (MUL) {
                    if (mul) {
#pragma unroll
                        for (int j = 0; j < 8; ++j) f[j] *= slope_of<T>(as_float(w[i].v[j]), kind, factor);
                    }
                }
                put<T, ROWS>(plane, row[i], chunk, f);
            } else {
                uint4 u;
                __builtin_memcpy(&u, &v[i], 16);
                *reinterpret_cast<uint4*>(plane + place<RB>(row[i], chunk)) = u;
            }
        }
    }
};

// Operand that lies across k, float32: value k of row r at p[k * stride + r].  A thread
// takes eight values of k of kWide consecutive rows and turns them.
template <typename T, int ROWS, bool MUL, int THREADS>
struct Across {
    static constexpr int kGroups = Form<T>::kStep / 8;
    static constexpr int kWide = ROWS * kGroups >= THREADS ? ROWS * kGroups / THREADS : 1;
    static constexpr int kUnits = ROWS / kWide * kGroups;
    const T* p;
    const typename Form<T>::Slope* m;
    int64_t stride, left;   // rows from this thread's first to the last
    int row, group;
    bool mul, works;
    float factor;
    int kind;
    Values<T, kWide> v[8];
    Values<typename Form<T>::Slope, kWide> w[8];

    template <bool>
    __device__ void start(const Side& a, int64_t row0, const void*, int64_t) {
        row = threadIdx.x % (ROWS / kWide) * kWide;
        group = threadIdx.x / (ROWS / kWide);
        works = threadIdx.x < kUnits;
        stride = a.stride;
        left = works ? a.rows - (row0 + row) : 0;
        mul = MUL && a.mul != nullptr;
        p = static_cast<const T*>(a.p) + row0 + row;
        factor = a.factor;
        kind = a.kind;
        m = mul ? static_cast<const typename Form<T>::Slope*>(a.mul) + row0 + row : nullptr;
    }
    __device__ void load(int64_t k0, int64_t k_end) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int64_t k = k0 + group * 8 + j;
            const int64_t n = k < k_end ? left : 0;
            v[j] = read<T, kWide>(p + k * stride, n);
            if constexpr (MUL) {
                if (mul) w[j] = read<typename Form<T>::Slope, kWide>(m + k * stride, n);
            }
        }
    }
    __device__ void store(char* plane) {
        if (!works) return;
#pragma unroll
        for (int i = 0; i < kWide; ++i) {
            float f[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                f[j] = as_float(v[j].v[i]);
                if constexpr (MUL) {
                    if (mul) f[j] *= slope_of<T>(as_float(w[j].v[i]), kind, factor);
                }
            }
            put<T, ROWS>(plane, row + i, group, f);
        }
    }
};

// Operand that lies across k, two bytes a value: rows of k go into LDS as they are, and the
// reads turn them (fetch_stacked).
template <typename T, int ROWS, bool MUL, int THREADS>
struct Stacked {
    using M = typename Form<T>::Slope;
    static constexpr int kChunks = ROWS / 8;
    static constexpr int kEach = Form<T>::kStep * kChunks / THREADS;
    static_assert(Form<T>::kStep * kChunks % THREADS == 0, "");
    const T* p;
    const M* m;
    int64_t stride, left;
    int chunk;
    bool mul;
    float factor;
    int kind;
    Values<T, 8> v[kEach];
    Values<M, 8> w[kEach];

    template <bool>
    __device__ void start(const Side& a, int64_t row0, const void*, int64_t) {
        chunk = threadIdx.x % kChunks;
        stride = a.stride;
        left = a.rows - (row0 + chunk * 8);
        mul = MUL && a.mul != nullptr;
        factor = a.factor;
        kind = a.kind;
        p = static_cast<const T*>(a.p) + row0 + chunk * 8;
        m = mul ? static_cast<const M*>(a.mul) + row0 + chunk * 8 : nullptr;
    }
    __device__ int row(int i) const { return (threadIdx.x + i * THREADS) / kChunks; }
    __device__ void load(int64_t k0, int64_t k_end) {
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const int64_t k = k0 + row(i);
            const int64_t n = k < k_end ? left : 0;
            v[i] = read<T, 8>(p + k * stride, n);
            if constexpr (MUL) {
                if (mul) w[i] = read<M, 8>(m + k * stride, n);
            }
        }
    }
    __device__ void store(char* plane) {
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            uint4 u;
            __builtin_memcpy(&u, &v[i], 16);
            if constexpr (MUL) {
                if (mul) {
                    float f[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) f[j] = as_float(v[i].v[j]) * slope_of<T>(as_float(w[i].v[j]), kind, factor);
                    u = packed<T>(f);
                }
            }
            *reinterpret_cast<uint4*>(plane + stacked_place<ROWS>(row(i), chunk)) = u;
        }
    }
};

// ------------------------------------------------------------------------ operands
// A lane's share of 16 rows of an operand: of row lane % 16 the chunk(s) lane / 16.
template <typename T> struct Fragment;
template <> struct Fragment<__bf16> { bf16x8 v; };
template <> struct Fragment<_Float16> { f16x8 v; };
template <> struct Fragment<float> { bf16x8 v[3]; };
template <> struct Fragment<E4M3> { i32x8 v; };
template <> struct Fragment<WideE4M3> { bf16x8 v; };

template <typename T, int ROWS>
__device__ inline Fragment<T> fetch(const char* plane, int row0, int inner) {
    constexpr int RB = Form<T>::kStep / Form<T>::kChunk * 16;
    const int lane = threadIdx.x & 63, row = row0 + (lane & 15), g = lane >> 4;
    Fragment<T> f;
    if constexpr (Form<T>::kParts == 3) {
#pragma unroll
        for (int part = 0; part < 3; ++part) {
            __builtin_memcpy(&f.v[part], plane + part * ROWS * RB + place<RB>(row, g), 16);
        }
    } else if constexpr (Form<T>::kIsByte) {
        uint4 half[2];
        half[0] = *reinterpret_cast<const uint4*>(plane + place<RB>(row, 2 * g));
        half[1] = *reinterpret_cast<const uint4*>(plane + place<RB>(row, 2 * g + 1));
        __builtin_memcpy(&f.v, half, 32);
    } else {
        __builtin_memcpy(&f.v, plane + place<RB>(row, inner * 4 + g), 16);
    }
    return f;
}

typedef short i16x4 __attribute__((ext_vector_type(4)));
// Of an operand whose rows of k are stacked: a read of four rows of k by sixteen lanes gives
// lane i the four values of column i.
template <typename T, int ROWS>
__device__ inline Fragment<T> fetch_stacked(char* plane, int row0, int inner) {
    const int lane = threadIdx.x & 63, i = lane & 15;
    const int k = inner * 32 + (lane >> 4) * 8 + (i >> 2), row = row0 + (i & 3) * 4;
    char* at = plane + stacked_place<ROWS>(k, row >> 3) + (row & 7) * 2;
    i16x4 half[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        half[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (__attribute__((address_space(3))) i16x4*)(at + h * 4 * ROWS * 2));
    }
    Fragment<T> f;
    __builtin_memcpy(&f.v, half, 16);
    return f;
}

__device__ inline f32x4 mma(const Fragment<__bf16>& q, const Fragment<__bf16>& p, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(q.v, p.v, c, 0, 0, 0);
}
__device__ inline f32x4 mma(const Fragment<_Float16>& q, const Fragment<_Float16>& p, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(q.v, p.v, c, 0, 0, 0);
}
__device__ inline f32x4 mma(const Fragment<float>& q, const Fragment<float>& p, f32x4 c) {
    // the smallest products first
    c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(q.v[0], p.v[2], c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(q.v[2], p.v[0], c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(q.v[1], p.v[1], c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(q.v[0], p.v[1], c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(q.v[1], p.v[0], c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(q.v[0], p.v[0], c, 0, 0, 0);
}
__device__ inline f32x4 mma(const Fragment<WideE4M3>& q, const Fragment<WideE4M3>& p, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(q.v, p.v, c, 0, 0, 0);
}
__device__ inline f32x4 mma(const Fragment<E4M3>& q, const Fragment<E4M3>& p, f32x4 c) {
    // block scales of one (2^(127 - 127)); the rows' own are applied to the sums
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(q.v, p.v, c, 0, 0, 0, 0x7F7F7F7F, 0, 0x7F7F7F7F);
}
// Row sums of P (every row of the result is the same): the bias' gradient.
__device__ inline f32x4 sum_rows(const Fragment<E4M3>&, f32x4 c) { return c; }   // 8-bit rows have none
__device__ inline f32x4 sum_rows(const Fragment<__bf16>& p, f32x4 c) {
    const bf16x8 one = {1.0f, 1.0f, 1.0f, 1.0f, 1.0f, 1.0f, 1.0f, 1.0f};
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(one, p.v, c, 0, 0, 0);
}
__device__ inline f32x4 sum_rows(const Fragment<_Float16>& p, f32x4 c) {
    const f16x8 one = {1.0f, 1.0f, 1.0f, 1.0f, 1.0f, 1.0f, 1.0f, 1.0f};
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(one, p.v, c, 0, 0, 0);
}
__device__ inline f32x4 sum_rows(const Fragment<float>& p, f32x4 c) {
#pragma unroll
    for (int part = 2; part >= 0; --part) c = sum_rows(Fragment<__bf16>{p.v[part]}, c);
    return c;
}

// --------------------------------------------------------------------- activations
template <bool FULL> __device__ inline float sigmoid(float v) { return __builtin_amdgcn_rcpf(1.0f + exp_of<FULL>(-v)); }

// The normal distribution's integral and its density at z, with e = exp(-z^2 / 2), x = |z| /
// sqrt(2).  FULL: the complementary error function is t exp(-x^2 + P(t)), t = 1 / (1 + x / 2),
// with the Chebyshev fit erfcc of Press et al., Numerical Recipes (1.2e-7 of the value,
// everywhere).  For results of 16 bits e t P(t), t = 1 / (1 + 0.46 x), P fitted to erfc(x)
// exp(x^2) / t such that the largest relative error is least, 2^-19.9 of the value everywhere:
// one exponential less (65 536 rows of 1024 bf16 to 1024 forward, of which the activation's
// arithmetic is a sixth: 183 us for 201).
template <bool FULL> __device__ inline void normal(float z, float& integral, float& density) {
    float e, tail;
    if constexpr (FULL) {
        const float x = fabsf(z) * 0.70710678f, t = __builtin_amdgcn_rcpf(fmaf(0.5f, x, 1.0f));
        float p = 0.17087277f;
        p = fmaf(p, t, -0.82215223f);
        p = fmaf(p, t, 1.48851587f);
        p = fmaf(p, t, -1.13520398f);
        p = fmaf(p, t, 0.27886807f);
        p = fmaf(p, t, -0.18628806f);
        p = fmaf(p, t, 0.09678418f);
        p = fmaf(p, t, 0.37409196f);
        p = fmaf(p, t, 1.00002368f);
        p = fmaf(p, t, -1.26551223f);
        e = exp_of<true>(-0.5f * z * z);
        tail = 0.5f * t * e * exp_of<true>(p);
    } else {
        const float t = __builtin_amdgcn_rcpf(fmaf(0.32526913f, fabsf(z), 1.0f));
        float p = 0.033857174f;   // P / 2
        p = fmaf(p, t, -0.11331463f);
        p = fmaf(p, t, 0.084595464f);
        p = fmaf(p, t, 0.02630535f);
        p = fmaf(p, t, 0.093423873f);
        p = fmaf(p, t, 0.11559094f);
        p = fmaf(p, t, 0.12977864f);
        p = fmaf(p, t, 0.12976353f);
        e = __builtin_amdgcn_exp2f(z * z * -0.72134752f);
        tail = e * t * p;
    }
    integral = z > 0.0f ? 1.0f - tail : tail;
    density = 0.39894228f * e;
}

// log(1 + e), e in [0, 1]
__device__ inline float log_of_one_and(float e) {
    const float u = 1.0f + e;
    const float far = fmaf(__builtin_amdgcn_logf(u), 0.69314718f, (e - (u - 1.0f)) * __builtin_amdgcn_rcpf(u));
    const float near = e * fmaf(e, fmaf(e, fmaf(e, fmaf(e, 0.2f, -0.25f), 0.33333333f), -0.5f), 1.0f);
    return e < 0.0625f ? near : far;
}

// Sine and cosine: the argument less multiples of pi / 2, by a constant in three parts (up
// to 2^17; in 64 bits beyond, good to 2^40), and the series up to r^9 and r^8.
__device__ inline void sine_cosine(float x, float& sine, float& cosine) {
    float k = rintf(x * 0.63661977f);
    float r = fmaf(k, -1.57079637f, x);
    r = fmaf(k, 4.37113900e-8f, r);
    r = fmaf(k, 1.71512489e-15f, r);
    int quarter = static_cast<int>(k);
    if (fabsf(x) > 131072.0f) {
        const double whole = rint(static_cast<double>(x) * 0.63661977236758134);
        r = static_cast<float>(fma(whole, -6.123233995736766e-17, fma(whole, -1.5707963267948966, static_cast<double>(x))));
        quarter = static_cast<int>(static_cast<int64_t>(whole));
    }
    const float q = r * r;
    const float s = fmaf(r * q, fmaf(q, fmaf(q, fmaf(q, 2.75573192e-6f, -1.98412698e-4f), 8.33333333e-3f), -0.16666667f), r);
    const float c = fmaf(q, fmaf(q, fmaf(q, fmaf(q, 2.48015873e-5f, -1.38888889e-3f), 4.16666667e-2f), -0.5f), 1.0f);
    sine = quarter & 1 ? c : s;
    cosine = quarter & 1 ? s : c;
    if (quarter & 2) sine = -sine;
    if ((quarter + 1) & 2) cosine = -cosine;
}

// Slopes that are kept for a backward pass are float32, for bf16 operands fp16: a rounding
// of them to the operands' type would be one more of the size of that of gz and of the
// result (half as much again in the gradients' error).  That of a sine is kept without the
// factor a, so that all fit fp16 (they are at most 1.13).
template <bool FULL, int N>
__device__ inline void activate(int kind, float a, const float (&z)[N], float (&y)[N], float (&d)[N]) {
    switch (kind) {
        case ASH_ACT_RELU:
#pragma unroll
            for (int i = 0; i < N; ++i) {
                y[i] = z[i] < 0.0f ? 0.0f : z[i];   // NaN stays NaN
                d[i] = z[i] > 0.0f ? 1.0f : 0.0f;
            }
            break;
        case ASH_ACT_SILU:
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float p = sigmoid<FULL>(z[i]);
                y[i] = z[i] * p;
                d[i] = p * fmaf(z[i], 1.0f - p, 1.0f);
            }
            break;
        case ASH_ACT_GELU:
#pragma unroll
            for (int i = 0; i < N; ++i) {
                float c, density;
                normal<FULL>(z[i], c, density);
                y[i] = z[i] * c;
                d[i] = fmaf(z[i], density, c);
            }
            break;
        case ASH_ACT_SOFTPLUS: {
            const float inverse = 1.0f / a;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float v = a * z[i], e = exp_of<FULL>(-fabsf(v)), r = __builtin_amdgcn_rcpf(1.0f + e);
                y[i] = fmaf(log_of_one_and(e), inverse, v < 0.0f ? 0.0f : z[i]);
                d[i] = v < 0.0f ? e * r : r;
            }
            break;
        }
        case ASH_ACT_SINE:
#pragma unroll
            for (int i = 0; i < N; ++i) sine_cosine(a * z[i], y[i], d[i]);
            break;
        default:
#pragma unroll
            for (int i = 0; i < N; ++i) {
                y[i] = z[i];
                d[i] = 1.0f;
            }
    }
}

// f'(z) (whole, of a sine too) and f''(z)
template <bool FULL, int N>
__device__ inline void curve(int kind, float a, const float (&z)[N], float (&d)[N], float (&dd)[N]) {
    switch (kind) {
        case ASH_ACT_SILU:
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float p = sigmoid<FULL>(z[i]);
                d[i] = p * fmaf(z[i], 1.0f - p, 1.0f);
                dd[i] = p * (1.0f - p) * fmaf(z[i], 1.0f - 2.0f * p, 2.0f);
            }
            break;
        case ASH_ACT_GELU:
#pragma unroll
            for (int i = 0; i < N; ++i) {
                float c, density;
                normal<FULL>(z[i], c, density);
                d[i] = fmaf(z[i], density, c);
                dd[i] = fmaf(-z[i], z[i], 2.0f) * density;
            }
            break;
        case ASH_ACT_SOFTPLUS:
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float v = a * z[i], e = exp_of<FULL>(-fabsf(v)), r = __builtin_amdgcn_rcpf(1.0f + e);
                d[i] = v < 0.0f ? e * r : r;
                dd[i] = a * e * r * r;
            }
            break;
        case ASH_ACT_SINE:
#pragma unroll
            for (int i = 0; i < N; ++i) {
                float s, c;
                sine_cosine(a * z[i], s, c);
                d[i] = a * c;
                dd[i] = -a * a * s;
            }
            break;
        case ASH_ACT_RELU:
#pragma unroll
            for (int i = 0; i < N; ++i) {
                d[i] = z[i] > 0.0f ? 1.0f : 0.0f;
                dd[i] = 0.0f;
            }
            break;
        default:
#pragma unroll
            for (int i = 0; i < N; ++i) {
                d[i] = 1.0f;
                dd[i] = 0.0f;
            }
    }
}

// --------------------------------------------------------------------- the product
struct Product {
    Side p, q;
    int64_t k;
    // weight's gradient: a second pair, the rows cut into parts
    Side p2, q2;
    int64_t part_rows;
    int32_t parts, pairs;
    bool second_has_bias;
    // second order: P's other operand
    const void* other;
    int64_t other_stride;
    int64_t row_tiles, col_tiles;
    LinearJob job;
};

// Whole pieces go past the caches: what is read of an output next is mostly more than they
// hold (16 384 rows of 4096 e4m3 to 4096 bf16 316 -> 278 us; of three layers of 64 to 64 in a
// row one takes 59.7 us for 60.7 of 524 288 rows float32, 10.7 for 11.5 of 131 072 bf16, 27 for
// 25 of 524 288 bf16, and as long as before of 16 384).
template <typename T, int N> __device__ inline void put_values(T* out, int64_t left, const float (&v)[N]) {
    typedef uint32_t Word __attribute__((ext_vector_type(N * sizeof(T) / 4), aligned(2)));
    Values<T, N> r;
#pragma unroll
    for (int i = 0; i < N; ++i) r.v[i] = static_cast<T>(v[i]);
    if (left >= N) {
        Word w;
        __builtin_memcpy(&w, &r, sizeof(r));
        __builtin_nontemporal_store(w, reinterpret_cast<Word*>(out));
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if (i < left) out[i] = r.v[i];
        }
    }
}

template <typename T, int N> __device__ inline void get_values(const T* in, int64_t left, float (&v)[N]) {
    const Values<T, N> r = read<T, N>(in, left);
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = as_float(r.v[i]);
}

// Workgroup -> tile.  Workgroups are dealt to the eight XCDs in turn, so those of one XCD
// take consecutive tiles; tiles go in bands of eight rows of tiles, down a band's rows
// first: the tiles that an XCD has under way at a time (64 of two a CU) then share eight
// row tiles and eight column tiles, which its L2 holds.
constexpr int kXcds = 8;
constexpr int kBand = 8;
__device__ inline bool tile_of(const Product& a, int64_t tiles, int64_t& tile) {
    const int64_t each = (tiles + kXcds - 1) / kXcds;
    tile = blockIdx.x % kXcds * each + blockIdx.x / kXcds;
    return blockIdx.x / kXcds < each && tile < tiles;
}
__device__ inline void banded(const Product& a, int64_t tile, int64_t& row, int64_t& col) {
    const int64_t band = tile / (kBand * a.col_tiles), in_band = tile % (kBand * a.col_tiles);
    const int64_t left = a.row_tiles - band * kBand, rows = left < kBand ? left : kBand;
    row = band * kBand + in_band % rows;
    col = in_band / rows;
}

// How a tile is shared out among wavefronts.
template <int BR, int BC>
struct Tile {
    static constexpr int kThreads = BR * BC >= 256 * 256 ? 512 : 256, kWaves = kThreads / 64;
    static constexpr int kWaveCols = BC >= 256 ? 4 : BC >= 128 ? 2 : BR >= 128 ? 1 : 2;
    static constexpr int kWaveRows = kWaves / kWaveCols;
    static constexpr int kR = BR / kWaveRows / 16, kC = BC / kWaveCols / 16;
    static constexpr int kSums = kR / kWaveCols;   // rows of P are summed by those that share them, so many of kR each
    static constexpr int kOutBytes = 16 * kC * 16 * 4;   // of sixteen rows of a wavefront's columns
};

template <typename T, int BR, int BC> struct Shared {
    static constexpr int kRowBytes = Form<T>::kStep / Form<T>::kChunk * 16;
    static constexpr int kP = Form<T>::kParts * BR * kRowBytes;
    static constexpr int kQ = Form<T>::kParts * BC * kRowBytes;
    static constexpr int kBytes = 2 * (kP + kQ);
};

// The way out of sixteen rows of a wavefront's sums (two sets of them for the second order).
// They go through LDS of the wavefront's own (16-byte pieces exchanged by the row's number, so
// that neither way meets a bank twice), after which a lane has the 16 bytes of a row next to
// those of its neighbours: operands and results come and go in whole lines, and no wavefront
// waits for another.  (Straight from the registers, where a lane has four columns of a row, or
// sixteen if the columns are dealt out for that, lines go in pieces: 524 288 rows of 64
// float32, with slopes, 200 us for 145 by way of LDS.)
template <typename TO, int KC, int KIND, bool SCALED>
struct Finish {
    using Slope = typename Form<TO>::Slope;
    static constexpr bool kTwo = KIND == kLinearSecond;
    static constexpr int N = 16 / sizeof(TO);                       // columns a lane
    static constexpr int kPieces = KC * 4, kLanes = KC * 16 / N, kDown = 64 / kLanes;
    static constexpr int kBytes = 16 * KC * 16 * 4;
    int lane, at;
    int64_t col, left;
    float bias[N], scale[N];

    // col0: of the wavefront
    __device__ void start(const Product& a, int64_t col0) {
        lane = threadIdx.x & 63;
        at = lane % kLanes * N;
        col = col0 + at;
        left = a.q.rows - col;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            bias[i] = 0.0f;
            scale[i] = 1.0f;
        }
        if (a.job.bias != nullptr) get_values(static_cast<const TO*>(a.job.bias) + col, left, bias);
        if constexpr (SCALED) get_values(a.job.weight_scales + col, left, scale);
    }
    __device__ void give(char* space, const f32x4 (&acc)[KC], int set = 0) const {
#pragma unroll
        for (int c = 0; c < KC; ++c) {
            const int piece = (c * 4 + (lane >> 4)) ^ (lane % 16 % kPieces);
            *reinterpret_cast<f32x4*>(space + set * kBytes + (lane % 16 * kPieces + piece) * 16) = acc[c];
        }
    }
    __device__ void take(const char* from, int r, float (&v)[N]) const {
#pragma unroll
        for (int h = 0; h < N / 4; ++h) {
            const int piece = (at / 4 + h) ^ (r % kPieces);
            __builtin_memcpy(v + 4 * h, from + (r * kPieces + piece) * 16, 16);
        }
    }
    // first_row: the same for a wavefront, so that a row's address is a scalar one and the
    // lane's offset from it
    // STAGED: the lane's 16 bytes of the residual lie at `staged` and every kilobyte from there
    template <bool STAGED = false>
    __device__ void rows(const Product& a, const char* space, int64_t first_row, const char* staged = nullptr) const {
        const LinearJob& j = a.job;
        const int r0 = lane / kLanes;
        const int32_t offset = r0 * static_cast<int32_t>(a.q.rows) + static_cast<int32_t>(col);
        const int64_t rows_left = a.p.rows - first_row;
        // (where there is nothing to compute, all at once: gradients of 524 288 rows of 64 float32
        // 132 -> 120 us)
#pragma unroll KIND == kLinearGradInput ? 4 : 1
        for (int i = 0; i < (16 + kDown - 1) / kDown; ++i) {
            const int r = r0 + i * kDown;
            if (r >= 16 || r >= rows_left || left <= 0) continue;
            const int64_t row = first_row + i * kDown, o = row * a.q.rows;   // (of lane 0)
            float z[N], y[N], d[N];
            take(space, r, z);
            const float row_scale = SCALED ? j.input_scales[row + r0] : 1.0f;
#pragma unroll
            for (int e = 0; e < N; ++e) {
                if constexpr (SCALED) z[e] *= row_scale * scale[e];
                z[e] += bias[e];
            }
            if constexpr (kTwo) {
                // t: the derivative of <second input, gradient of the input> by gz
                float t[N], g[N], dd[N];
                take(space + kBytes, r, t);
                if (j.addend != nullptr) {
                    get_values(static_cast<const TO*>(j.addend) + row * j.addend_stride + (r0 * j.addend_stride + col), left, g);
#pragma unroll
                    for (int e = 0; e < N; ++e) t[e] += g[e];
                }
                get_values(static_cast<const TO*>(j.grad) + o + offset, left, g);
                curve<sizeof(TO) == 4>(j.activation, j.act_scale, z, d, dd);
#pragma unroll
                for (int e = 0; e < N; ++e) {
                    y[e] = t[e] * d[e];
                    dd[e] *= t[e] * g[e];
                }
                if (j.out != nullptr) put_values(static_cast<TO*>(j.out) + o + offset, left, y);
                if (j.curvature_out != nullptr) {
                    put_values(static_cast<TO*>(j.curvature_out) + o + offset, left, dd);
                }
            } else {
                float more[N];
                if constexpr (STAGED) {
                    Values<TO, N> v;
                    __builtin_memcpy(&v, staged + i * 1024, 16);
#pragma unroll
                    for (int e = 0; e < N; ++e) more[e] = as_float(v.v[e]);
                } else if (j.residual != nullptr) {
                    get_values(static_cast<const TO*>(j.residual) + row * j.residual_stride + (r0 * j.residual_stride + col),
                               left, more);
                }
                if constexpr (KIND == kLinearGradInput) {
#pragma unroll
                    for (int e = 0; e < N; ++e) y[e] = z[e];
                } else {
                    activate<sizeof(TO) == 4>(j.activation, j.act_scale, z, y, d);
                    if (j.slope_out != nullptr) {
                        put_values(static_cast<Slope*>(j.slope_out) + o + offset, left, d);
                    }
                }
                if (STAGED || j.residual != nullptr) {
#pragma unroll
                    for (int e = 0; e < N; ++e) y[e] += more[e];
                }
                put_values(static_cast<TO*>(j.out) + o + offset, left, y);
            }
        }
    }
};

// The same of all of a wavefront's rows of a tile.
template <typename TO, int BR, int BC, int KIND, bool SCALED>
__device__ inline void finish(const Product& a, char* space, const f32x4 (&acc)[Tile<BR, BC>::kR][Tile<BR, BC>::kC],
                              int64_t row0, int64_t col0) {
    using W = Tile<BR, BC>;
    constexpr bool kTwo = KIND == kLinearSecond;
    constexpr int kTiles = kTwo ? W::kR / 2 : W::kR;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    Finish<TO, W::kC, KIND, SCALED> out;
    out.start(a, col0 + wave % W::kWaveCols * W::kC * 16);
    const int64_t first_row = row0 + wave / W::kWaveCols * kTiles * 16;
#pragma unroll 1
    for (int n = 0; n < kTiles; ++n) {
        // (accumulators are registers: which of them is said in the code, and the rest of it is
        // there once)
#pragma unroll
        for (int now = 0; now < kTiles; ++now) {
            if (now != n) continue;
            out.give(space, acc[kTwo ? 2 * now : now]);
            if constexpr (kTwo) out.give(space, acc[2 * now + 1], 1);
        }
        out.rows(a, space, first_row + n * 16);
    }
}

// A part's sums of a weight's gradient, in float32; join_kernel joins the parts.
template <int BR, int BC>
__device__ inline void leave_part(const Product& a, const f32x4 (&acc)[Tile<BR, BC>::kR][Tile<BR, BC>::kC],
                                  const f32x4 (&rows_sum)[Tile<BR, BC>::kSums], int64_t part, int64_t row0, int64_t col0,
                                  bool sums) {
    using W = Tile<BR, BC>;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wave_row = wave / W::kWaveCols * W::kR * 16, wave_col = wave % W::kWaveCols * W::kC * 16;
    float* out = static_cast<float*>(a.job.scratch) + part * (a.p.rows * a.q.rows + a.p.rows);
    float* bias = out + a.p.rows * a.q.rows;
#pragma unroll
    for (int r = 0; r < W::kR; ++r) {
        const int64_t row = row0 + wave_row + r * 16 + (lane & 15);
        if (row >= a.p.rows) continue;
#pragma unroll
        for (int c = 0; c < W::kC; ++c) {
            const int64_t col = col0 + wave_col + c * 16 + (lane >> 4) * 4;
            float* at = out + row * a.q.rows + col;
            if (col + 4 <= a.q.rows) {
                __builtin_memcpy(at, &acc[r][c], 16);
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (col + i < a.q.rows) at[i] = acc[r][c][i];
                }
            }
        }
        if (sums && r / W::kSums == wave % W::kWaveCols && lane < 16) bias[row] = rows_sum[r % W::kSums][0];
    }
}

// The tile of a workgroup: what it computes (of a weight's gradient, which part of k too).
struct Place {
    int64_t row_tile, col_tile, part, k0, k_end;
    bool second, sums;
};
template <int KIND> __device__ inline bool place_of(const Product& a, Place& w) {
    const int64_t tiles = a.row_tiles * a.col_tiles;
    int64_t tile;
    if (!tile_of(a, tiles * (KIND == kLinearGradWeight ? a.parts * a.pairs : 1), tile)) return false;
    w.part = 0;
    w.k0 = 0;
    w.k_end = a.k;
    w.second = w.sums = false;
    if constexpr (KIND == kLinearGradWeight) {
        w.part = tile / tiles;
        tile = tile % tiles;
        w.second = w.part >= a.parts;
        w.k0 = (w.second ? w.part - a.parts : w.part) * a.part_rows;
        w.k_end = w.k0 + a.part_rows < a.k ? w.k0 + a.part_rows : a.k;
        w.row_tile = tile % a.row_tiles;
        w.col_tile = tile / a.row_tiles;
        w.sums = a.job.bias_out != nullptr && w.col_tile == 0 && w.second == a.second_has_bias;
    } else {
        banded(a, tile, w.row_tile, w.col_tile);
    }
    return true;
}

template <typename T, typename TO, int BR, int BC, int KIND>
__global__ __launch_bounds__((Tile<BR, BC>::kThreads)) void product_kernel(const Product a) {
    using S = Shared<T, BR, BC>;
    using W = Tile<BR, BC>;
    constexpr int kThreads = W::kThreads;
    constexpr bool kGrad = KIND == kLinearGradInput || KIND == kLinearGradWeight;
    constexpr int kStep = Form<T>::kStep;
    __shared__ __attribute__((aligned(16))) char lds[S::kBytes];
    static_assert(W::kWaves * W::kOutBytes * (KIND == kLinearSecond ? 2 : 1) <= S::kBytes, "");

    Place w;
    if (!place_of<KIND>(a, w)) return;
    const int64_t k0 = w.k0, k_end = w.k_end;
    const int64_t row0 = w.row_tile * (KIND == kLinearSecond ? BR / 2 : BR), col0 = w.col_tile * BC;

    constexpr bool kStackP = KIND == kLinearGradWeight && sizeof(T) == 2, kStackQ = kGrad && sizeof(T) == 2;
    using LoadP = std::conditional_t<kStackP, Stacked<T, BR, true, kThreads>,
                                     std::conditional_t<KIND == kLinearGradWeight, Across<T, BR, true, kThreads>,
                                                        Along<T, BR, kGrad, kThreads>>>;
    using LoadQ = std::conditional_t<kStackQ, Stacked<T, BC, false, kThreads>,
                                     std::conditional_t<kGrad, Across<T, BC, false, kThreads>,
                                                        Along<T, BC, false, kThreads>>>;
    LoadP p;
    LoadQ q;
    p.template start<KIND == kLinearSecond>(w.second ? a.p2 : a.p, row0, a.other, a.other_stride);
    q.template start<false>(w.second ? a.q2 : a.q, col0, nullptr, 0);

    // (matrix instructions do not go by the mask of lanes: what they depend on has to be known
    // to be the same for a wavefront)
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wave_row = wave / W::kWaveCols * W::kR * 16, wave_col = wave % W::kWaveCols * W::kC * 16;
    f32x4 acc[W::kR][W::kC], rows_sum[W::kSums];
#pragma unroll
    for (int r = 0; r < W::kSums; ++r) rows_sum[r] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int r = 0; r < W::kR; ++r) {
#pragma unroll
        for (int c = 0; c < W::kC; ++c) acc[r][c] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }

    const int64_t steps = k_end > k0 ? (k_end - k0 + kStep - 1) / kStep : 0;
    if (steps > 0) {
        p.load(k0, k_end);
        q.load(k0, k_end);
        p.store(lds);
        q.store(lds + S::kP);
    }
    for (int64_t step = 0; step < steps; ++step) {
        const int64_t k = k0 + step * kStep;
        char* now = lds + (step & 1) * (S::kP + S::kQ);
        char* next = lds + (~step & 1) * (S::kP + S::kQ);
        if (step + 1 < steps) {
            p.load(k + kStep, k_end);
            q.load(k + kStep, k_end);
        }
        __syncthreads();   // this step's operands are there, and nobody reads the other half any more
#pragma unroll
        for (int inner = 0; inner < Form<T>::kInner; ++inner) {
            if (Form<T>::kInner > 1 && k + inner * (kStep / Form<T>::kInner) >= k_end) break;
            Fragment<T> fq[W::kC];
#pragma unroll
            for (int c = 0; c < W::kC; ++c) {
                if constexpr (kStackQ) fq[c] = fetch_stacked<T, BC>(now + S::kP, wave_col + c * 16, inner);
                else fq[c] = fetch<T, BC>(now + S::kP, wave_col + c * 16, inner);
            }
#pragma unroll
            for (int r = 0; r < W::kR; ++r) {
                Fragment<T> fp;
                if constexpr (kStackP) fp = fetch_stacked<T, BR>(now, wave_row + r * 16, inner);
                else fp = fetch<T, BR>(now, wave_row + r * 16, inner);
#pragma unroll
                for (int c = 0; c < W::kC; ++c) acc[r][c] = mma(fq[c], fp, acc[r][c]);
                if constexpr (KIND == kLinearGradWeight) {
                    if (w.sums && r / W::kSums == wave % W::kWaveCols) {
                        rows_sum[r % W::kSums] = sum_rows(fp, rows_sum[r % W::kSums]);
                    }
                }
            }
        }
        if (step + 1 < steps) {
            p.store(next);
            q.store(next + S::kP);
        }
    }

    if constexpr (KIND == kLinearGradWeight) {
        leave_part<BR, BC>(a, acc, rows_sum, w.part, row0, col0, w.sums);
    } else {
        __syncthreads();   // of all wavefronts' reads of their operands
        finish<TO, BR, BC, KIND, Form<T>::kScaled>(a, lds + wave * W::kOutBytes * (KIND == kLinearSecond ? 2 : 1), acc,
                                                   row0, col0);
    }
}

// Products of operands of one or two bytes whose pieces of 16 bytes are aligned: operands go
// from memory into LDS without passing through registers.  Of tiles of 256 x 256 a wavefront
// holds 128 x 64 sums (with 64 x 64 the reads from LDS take as long as the products).  The
// 16-byte pieces of a stage are fetched such that they land where Reader looks for them.
// Pieces past an operand's end, and past the last k, are outside of the buffer that the
// loads are told of, and come as zeros.
//
// bf16, fp16: four stages of 32 values of k, of which three are on their way while one is
// multiplied; e4m3, whose instructions take 128 values of k, two.  65 536 rows of 1024 bf16 to
// 1024 152 us (900 TFLOP/s), 16 384 of 4096 e4m3 to 4096, 16-bit outputs, 268 us (2050).
constexpr uint32_t kNowhere = 0x80000000u;   // beyond every such buffer

// SIZE: rows and columns of a tile, 256 or (where those would be too few) 128.
template <typename T, int SIZE> struct Stage {
    using W = Tile<SIZE, SIZE>;
    static constexpr int kRow = Form<T>::kIsByte ? 128 : 64;        // bytes of k
    static constexpr int kK = kRow / static_cast<int>(sizeof(T));   // values of k
    static constexpr int kStages = Form<T>::kIsByte ? 2 : 4;
    static constexpr int kEach = SIZE * kRow / 16 / W::kThreads;    // pieces a thread and operand
    static constexpr int kPlane = SIZE * kRow;
    // stacked: 128 bytes more for every eight rows of k, which puts the rows that a turning
    // read takes together on different banks
    static constexpr int kStacked = kPlane + kK / 8 * 128;
    // until all but the newest stages have come, and all reads from LDS (s_waitcnt: vmcnt in
    // bits 0-3 and 14-15, lgkmcnt in 8-11)
    static constexpr int kUnderWay = (kStages - 2) * 2 * kEach;
    static constexpr int kWait = 0x0070 | (kUnderWay & 15) | (kUnderWay >> 4 << 14);
};
constexpr int kWaitAll = 0x0070;

template <typename T, int SIZE, bool STACKED>
struct Direct {
    using S = Stage<T, SIZE>;
    static constexpr int kThreads = S::W::kThreads;
    const char* base;       // of the tile, at the first k
    uint32_t offset[S::kEach], stride;
    int k_of;               // first k of this thread's pieces along a row
    int64_t extent;         // bytes from base to the operand's end (of k_end)

    __device__ void start(const Side& a, int64_t row0, int64_t k0, int64_t k_end) {
        const int64_t rows = a.rows - row0 < SIZE ? a.rows - row0 : SIZE;
        stride = static_cast<uint32_t>(a.stride * sizeof(T));
        if constexpr (STACKED) {
            base = static_cast<const char*>(a.p) + (k0 * a.stride + row0) * sizeof(T);
            extent = ((k_end - k0 - 1) * a.stride + rows) * sizeof(T);
        } else {
            base = static_cast<const char*>(a.p) + (row0 * a.stride + k0) * sizeof(T);
            extent = ((rows - 1) * a.stride + (k_end - k0)) * sizeof(T);
        }
        k_of = 0;
#pragma unroll
        for (int i = 0; i < S::kEach; ++i) {
            const int piece = threadIdx.x + i * kThreads;
            if constexpr (STACKED) {
                constexpr int kPieces = SIZE / 8;
                const int k = piece / kPieces, c = piece % kPieces ^ ((k & 3) << 1);
                offset[i] = k * stride + c * 16;
            } else {
                constexpr int kPieces = S::kRow / 16;
                const int row = piece / kPieces, c = (piece ^ (kPieces == 8 ? row & 7 : (row >> 2) & 3)) % kPieces;
                k_of = c * Form<T>::kChunk;   // (the same for every i)
                offset[i] = row * stride + c * 16;
            }
        }
    }
    // `k`: from k0
    __device__ void issue(char* plane, int k, int k_left) {
        const int64_t past = STACKED ? static_cast<int64_t>(k) * stride : k * static_cast<int>(sizeof(T));
        const int64_t left = extent > past ? extent - past : 0;
        const auto buffer = __builtin_amdgcn_make_buffer_rsrc(
                const_cast<char*>(base + past), 0, static_cast<int>(left < 0x7FFFFFFF ? left : 0x7FFFFFFF), 0x00020000);
        const bool there = STACKED || k_of < k_left;
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
#pragma unroll
        for (int i = 0; i < S::kEach; ++i) {
            // a wavefront's pieces are consecutive (stacked: of whole rows of k, of one eight)
            const int first = wave * 64 + i * kThreads;
            char* at = plane + first * 16;
            if constexpr (STACKED) at += first / SIZE * 128;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(
                    buffer, (__attribute__((address_space(3))) void*)at, 16, there ? offset[i] : kNowhere, 0, 0, 0);
        }
    }
};

// Where a lane's pieces lie in a stage: addresses differ from one another by constants, or
// (stacked) go round in four, so that a wavefront keeps a few of them in registers.
template <typename T, int SIZE, bool STACKED>
struct Reader {
    static constexpr int kAt = STACKED ? 4 : Form<T>::kIsByte ? 2 : 1;
    const char* at[kAt];

    __device__ Reader(const char* plane, int row0) {
        const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
#pragma unroll
        for (int n = 0; n < kAt; ++n) {
            if constexpr (STACKED) {
                const int k = g * 8 + (i >> 2), c = ((row0 >> 3) + ((i & 3) >> 1)) ^ (((k & 3) ^ n) << 1);
                at[n] = plane + k * SIZE * 2 + g * 128 + (c << 4) + (i & 1) * 8;
            } else if constexpr (Form<T>::kIsByte) {
                at[n] = plane + (row0 + i) * 128 + (((2 * g + n) ^ (i & 7)) << 4);
            } else {
                at[n] = plane + (row0 + i) * 64 + ((g ^ (i >> 2)) << 4);
            }
        }
    }
    // rows 16 (4 QUAD) and on from row0: four fragments
    template <int QUAD>
    __device__ void get(Fragment<T> (&f)[4]) const {
        if constexpr (STACKED) {
            // The compiler takes a turning read to need whatever is on its way into LDS, and
            // would wait for the stages to come; so they are written out, with their wait.
            i16x4 part[8];
#if defined(__HIP_DEVICE_COMPILE__)
            uint32_t from[4];
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                from[n] = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(
                        (__attribute__((address_space(3))) const char*)at[n]));
            }
            asm volatile(
                    "ds_read_b64_tr_b16 %0, %8 offset:%12\n\t"
                    "ds_read_b64_tr_b16 %1, %8 offset:%13\n\t"
                    "ds_read_b64_tr_b16 %2, %9 offset:%12\n\t"
                    "ds_read_b64_tr_b16 %3, %9 offset:%13\n\t"
                    "ds_read_b64_tr_b16 %4, %10 offset:%12\n\t"
                    "ds_read_b64_tr_b16 %5, %10 offset:%13\n\t"
                    "ds_read_b64_tr_b16 %6, %11 offset:%12\n\t"
                    "ds_read_b64_tr_b16 %7, %11 offset:%13\n\t"
                    "s_waitcnt lgkmcnt(0)"
                    : "=&v"(part[0]), "=&v"(part[1]), "=&v"(part[2]), "=&v"(part[3]), "=&v"(part[4]), "=&v"(part[5]),
                      "=&v"(part[6]), "=&v"(part[7])
                    : "v"(from[0]), "v"(from[1]), "v"(from[2]), "v"(from[3]), "n"(QUAD * 128),
                      "n"(QUAD * 128 + 4 * SIZE * 2)
                    : "memory");
#endif
#pragma unroll
            for (int r = 0; r < 4; ++r) __builtin_memcpy(&f[r].v, part + 2 * r, 16);
        } else {
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                if constexpr (Form<T>::kIsByte) {
                    uint4 part[2];
#pragma unroll
                    for (int n = 0; n < 2; ++n) {
                        part[n] = *reinterpret_cast<const uint4*>(at[n] + (QUAD * 4 + r) * 2048);
                    }
                    __builtin_memcpy(&f[r].v, part, 32);
                } else {
                    __builtin_memcpy(&f[r].v, at[0] + (QUAD * 4 + r) * 1024, 16);
                }
            }
        }
    }
};

template <typename T, int SIZE, int QUAD, bool SUMS>
__device__ inline void multiply_quad(const Fragment<T> (&fq)[4], const Fragment<T> (&fp)[4],
                                     f32x4 (&acc)[Tile<SIZE, SIZE>::kR][4], f32x4 (&rows_sum)[Tile<SIZE, SIZE>::kSums],
                                     int wave) {
    using W = Tile<SIZE, SIZE>;
    static_assert(W::kC == 4 && W::kR % 4 == 0, "");
#pragma unroll
    for (int n = 0; n < 4; ++n) {
        const int r = QUAD * 4 + n;
#pragma unroll
        for (int c = 0; c < 4; ++c) acc[r][c] = mma(fq[c], fp[n], acc[r][c]);
        if constexpr (SUMS) {
            if (r / W::kSums == wave % W::kWaveCols) rows_sum[r % W::kSums] = sum_rows(fp[n], rows_sum[r % W::kSums]);
        }
    }
}

// What a wavefront has of a large tile, and what it does in a step.  SUMS: the sums of P's
// rows too (by the workgroups that are the first of a row of tiles).
template <typename T, int SIZE, bool STACK_P, bool STACK_Q>
struct LargeWork {
    using W = Tile<SIZE, SIZE>;
    using S = Stage<T, SIZE>;
    static constexpr int kP = STACK_P ? S::kStacked : S::kPlane, kQ = STACK_Q ? S::kStacked : S::kPlane;
    Direct<T, SIZE, STACK_P> p;
    Direct<T, SIZE, STACK_Q> q;
    int length, wave;
    f32x4 acc[W::kR][W::kC], rows_sum[W::kSums];

    __device__ void start(const Side& sp, const Side& sq, int64_t row0, int64_t col0, int64_t k0, int64_t k_end) {
        p.start(sp, row0, k0, k_end);
        q.start(sq, col0, k0, k_end);
        length = k_end > k0 ? static_cast<int>(k_end - k0) : 0;
        wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
#pragma unroll
        for (int r = 0; r < W::kSums; ++r) rows_sum[r] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int r = 0; r < W::kR; ++r) {
#pragma unroll
            for (int c = 0; c < W::kC; ++c) acc[r][c] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        }
    }
    struct Planes {
        char* p;
        char* q;
    };
    __device__ void issue(const Planes& to, int k) {
        p.issue(to.p, k, length - k);
        q.issue(to.q, k, length - k);
    }
    template <bool SUMS>
    __device__ void step(const Planes& stage, const Planes& next, int k_next) {
        // the stage's operands are there, and nobody reads the next to be filled any more
        // (__syncthreads would wait for the stages under way too)
        __builtin_amdgcn_s_waitcnt(S::kWait);
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        issue(next, k_next);
        const Reader<T, SIZE, STACK_P> rp(stage.p, wave / W::kWaveCols * W::kR * 16);
        const Reader<T, SIZE, STACK_Q> rq(stage.q, wave % W::kWaveCols * W::kC * 16);
        Fragment<T> fq[4], fp[4];
        rq.template get<0>(fq);
        rp.template get<0>(fp);
        multiply_quad<T, SIZE, 0, SUMS>(fq, fp, acc, rows_sum, wave);
        if constexpr (W::kR == 8) {
            rp.template get<1>(fp);
            multiply_quad<T, SIZE, 1, SUMS>(fq, fp, acc, rows_sum, wave);
        }
    }
    // All stages a turn; those past the end are of zeros (a way out between them costs a
    // second set of accumulators).
    template <bool SUMS>
    __device__ void run(const Planes& stage0, const Planes& stage1, const Planes& stage2, const Planes& stage3) {
        constexpr int kK = S::kK;
        if constexpr (S::kStages == 4) {
            issue(stage0, 0);
            issue(stage1, kK);
            issue(stage2, 2 * kK);
            for (int k = 0; k < length; k += 4 * kK) {
                step<SUMS>(stage0, stage3, k + 3 * kK);
                step<SUMS>(stage1, stage0, k + 4 * kK);
                step<SUMS>(stage2, stage1, k + 5 * kK);
                step<SUMS>(stage3, stage2, k + 6 * kK);
            }
        } else {
            issue(stage0, 0);
            for (int k = 0; k < length; k += 2 * kK) {
                step<SUMS>(stage0, stage1, k + kK);
                step<SUMS>(stage1, stage0, k + 2 * kK);
            }
        }
        __builtin_amdgcn_s_waitcnt(kWaitAll);   // nothing may land in LDS from here on
    }
};

// The way out with a residual, which comes by way of LDS (`staged`, 8 KB of the wavefront's
// own) sixty-four rows at a time: loads into registers between the stores would wait for
// those stores, sixteen times a tile (65 536 rows of 1024 bf16 to 1024, GELU, slopes and
// residual: 250 us for 276).
template <typename TO, int SIZE, bool SCALED>
__device__ inline void finish_staged(const Product& a, char* space, char* staged,
                                     const f32x4 (&acc)[Tile<SIZE, SIZE>::kR][Tile<SIZE, SIZE>::kC], int64_t row0,
                                     int64_t col0) {
    using W = Tile<SIZE, SIZE>;
    using Out = Finish<TO, W::kC, kLinearForward, SCALED>;
    static_assert(sizeof(TO) == 2 && Out::kDown == 8 && W::kR % 4 == 0, "a strip of sixteen rows is two kilobytes");
    const LinearJob& j = a.job;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int64_t first_col = col0 + wave % W::kWaveCols * W::kC * 16;
    const int64_t first_row = row0 + wave / W::kWaveCols * W::kR * 16;
    Out out;
    out.start(a, first_col);
    const uint32_t step = static_cast<uint32_t>(j.residual_stride) * 2;
    const char* base = static_cast<const char*>(j.residual) + (first_row * j.residual_stride + first_col) * 2;
    const auto buffer = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(base), 0, 0x7FFFFFFF, 0x00020000);
#pragma unroll 1
    for (int quad = 0; quad < W::kR / 4; ++quad) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int row = quad * 64 + i * 8 + lane / 8;
            const bool there = first_row + row < a.p.rows && out.left > 0;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(
                    buffer, (__attribute__((address_space(3))) void*)(staged + i * 1024), 16,
                    there ? row * step + lane % 8 * 16 : kNowhere, 0, 0, 0);
        }
        __builtin_amdgcn_s_waitcnt(kWaitAll);
        asm volatile("" ::: "memory");
#pragma unroll 1
        for (int n = 0; n < 4; ++n) {
#pragma unroll
            for (int now = 0; now < W::kR; ++now) {
                if (now == quad * 4 + n) out.give(space, acc[now]);
            }
            out.template rows<true>(a, space, first_row + (quad * 4 + n) * 16, staged + n * 2048 + lane * 16);
        }
        asm volatile("" ::: "memory");
    }
}

template <typename T, typename TO, int SIZE, int KIND>
__global__ __launch_bounds__((Tile<SIZE, SIZE>::kThreads), 2) void large_kernel(const Product a) {
    constexpr bool kStackP = KIND == kLinearGradWeight, kStackQ = KIND != kLinearForward;
    using Work = LargeWork<T, SIZE, kStackP, kStackQ>;
    using W = Tile<SIZE, SIZE>;
    constexpr int kHalf = W::kWaves / 2;
    static_assert(kHalf * W::kOutBytes <= Work::kP && kHalf * W::kOutBytes <= Work::kQ, "");
    constexpr bool kFour = Stage<T, SIZE>::kStages > 2;
    // Planes under names of their own: the compiler then sees that reads of one need not wait
    // for loads into another (it looks only so far through an address, hence one each).
    __shared__ __attribute__((aligned(16))) char p0[Work::kP], p1[Work::kP], p2[kFour ? Work::kP : 16], p3[kFour ? Work::kP : 16];
    __shared__ __attribute__((aligned(16))) char q0[Work::kQ], q1[Work::kQ], q2[kFour ? Work::kQ : 16],
            q3[kFour ? Work::kQ : 16];

    Place w;
    if (!place_of<KIND>(a, w)) return;
    const int64_t row0 = w.row_tile * SIZE, col0 = w.col_tile * SIZE;
    Work work;
    work.start(w.second ? a.p2 : a.p, w.second ? a.q2 : a.q, row0, col0, w.k0, w.k_end);
    if constexpr (KIND == kLinearGradWeight) {
        if (w.sums) work.template run<true>({p0, q0}, {p1, q1}, {p2, q2}, {p3, q3});
        else work.template run<false>({p0, q0}, {p1, q1}, {p2, q2}, {p3, q3});
        leave_part<SIZE, SIZE>(a, work.acc, work.rows_sum, w.part, row0, col0, w.sums);
    } else {
        work.template run<false>({p0, q0}, {p1, q1}, {p2, q2}, {p3, q3});
        __syncthreads();   // of all wavefronts' reads of their operands
        char* space = (work.wave < kHalf ? p0 : q0) + work.wave % kHalf * W::kOutBytes;
        if constexpr (KIND == kLinearForward && sizeof(TO) == 2) {
            const LinearJob& j = a.job;
            if (j.residual != nullptr && reinterpret_cast<uintptr_t>(j.residual) % 16 == 0 && j.residual_stride % 8 == 0 &&
                j.residual_stride < (1 << 21) && a.q.rows % 8 == 0) {
                constexpr int kEach = kFour ? W::kWaves / 4 : W::kWaves / 2;   // wavefronts a plane
                static_assert(kEach * 8192 <= Work::kP, "");
                const int of = work.wave / kEach;
                char* plane = kFour ? (of == 0 ? p1 : of == 1 ? p2 : of == 2 ? q1 : q2) : (of == 0 ? p1 : q1);
                finish_staged<TO, SIZE, Form<T>::kScaled>(a, space, plane + work.wave % kEach * 8192, work.acc, row0, col0);
                return;
            }
        }
        finish<TO, SIZE, SIZE, KIND, Form<T>::kScaled>(a, space, work.acc, row0, col0);
    }
}

// Few rows: 16 columns for RB times 16 rows a workgroup, whose eight wavefronts share out k
// and join their sums in LDS.  Operands go from memory straight into the matrix instructions:
// a value of the weight is read once and used for the workgroup's rows, so there is nothing
// to keep.  Sixteen rows are bound by the weight's bytes: of 4096 float32 to 4096 19.6 us
// (67 MB, 3.4 TB/s), in bf16 9.7, in e4m3 6.2; one row of 64 by the launch, 2.3 us.
constexpr int kFewThreads = 512;
constexpr int kFewWaves = kFewThreads / 64;

template <typename T> __device__ inline Fragment<T> formed(const Values<T, Form<T>::kLane>& v) {
    Fragment<T> f;
    if constexpr (Form<T>::kParts == 3) {
        const Three t = split(v.v);
#pragma unroll
        for (int part = 0; part < 3; ++part) f.v[part] = t.part[part];
    } else if constexpr (Form<T>::kScaled && !Form<T>::kIsByte) {
#pragma unroll
        for (int i = 0; i < 8; ++i) f.v[i] = static_cast<__bf16>(as_float(v.v[i]));
    } else {
        __builtin_memcpy(&f.v, &v, sizeof(f.v));
    }
    return f;
}

template <typename T, typename TO, int RB>
__global__ __launch_bounds__(kFewThreads) void few_rows_kernel(const Product a) {
    constexpr int kEach = Form<T>::kLane * 4;   // values of k a step
    constexpr int kAhead = RB == 1 ? 4 : 2;     // steps whose operands are on their way at a time
    __shared__ float sums[kFewWaves][RB * 16][20];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4;
    const int64_t col0 = static_cast<int64_t>(blockIdx.x) * 16, row0 = static_cast<int64_t>(blockIdx.y) * RB * 16;
    const int64_t row = row0 + (lane & 15), col = col0 + (lane & 15);
    // (what rows and columns beyond the last ones get is not written: they take the first's)
    const T* p[RB];
#pragma unroll
    for (int r = 0; r < RB; ++r) p[r] = static_cast<const T*>(a.p.p) + (row + r * 16 < a.p.rows ? row + r * 16 : 0) * a.p.stride;
    const T* q = static_cast<const T*>(a.q.p) + (col < a.q.rows ? col : 0) * a.q.stride;
    f32x4 acc[RB] = {};
    int64_t k0 = static_cast<int64_t>(wave) * kEach;
    for (; k0 + (kAhead - 1) * kFewWaves * kEach + kEach <= a.k; k0 += kAhead * kFewWaves * kEach) {
        Values<T, Form<T>::kLane> vp[kAhead][RB], vq[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const int64_t k = k0 + i * kFewWaves * kEach + g * Form<T>::kLane;
            vq[i] = read<T, Form<T>::kLane>(q + k);
#pragma unroll
            for (int r = 0; r < RB; ++r) vp[i][r] = read<T, Form<T>::kLane>(p[r] + k);
        }
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const Fragment<T> fq = formed<T>(vq[i]);
#pragma unroll
            for (int r = 0; r < RB; ++r) acc[r] = mma(fq, formed<T>(vp[i][r]), acc[r]);
        }
    }
    for (; k0 + kEach <= a.k; k0 += kFewWaves * kEach) {
        const int64_t k = k0 + g * Form<T>::kLane;
        const Values<T, Form<T>::kLane> vq = read<T, Form<T>::kLane>(q + k);
        Values<T, Form<T>::kLane> vp[RB];
#pragma unroll
        for (int r = 0; r < RB; ++r) vp[r] = read<T, Form<T>::kLane>(p[r] + k);
        const Fragment<T> fq = formed<T>(vq);
#pragma unroll
        for (int r = 0; r < RB; ++r) acc[r] = mma(fq, formed<T>(vp[r]), acc[r]);
    }
    if (k0 < a.k) {   // at most one step of one wavefront
        const int64_t k = k0 + g * Form<T>::kLane;
        const Fragment<T> fq = formed<T>(read<T, Form<T>::kLane>(q + k, a.k - k));
#pragma unroll
        for (int r = 0; r < RB; ++r) acc[r] = mma(fq, formed<T>(read<T, Form<T>::kLane>(p[r] + k, a.k - k)), acc[r]);
    }
#pragma unroll
    for (int r = 0; r < RB; ++r) *reinterpret_cast<f32x4*>(&sums[wave][r * 16 + (lane & 15)][g * 4]) = acc[r];
    __syncthreads();
    const LinearJob& j = a.job;
    for (int at = threadIdx.x; at < RB * 256; at += kFewThreads) {
        const int r = at >> 4, c = at & 15;
        const int64_t out_row = row0 + r, out_col = col0 + c;
        if (out_row >= a.p.rows || out_col >= a.q.rows) continue;
        float z[1] = {0.0f}, y[1], d[1];
#pragma unroll
        for (int i = 0; i < kFewWaves; ++i) z[0] += sums[i][r][c];
        if constexpr (Form<T>::kScaled) z[0] *= j.input_scales[out_row] * j.weight_scales[out_col];
        if (j.bias != nullptr) z[0] += as_float(static_cast<const TO*>(j.bias)[out_col]);
        activate<sizeof(TO) == 4>(j.activation, j.act_scale, z, y, d);
        if (j.residual != nullptr) y[0] += as_float(static_cast<const TO*>(j.residual)[out_row * j.residual_stride + out_col]);
        const int64_t o = out_row * a.q.rows + out_col;
        static_cast<TO*>(j.out)[o] = static_cast<TO>(y[0]);
        if (j.slope_out != nullptr) {
            using Slope = typename Form<TO>::Slope;
            static_cast<Slope*>(j.slope_out)[o] = static_cast<Slope>(d[0]);
        }
    }
}

// Narrow layers: the weight's fragments stay in registers, and every wavefront takes sixteen
// rows after sixteen rows through them, straight from memory (a lane's operand of an
// instruction is 16 or 32 consecutive bytes of a row; the next rows are on their way while
// these are multiplied).  No barriers, LDS only on the way out.  524 288 rows of 64 float32
// to 64 take 53 us without an activation (268 MB, 5.1 TB/s: bound by memory) and 73 with
// softplus, whose arithmetic (half of it transcendental or in twice the precision) adds to
// that at two wavefronts a SIMD; two steps of rows on their way instead of one: 79.
// KS: steps of k (4 kLane values each), KC: times sixteen columns.
constexpr int kNarrowThreads = 256;
template <typename T, typename TO, int KS, int KC, int KIND>
__global__ __launch_bounds__(kNarrowThreads, 2) void narrow_kernel(const Product a) {
    using Out = Finish<TO, KC, KIND, Form<T>::kScaled>;
    using M = typename Form<T>::Slope;
    constexpr int L = Form<T>::kLane;
    constexpr bool kGrad = KIND == kLinearGradInput, kTwo = KIND == kLinearSecond;
    constexpr int kSpace = Out::kBytes * (kTwo ? 2 : 1);
    __shared__ __attribute__((aligned(16))) char lds[kNarrowThreads / 64 * kSpace];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4;
    char* space = lds + wave * kSpace;
    Fragment<T> fq[KS][KC];
#pragma unroll
    for (int c = 0; c < KC; ++c) {
        const int64_t col = c * 16 + (lane & 15);
        const bool there = col < a.q.rows;
        const T* q = static_cast<const T*>(a.q.p) + (there ? col : 0) * (kGrad ? 1 : a.q.stride);
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const int64_t k = (s * 4 + g) * L, left = there ? a.k - k : 0;
            if constexpr (kGrad) {   // the weight lies across
                Values<T, L> v;
                __builtin_memset(&v, 0, sizeof(v));
#pragma unroll
                for (int i = 0; i < L; ++i) {
                    if (i < left) v.v[i] = q[(k + i) * a.q.stride];
                }
                fq[s][c] = formed<T>(v);
            } else {
                fq[s][c] = formed<T>(read<T, L>(q + k, left));
            }
        }
    }
    Out out;
    out.start(a, 0);
    const int64_t step = static_cast<int64_t>(gridDim.x) * (kNarrowThreads / 64) * 16;
    int64_t row0 = (static_cast<int64_t>(blockIdx.x) * (kNarrowThreads / 64) + wave) * 16;
    Values<T, L> next[KS], other[kTwo ? KS : 1];
    Values<M, L> slope[kGrad ? KS : 1];
    const bool mul = kGrad && a.p.mul != nullptr;
    const auto load = [&](int64_t first) {
        const int64_t row = first + (lane & 15);
        const bool there = row < a.p.rows;
        const int64_t at = there ? row : 0;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const int64_t k = (s * 4 + g) * L, left = there ? a.k - k : 0;
            next[s] = read<T, L>(static_cast<const T*>(a.p.p) + at * a.p.stride + k, left);
            if constexpr (kTwo) {
                other[s] = read<T, L>(static_cast<const T*>(a.other) + at * a.other_stride + k, a.other != nullptr ? left : 0);
            }
            if constexpr (kGrad) {
                if (mul) slope[s] = read<M, L>(static_cast<const M*>(a.p.mul) + at * a.p.stride + k, left);
            }
        }
    };
    if (row0 < a.p.rows) load(row0);
    for (; row0 < a.p.rows; row0 += step) {
        f32x4 acc[KC], more[kTwo ? KC : 1];
        Fragment<T> fp[KS], fo[kTwo ? KS : 1];
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            if constexpr (kGrad) {
                if (mul) {
#pragma unroll
                    for (int i = 0; i < L; ++i) {
                        next[s].v[i] = static_cast<T>(as_float(next[s].v[i]) *
                                                      slope_of<T>(as_float(slope[s].v[i]), a.p.kind, a.p.factor));
                    }
                }
            }
            fp[s] = formed<T>(next[s]);
            if constexpr (kTwo) fo[s] = formed<T>(other[s]);
        }
        if (row0 + step < a.p.rows) load(row0 + step);
#pragma unroll
        for (int c = 0; c < KC; ++c) {
            acc[c] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            if constexpr (kTwo) more[c] = acc[c];
        }
#pragma unroll
        for (int s = 0; s < KS; ++s) {
#pragma unroll
            for (int c = 0; c < KC; ++c) {
                acc[c] = mma(fq[s][c], fp[s], acc[c]);
                if constexpr (kTwo) more[c] = mma(fq[s][c], fo[s], more[c]);
            }
        }
        out.give(space, acc);
        if constexpr (kTwo) out.give(space, more, 1);
        out.rows(a, space, row0);
    }
}

// The gradients of a narrow layer (up to 64 features in and out) in one pass over the rows:
// 64 rows at a time, gz = grad * slope and the input, formed once, lie in LDS as rows of
// features, which the input's gradient reads along (a wavefront has sixteen rows of it) and
// the weight's reads turned (a wavefront has sixteen of its rows, or some columns of them).
// The next rows are on their way into registers meanwhile.  Persistent workgroups; each
// leaves a part of the weight's gradient, which join_kernel joins.
//
// A second pair of operands (second order) is gone through after the first; the input's
// gradient and the bias' are of the last pair.
constexpr int kSlab = 64;   // rows at a time

// Byte of 16-byte piece `c` of row `n` of rows of RB bytes, such that neither eight or sixteen
// rows read along nor four and four rows read turned meet a bank twice.
template <int RB> __device__ inline int both_place(int n, int c) {
    if constexpr (RB == 128) return n * 128 + ((c ^ ((n & 2) | ((n >> 1) & 4) | ((n >> 2) & 1))) << 4);
    else return n * 64 + ((c ^ ((n >> 2) & 3)) << 4);
}

template <typename T, int MT, int KT>
__global__ __launch_bounds__(kNarrowThreads, 2) void narrow_backward_kernel(const Product a) {
    using Out = Finish<T, KT, kLinearGradInput, false>;
    using F = Form<T>;
    using M = typename F::Slope;
    constexpr int kParts = F::kParts, kMB = MT * 32, kKB = KT * 32;   // bytes of a row
    constexpr int kGz = kSlab * kMB, kX = kSlab * kKB, kW = KT * 16 * kMB;
    constexpr int kPlanes = kParts * (kGz + kX), kSpace = 4 * Out::kBytes;
    constexpr bool kApart = sizeof(T) == 2;   // the way out has LDS of its own (float32: there would be one workgroup a CU)
    constexpr int kOperands = kApart || kPlanes > kSpace ? kPlanes : kSpace;
    constexpr int kEachM = MT / 2, kEachK = KT / 2;                   // units of eight values a thread
    constexpr int kWaveM = MT < 4 ? MT : 4, kWaveK = 4 / kWaveM, kC = KT / kWaveK;
    __shared__ __attribute__((aligned(16))) char lds[kOperands + kParts * kW + (kApart ? kSpace : 0)];
    char* const gz = lds;
    char* const x = lds + kParts * kGz;
    char* const wt = lds + kOperands;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4;
    char* const space = (kApart ? wt + kParts * kW : lds) + wave * Out::kBytes;
    const int64_t rows = a.k, out_features = a.job.cols, in_features = a.q.rows;

    const auto put8 = [&](char* plane, int part_bytes, int at, const float (&v)[8]) {
        if constexpr (kParts == 3) {
            const Three t = split(v);
#pragma unroll
            for (int part = 0; part < 3; ++part) __builtin_memcpy(plane + part * part_bytes + at, &t.part[part], 16);
        } else {
            *reinterpret_cast<uint4*>(plane + at) = packed<T>(v);
        }
    };
    // the weight, turned: row k, along m
    const bool wants_input = a.job.out != nullptr;
    if (wants_input) {
        for (int u = threadIdx.x; u < KT * 16 * MT * 2; u += kNarrowThreads) {
            const int k = u % (KT * 16), c = u / (KT * 16);
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int m = c * 8 + i;
                v[i] = m < out_features && k < in_features
                               ? as_float(static_cast<const T*>(a.job.weight)[m * in_features + k]) : 0.0f;
            }
            put8(wt, kW, both_place<kMB>(k, c), v);
        }
    }

    Values<T, 8> vg[kEachM], vx[kEachK];
    Values<M, 8> vd[kEachM];
    const int64_t slabs = (rows + kSlab - 1) / kSlab, all = slabs * a.pairs;
    const auto load = [&](int64_t slab) {
        const bool second = slab >= slabs;
        const Side& p = second ? a.p2 : a.p;
        const Side& q = second ? a.q2 : a.q;
        const int64_t row0 = (second ? slab - slabs : slab) * kSlab;
#pragma unroll
        for (int i = 0; i < kEachM; ++i) {
            const int u = threadIdx.x + i * kNarrowThreads;
            const int64_t row = row0 + u / (MT * 2), m = u % (MT * 2) * 8;
            const int64_t left = row < rows ? out_features - m : 0;
            vg[i] = read<T, 8>(static_cast<const T*>(p.p) + row * p.stride + m, left);
            if (p.mul != nullptr) vd[i] = read<M, 8>(static_cast<const M*>(p.mul) + row * p.stride + m, left);
        }
#pragma unroll
        for (int i = 0; i < kEachK; ++i) {
            const int u = threadIdx.x + i * kNarrowThreads;
            const int64_t row = row0 + u / (KT * 2), k = u % (KT * 2) * 8;
            vx[i] = read<T, 8>(static_cast<const T*>(q.p) + row * q.stride + k, row < rows ? in_features - k : 0);
        }
    };
    // sixteen rows' values along a row's piece, or sixteen columns' values down rows
    const auto along = [&](const char* plane, auto row_bytes, int part_bytes, int row0, int inner) {
        Fragment<T> f;
#pragma unroll
        for (int part = 0; part < kParts; ++part) {
            const char* at = plane + part * part_bytes + both_place<decltype(row_bytes)::value>(row0 + (lane & 15), inner * 4 + g);
            if constexpr (kParts == 3) __builtin_memcpy(&f.v[part], at, 16);
            else __builtin_memcpy(&f.v, at, 16);
        }
        return f;
    };
    const auto down = [&](char* plane, auto row_bytes, int part_bytes, int col0, int inner) {
        Fragment<T> f;
        const int i = lane & 15, n = inner * 32 + g * 8 + (i >> 2), col = col0 + (i & 3) * 4;
#pragma unroll
        for (int part = 0; part < kParts; ++part) {
            i16x4 half[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                char* at = plane + part * part_bytes + both_place<decltype(row_bytes)::value>(n + h * 4, col >> 3) + (col & 7) * 2;
                half[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4*)at);
            }
            if constexpr (kParts == 3) __builtin_memcpy(&f.v[part], half, 16);
            else __builtin_memcpy(&f.v, half, 16);
        }
        return f;
    };
    using RowM = std::integral_constant<int, kMB>;
    using RowK = std::integral_constant<int, kKB>;
    const int tile_m = wave % kWaveM, tile_k = wave / kWaveM * kC;
    const bool has_bias = a.job.bias_out != nullptr && tile_k == 0;

    Out out;
    out.start(a, 0);
    f32x4 acc[kC], bias_sum = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int c = 0; c < kC; ++c) acc[c] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    if (blockIdx.x < all) load(blockIdx.x);
    for (int64_t slab = blockIdx.x; slab < all; slab += gridDim.x) {
        const bool last = slab >= slabs * (a.pairs - 1), second = slab >= slabs;
        const Side& p = second ? a.p2 : a.p;
        __syncthreads();   // of the last slab's reads
#pragma unroll
        for (int i = 0; i < kEachM; ++i) {
            const int u = threadIdx.x + i * kNarrowThreads;
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = as_float(vg[i].v[e]);
            if (p.mul != nullptr) {
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] *= slope_of<T>(as_float(vd[i].v[e]), p.kind, p.factor);
            }
            put8(gz, kGz, both_place<kMB>(u / (MT * 2), u % (MT * 2)), v);
        }
#pragma unroll
        for (int i = 0; i < kEachK; ++i) {
            const int u = threadIdx.x + i * kNarrowThreads;
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = as_float(vx[i].v[e]);
            put8(x, kX, both_place<kKB>(u / (KT * 2), u % (KT * 2)), v);
        }
        __syncthreads();
        if (slab + gridDim.x < all) load(slab + gridDim.x);
        f32x4 of_input[KT];
        const bool input = wants_input && last;
        if (input) {
#pragma unroll
            for (int c = 0; c < KT; ++c) of_input[c] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int inner = 0; inner < MT / 2; ++inner) {
                const Fragment<T> fp = along(gz, RowM{}, kGz, wave * 16, inner);
#pragma unroll
                for (int c = 0; c < KT; ++c) of_input[c] = mma(along(wt, RowM{}, kW, c * 16, inner), fp, of_input[c]);
            }
        }
#pragma unroll
        for (int inner = 0; inner < kSlab / 32; ++inner) {
            const Fragment<T> fp = down(gz, RowM{}, kGz, tile_m * 16, inner);
#pragma unroll
            for (int c = 0; c < kC; ++c) acc[c] = mma(down(x, RowK{}, kX, (tile_k + c) * 16, inner), fp, acc[c]);
            if (has_bias && last) bias_sum = sum_rows(fp, bias_sum);
        }
        if (input) {
            if constexpr (!kApart) __syncthreads();   // of this slab's reads: the way out goes over them
            out.give(space, of_input);
            out.rows(a, space, (second ? slab - slabs : slab) * kSlab + wave * 16);
        }
    }
    float* part = static_cast<float*>(a.job.scratch) + blockIdx.x * (out_features * in_features + out_features);
    const int64_t m = tile_m * 16 + (lane & 15);
    if (m < out_features) {
#pragma unroll
        for (int c = 0; c < kC; ++c) {
            const int64_t k = (tile_k + c) * 16 + g * 4;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (k + i < in_features) part[m * in_features + k + i] = acc[c][i];
            }
        }
        if (has_bias && g == 0) part[out_features * in_features + m] = bias_sum[0];
    }
}

// Joins the parts of a weight's gradient, in their order: kJoin values a workgroup, four a
// thread, whose other threads share out the parts.
constexpr int kJoinThreads = 256;
template <typename T, int kJoin>
__global__ __launch_bounds__(kJoinThreads) void join_kernel(const float* parts, int64_t values, int64_t bias_values,
                                                            int64_t n_parts, int64_t bias_first, int64_t bias_parts,
                                                            T* weight, T* bias) {
    constexpr int kGroups = kJoinThreads / (kJoin / 4);
    __shared__ f32x4 sums[kGroups][kJoin / 4];
    const int group = threadIdx.x / (kJoin / 4), lane = threadIdx.x % (kJoin / 4);
    const int64_t at = static_cast<int64_t>(blockIdx.x) * kJoin + lane * 4;
    const int64_t stride = values + bias_values, left = values - at;
    f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
    const auto add = [&](int64_t first, int64_t n, int64_t from, int64_t most) {
        const int64_t each = (n + kGroups - 1) / kGroups;
        const int64_t end = (group + 1) * each < n ? (group + 1) * each : n;
#pragma unroll 4
        for (int64_t part = group * each; part < end; ++part) {
            const Values<float, 4> v = read<float, 4>(parts + (first + part) * stride + from, most);
#pragma unroll
            for (int i = 0; i < 4; ++i) sum[i] += v.v[i];
        }
    };
    // workgroups past the weight's values have the bias'
    const int64_t weight_groups = (values + kJoin - 1) / kJoin;
    const bool of_bias = static_cast<int64_t>(blockIdx.x) >= weight_groups;
    const int64_t bias_at = at - weight_groups * kJoin;
    if (of_bias) {
        if (bias != nullptr) add(bias_first, bias_parts, values + bias_at, bias_values - bias_at);
    } else if (weight != nullptr) {
        add(0, n_parts, at, left);
    }
    sums[group][lane] = sum;
    __syncthreads();
    if (group != 0) return;
#pragma unroll
    for (int i = 1; i < kGroups; ++i) sum += sums[i][lane];
    const float out[4] = {sum[0], sum[1], sum[2], sum[3]};
    if (of_bias) {
        if (bias != nullptr && bias_at < bias_values) put_values(bias + bias_at, bias_values - bias_at, out);
    } else if (weight != nullptr && left > 0) {
        put_values(weight + at, left, out);
    }
}

// ------------------------------------------------------------------------ launches
// Workgroups of few_rows_kernel, of eight wavefronts each, up to which it is taken: two for
// every CU, which run at once (twice as many of 32 rows in types whose products cost more
// than their bytes).  us of the tiles and of few rows, to both sides of the rule:
//   rows x in x out        float32       bf16         e4m3 to bf16
//     64 x 256 x 256       10.1   3.4    5.8   2.7     5.4   2.6
//    512 x 256 x 256       10.1   4.1    5.9   3.2     5.4   2.9
//     16 x 4096 x 4096      126  19.6   61.4   9.7    44.4   6.2
//     64 x 4096 x 4096      107  46.7   43.0  23.5    19.8  13.4
//    256 x 1024 x 1024     29.4  14.2   12.9   7.8     8.3   5.2
//    512 x 1024 x 1024     29.5  25.1   13.1  13.2     8.4   8.4 (beyond it)
//   1024 x 1024 x 1024     30.2  46.7   13.3  23.7     8.7  14.3 (beyond it for all)
//   2048 x 64 x 64          6.5   3.1    3.7   2.7     8.0   4.3
//   8192 x 64 x 64          6.8   5.5    3.8   3.6     8.1   8.0 (beyond it)
constexpr int64_t kFewGroups = 512;

int64_t tiles_of(int64_t n, int size) { return (n + size - 1) / size; }
int power_of(int64_t n) {   // the next power of two, up to 64
    int p = 1;
    while (p < n && p < 64) p *= 2;
    return p;
}

template <typename T, typename TO, int BR, int BC, int KIND>
int launch(Product a, hipStream_t s) {
    a.row_tiles = tiles_of(a.p.rows, KIND == kLinearSecond ? BR / 2 : BR);
    a.col_tiles = tiles_of(a.q.rows, BC);
    const int64_t tiles = a.row_tiles * a.col_tiles * (KIND == kLinearGradWeight ? a.parts * a.pairs : 1);
    const int64_t groups = (tiles + kXcds - 1) / kXcds * kXcds;
    if (groups * Tile<BR, BC>::kThreads > 0xFFFFFFFFll) ASH_FAIL("linear: too many rows");   // HIP's limit of a grid
    product_kernel<T, TO, BR, BC, KIND><<<static_cast<unsigned>(groups), Tile<BR, BC>::kThreads, 0, s>>>(a);
    ASH_LAUNCH_CHECK();
    return 0;
}

// Whether the large tiles take an operand: 16-byte pieces, rows that do not overlap, tiles
// of less than 2^31 bytes.  `across`: values along the rows in memory.
template <typename T> bool takes_large(const Side& a, int64_t across) {
    return a.mul == nullptr && reinterpret_cast<uintptr_t>(a.p) % 16 == 0 && a.stride * sizeof(T) % 16 == 0 &&
           across * sizeof(T) % 16 == 0 && a.stride >= across && a.stride < (1 << 21);
}

template <typename T, typename TO, int SIZE, int KIND>
int launch_large(Product a, hipStream_t s) {
    a.row_tiles = tiles_of(a.p.rows, SIZE);
    a.col_tiles = tiles_of(a.q.rows, SIZE);
    const int64_t tiles = a.row_tiles * a.col_tiles * (KIND == kLinearGradWeight ? a.parts * a.pairs : 1);
    const int64_t groups = (tiles + kXcds - 1) / kXcds * kXcds;
    if (groups * Tile<SIZE, SIZE>::kThreads > 0xFFFFFFFFll) ASH_FAIL("linear: too many rows");
    large_kernel<T, TO, SIZE, KIND><<<static_cast<unsigned>(groups), Tile<SIZE, SIZE>::kThreads, 0, s>>>(a);
    ASH_LAUNCH_CHECK();
    return 0;
}

// Registers of a weight's fragments, in 16 bytes a lane; up to 32 fit beside the rows' own
// (8-bit rows, which are wider or have to be formed, leave less, and so do gradients, whose
// rows come in twos).
template <typename T> constexpr int narrow_registers(int ks, int kc) {
    return ks * kc * Form<T>::kParts * (Form<T>::kIsByte ? 2 : 1);
}
template <typename T> constexpr bool narrow_fits(int kind, int ks, int kc) {
    return narrow_registers<T>(ks, kc) <= (kind != kLinearForward && ks == 4 ? 16 : 32) &&
           (!Form<T>::kScaled || ks * kc < 16 || (ks < 4 && Form<T>::kIsByte));
}

template <typename T, typename TO, int KIND, int KS, int KC> int launch_narrow(const Product& a, hipStream_t s) {
    if constexpr (narrow_fits<T>(KIND, KS, KC)) {
        const int64_t groups = tiles_of(a.p.rows, kNarrowThreads / 64 * 16);
        // as many workgroups as are under way at once, two a CU or, with fewer registers, three
        // (524 288 rows of 32 float32 to 64: 48 us for 50 forward, 52 for 72 the gradient of the
        // input, 74 for 93 the second order; four a CU 72 and 92; 64 to 64, whose workgroups are
        // two a CU, 98 us forward by two and 104 by three)
        const int64_t most = narrow_registers<T>(KS, KC) <= 12 ? 768 : 512;
        narrow_kernel<T, TO, KS, KC, KIND><<<static_cast<unsigned>(groups < most ? groups : most), kNarrowThreads, 0, s>>>(a);
        ASH_LAUNCH_CHECK();
    }
    return 0;
}
template <typename T, typename TO, int KIND, int KS> int launch_narrow(const Product& a, int kc, hipStream_t s) {
    switch (kc) {
        case 1: return launch_narrow<T, TO, KIND, KS, 1>(a, s);
        case 2: return launch_narrow<T, TO, KIND, KS, 2>(a, s);
        case 4: return launch_narrow<T, TO, KIND, KS, 4>(a, s);
        default: return launch_narrow<T, TO, KIND, KS, 8>(a, s);
    }
}

template <typename T> int join(const LinearJob& j, int64_t parts, int64_t bias_first, int64_t bias_parts, hipStream_t s) {
    const int64_t values = j.cols * j.in;
#define ASH_JOIN(n)                                                                                              \
    join_kernel<T, n><<<static_cast<unsigned>(tiles_of(values, n) + tiles_of(j.cols, n)), kJoinThreads, 0, s>>>( \
            static_cast<const float*>(j.scratch), values, j.cols, parts, bias_first, bias_parts,                 \
            static_cast<T*>(j.weight_out), static_cast<T*>(j.bias_out))
    // 32 threads for a value's parts where there are many (narrow layers: 65 536 rows of 32 bf16
    // to 128 14.8 us with the product, by eight 17.1), eight, or one (8192 rows of 4096 to 4096
    // 270 us with the product, by eight 310, and a grid holds weights of 2^32 values so)
    if (parts > 64) ASH_JOIN(32);
    else if (parts > 4) ASH_JOIN(128);
    else ASH_JOIN(1024);
#undef ASH_JOIN
    ASH_LAUNCH_CHECK();
    return 0;
}

template <typename T, typename TO, int RB> int launch_few(const Product& a, hipStream_t s) {
    few_rows_kernel<T, TO, RB><<<dim3(static_cast<unsigned>(tiles_of(a.q.rows, 16)),
                                      static_cast<unsigned>(tiles_of(a.p.rows, RB * 16))), kFewThreads, 0, s>>>(a);
    ASH_LAUNCH_CHECK();
    return 0;
}

template <typename T> int launch_narrow_backward(const Product& a, hipStream_t s) {
    const unsigned grid = static_cast<unsigned>(narrow_backward_parts(a.k, a.pairs));
    const bool m = a.job.cols > 32, k = a.q.rows > 32;
    if (m && k) narrow_backward_kernel<T, 4, 4><<<grid, kNarrowThreads, 0, s>>>(a);
    else if (m) narrow_backward_kernel<T, 4, 2><<<grid, kNarrowThreads, 0, s>>>(a);
    else if (k) narrow_backward_kernel<T, 2, 4><<<grid, kNarrowThreads, 0, s>>>(a);
    else narrow_backward_kernel<T, 2, 2><<<grid, kNarrowThreads, 0, s>>>(a);
    ASH_LAUNCH_CHECK();
    return 0;
}

template <typename T, typename TO, int KIND>
int launch_by_size(const Product& a, hipStream_t s) {
    if constexpr (KIND == kLinearForward) {
        const int64_t across = tiles_of(a.q.rows, 16);
        if (a.p.rows <= 16 || across * tiles_of(a.p.rows, 16) <= kFewGroups) return launch_few<T, TO, 1>(a, s);
        if (across * tiles_of(a.p.rows, 32) <= (sizeof(T) == 1 ? kFewGroups : 2 * kFewGroups)) return launch_few<T, TO, 2>(a, s);
    }
    if constexpr (KIND != kLinearGradWeight) {
        const int ks = power_of(tiles_of(a.k, 4 * Form<T>::kLane)), kc = power_of(tiles_of(a.q.rows, 16));
        if (ks <= 4 && kc <= 8 && narrow_fits<T>(KIND, ks, kc)) {
            if (ks == 1) return launch_narrow<T, TO, KIND, 1>(a, kc, s);
            if (ks == 2) return launch_narrow<T, TO, KIND, 2>(a, kc, s);
            return launch_narrow<T, TO, KIND, 4>(a, kc, s);
        }
    }
    if constexpr (KIND == kLinearGradWeight) {
        const WeightTile t = weight_tile(a.q.rows, a.p.rows, ASH_LINEAR_DTYPE);
        if (t.cols == 32) return launch<T, TO, 128, 32, KIND>(a, s);
        if (t.rows == 64) return launch<T, TO, 64, 64, KIND>(a, s);
        if constexpr (Form<T>::kParts == 1) {
            if (t.cols >= 128 && takes_large<T>(a.p, a.p.rows) && takes_large<T>(a.q, a.q.rows) &&
                (a.pairs == 1 || (takes_large<T>(a.p2, a.p.rows) && takes_large<T>(a.q2, a.q.rows)))) {
                return t.cols == 256 ? launch_large<T, TO, 256, KIND>(a, s) : launch_large<T, TO, 128, KIND>(a, s);
            }
            return launch<T, TO, 64, 64, KIND>(a, s);
        } else {
            return launch<T, TO, 128, 64, KIND>(a, s);
        }
    }
    if (a.q.rows <= 32) return launch<T, TO, 128, 32, KIND>(a, s);
    // Direct loads: tiles of 256 x 256 from one a CU on (forward of rows x in x out bf16, us of 256,
    // 128 and, without direct loads, 64: 16 384 x 1024 x 1024 38.1 48.6, 10 007 x 1024 x 1024
    // 34.8 36.9 56.7, 8192 x 1024 x 1024 33.7 25.7 30.3), of 128 x 128 from half of that (4096 x
    // 1024 x 1024 33.1 17.1 23.0, gradient of the input 31.0 16.4 37.1; 3000 x 256 x 256 16.9
    // 9.2 6.9).
    if constexpr (Form<T>::kParts == 1 && KIND != kLinearSecond && !std::is_same<T, WideE4M3>::value) {
        if (a.q.rows > 64 && takes_large<T>(a.p, a.k) && takes_large<T>(a.q, KIND == kLinearForward ? a.k : a.q.rows)) {
            if (a.q.rows > 128 && tiles_of(a.p.rows, 256) * tiles_of(a.q.rows, 256) >= 256) {
                return launch_large<T, TO, 256, KIND>(a, s);
            }
            if (tiles_of(a.p.rows, 128) * tiles_of(a.q.rows, 128) >= 128) return launch_large<T, TO, 128, KIND>(a, s);
        }
    }
    // Tiles of 64 x 64 keep most workgroups under way and waste least (us of 64 x 64, 128 x 64,
    // 128 x 128; 10 007 rows of 131 fp16 to 257: 13.6 15.2 19.3, its gradient of the input 14.1
    // 18.9 21.8; 10 007 rows of 512 fp32 to 512: 54 62, the gradient 73 98; 40 000 rows of 333
    // e4m3 to 515: 56 53 62).  Larger ones read less where there are many: in 16 bits from two
    // a CU on, unless the last one is mostly nothing (65 536 rows of 256, gradient of the
    // input: 58 72 44; 40 000 of 131 to 257 forward 55 52 46), of the second order, which keeps
    // twice as much a row, from sixteen of the small ones (65 536 rows of 256: 67 59 63; 5000
    // of 131 to 257 11.7 12.7 16.0), and in float32 from eight with long k, but not of the
    // gradient of the input, whose turning loads take more registers (65 536 rows of 512:
    // forward 291 278, second 512 492, gradient 363 390; second of 10 007 of 2048 to 256, below
    // the rule, 161 201).
    const int64_t row_tiles = tiles_of(a.p.rows, KIND == kLinearSecond ? 32 : 64), tiles = row_tiles * tiles_of(a.q.rows, 64);
    if constexpr (KIND == kLinearSecond || (KIND == kLinearForward && Form<T>::kIsFloat)) {
        if (Form<T>::kIsFloat ? tiles >= 2048 && a.k >= 512 : tiles >= 4096) return launch<T, TO, 128, 64, KIND>(a, s);
    } else if constexpr (KIND != kLinearGradWeight && !Form<T>::kIsFloat && !Form<T>::kScaled) {
        const int64_t across = tiles_of(a.q.rows, 128);
        if (tiles_of(a.p.rows, 128) * across >= 512 && across * 8 <= tiles_of(a.q.rows, 64) * 5) {
            return launch<T, TO, 128, 128, KIND>(a, s);
        }
    }
    return launch<T, TO, 64, 64, KIND>(a, s);
}

}  // namespace

using Operand = TypeOf<ASH_LINEAR_DTYPE>::T;

template <>
int linear_run<ASH_LINEAR_DTYPE>(LinearKind kind, const LinearJob& j, hipStream_t s) {
    using T = Operand;
    Product a{};
    a.job = j;
    switch (kind) {
        case kLinearForward:
            a.p = {j.input, nullptr, j.input_stride, j.rows, 1.0f};
            a.q = {j.weight, nullptr, j.in, j.cols, 1.0f};
            a.k = j.in;
            if constexpr (sizeof(T) == 1) {
                if (j.out_dtype == ASH_F32) return launch_by_size<WideE4M3, float, kLinearForward>(a, s);
                if (j.out_dtype == ASH_F16) return launch_by_size<T, _Float16, kLinearForward>(a, s);
                return launch_by_size<T, __bf16, kLinearForward>(a, s);
            } else {
                return launch_by_size<T, T, kLinearForward>(a, s);
            }
        default:
            break;
    }
    if constexpr (sizeof(T) > 1) {
        switch (kind) {
            case kLinearSecond:
                a.p = {j.input, nullptr, j.input_stride, j.rows, 1.0f};
                a.q = {j.weight, nullptr, j.in, j.cols, 1.0f};
                a.k = j.in;
                a.other = j.second_input;
                a.other_stride = j.second_stride;
                return launch_by_size<T, T, kLinearSecond>(a, s);
            case kLinearGradInput:
                a.p = {j.grad, j.slope, j.cols, j.rows, j.slope_factor, j.slope_kind};
                a.q = {j.weight, nullptr, j.in, j.in, 1.0f};
                a.k = j.cols;
                return launch_by_size<T, T, kLinearGradInput>(a, s);
            case kLinearGradWeight: {
                a.p = {j.grad, j.slope, j.cols, j.cols, j.slope_factor, j.slope_kind};
                a.q = {j.input, nullptr, j.input_stride, j.in, 1.0f};
                a.p2 = {j.second_grad, j.second_slope, j.cols, j.cols, j.slope_factor, j.slope_kind};
                a.q2 = {j.second_factor, nullptr, j.second_stride, j.in, 1.0f};
                a.k = j.rows;
                a.pairs = j.second_grad != nullptr ? 2 : 1;
                a.parts = j.splits;
                a.second_has_bias = j.second_has_bias;
                const int64_t steps = tiles_of(j.rows, Form<T>::kStep);
                a.part_rows = tiles_of(steps, j.splits) * Form<T>::kStep;
                if (j.rows > 0 && launch_by_size<T, T, kLinearGradWeight>(a, s) != 0) return 1;
                return join<T>(j, j.rows > 0 ? a.parts * a.pairs : 0, a.second_has_bias ? a.parts : 0,
                               j.rows > 0 ? a.parts : 0, s);
            }
            case kLinearGradBoth: {
                a.p = {j.grad, j.slope, j.cols, j.rows, j.slope_factor, j.slope_kind};
                a.q = {j.input, nullptr, j.input_stride, j.in, 1.0f};
                a.p2 = {j.second_grad, j.second_slope, j.cols, j.rows, j.slope_factor, j.slope_kind};
                a.q2 = {j.second_factor, nullptr, j.second_stride, j.in, 1.0f};
                a.k = j.rows;
                a.pairs = j.second_grad != nullptr ? 2 : 1;
                a.job.bias = nullptr;
                a.job.residual = nullptr;
                a.job.slope_out = nullptr;
                a.job.activation = ASH_ACT_NONE;
                if (launch_narrow_backward<T>(a, s) != 0) return 1;
                return join<T>(j, narrow_backward_parts(j.rows, a.pairs), 0, narrow_backward_parts(j.rows, a.pairs), s);
            }
            default:
                break;
        }
    }
    ASH_FAIL("linear: no such product of this type");
}

}  // namespace ash
