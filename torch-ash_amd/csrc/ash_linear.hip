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
};

constexpr int kThreads = 256;

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
    const void* mul;    // of the same layout, or null
    int64_t stride;     // values between rows (lying along k) or between values of k
    int64_t rows;
};

template <typename T> __device__ inline uint4 packed(const float (&v)[8]) {
    Values<T, 8> r;
#pragma unroll
    for (int i = 0; i < 8; ++i) r.v[i] = static_cast<T>(v[i]);
    uint4 u;
    __builtin_memcpy(&u, &r, 16);
    return u;
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
template <typename T, int ROWS, bool MUL>
struct Along {
    static constexpr int kChunks = Form<T>::kStep / Form<T>::kChunk;
    static constexpr int kEach = (ROWS * kChunks + kThreads - 1) / kThreads;
    static constexpr int N = Form<T>::kChunk;
    static_assert(ROWS * kChunks % kThreads == 0 || kEach == 1, "");
    const T* p[kEach];
    const T* m[kEach];
    int row[kEach], chunk;
    bool mul;
    Values<T, N> v[kEach], w[kEach];

    // kHalves: rows ROWS / 2 and beyond are rows of another operand of the same shape, zeros
    // where there is none (second order)
    template <bool kHalves>
    __device__ void start(const Side& a, int64_t row0, const void* other, int64_t other_stride) {
        chunk = threadIdx.x % kChunks;
        mul = MUL && a.mul != nullptr;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            row[i] = (threadIdx.x + i * kThreads) / kChunks;
            int r = row[i];
            const T* base = static_cast<const T*>(a.p);
            int64_t stride = a.stride;
            if (kHalves && r >= ROWS / 2) {
                r -= ROWS / 2;
                base = static_cast<const T*>(other);
                stride = other_stride;
            }
            const bool there = base != nullptr && row[i] < ROWS && row0 + r < a.rows;
            p[i] = there ? base + (row0 + r) * stride : nullptr;
            if constexpr (MUL) m[i] = there && mul ? static_cast<const T*>(a.mul) + (row0 + r) * stride : nullptr;
        }
    }
    __device__ void load(int64_t k0, int64_t k_end) {
        const int64_t k = k0 + chunk * N;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const int64_t left = p[i] != nullptr ? k_end - k : 0;
            v[i] = read<T, N>(p[i] + k, left);
            if constexpr (MUL) {
                if (mul) w[i] = read<T, N>(m[i] + k, left);
            }
        }
    }
    __device__ void store(char* plane) {
        constexpr int RB = kChunks * 16;
        if (ROWS * kChunks < kThreads && row[0] >= ROWS) return;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            if constexpr (Form<T>::kParts == 3 || MUL || (Form<T>::kScaled && !Form<T>::kIsByte)) {
                float f[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) f[j] = as_float(v[i].v[j]);
                if constexpr (MUL) {
                    if (mul) {
#pragma unroll
                        for (int j = 0; j < 8; ++j) f[j] *= as_float(w[i].v[j]);
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

// Operand that lies across k: value k of row r at p[k * stride + r].  A thread takes
// eight values of k of kWide consecutive rows and turns them.
template <typename T, int ROWS, bool MUL>
struct Across {
    static constexpr int kGroups = Form<T>::kStep / 8;
    static constexpr int kWide = ROWS * kGroups >= kThreads ? ROWS * kGroups / kThreads : 1;
    static constexpr int kUnits = ROWS / kWide * kGroups;
    const T* p;
    const T* m;
    int64_t stride, left;   // rows from this thread's first to the last
    int row, group;
    bool mul, works;
    Values<T, kWide> v[8], w[8];

    template <bool>
    __device__ void start(const Side& a, int64_t row0, const void*, int64_t) {
        row = threadIdx.x % (ROWS / kWide) * kWide;
        group = threadIdx.x / (ROWS / kWide);
        works = threadIdx.x < kUnits;
        stride = a.stride;
        left = works ? a.rows - (row0 + row) : 0;
        mul = MUL && a.mul != nullptr;
        p = static_cast<const T*>(a.p) + row0 + row;
        m = mul ? static_cast<const T*>(a.mul) + row0 + row : nullptr;
    }
    __device__ void load(int64_t k0, int64_t k_end) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int64_t k = k0 + group * 8 + j;
            const int64_t n = k < k_end ? left : 0;
            v[j] = read<T, kWide>(p + k * stride, n);
            if constexpr (MUL) {
                if (mul) w[j] = read<T, kWide>(m + k * stride, n);
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
                    if (mul) f[j] *= as_float(w[j].v[i]);
                }
            }
            put<T, ROWS>(plane, row + i, group, f);
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
__device__ inline float sigmoid(float v) { return 1.0f / (1.0f + expf(-v)); }

// f(z), f'(z) and f''(z) of eight values at a time.
template <int N>
__device__ inline void activate(int kind, float a, const float (&z)[N], float (&y)[N], float (&d)[N]) {
    switch (kind) {
        case ASH_ACT_RELU:
#pragma unroll
            for (int i = 0; i < N; ++i) {
                // NaN stays NaN
                y[i] = z[i] < 0.0f ? 0.0f : z[i];
                d[i] = z[i] > 0.0f ? 1.0f : 0.0f;
            }
            break;
        case ASH_ACT_SILU:
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float p = sigmoid(z[i]);
                y[i] = z[i] * p;
                d[i] = p * (1.0f + z[i] * (1.0f - p));
            }
            break;
        case ASH_ACT_GELU:
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float c = 0.5f * erfcf(-0.70710678f * z[i]);
                y[i] = z[i] * c;
                d[i] = c + z[i] * 0.39894228f * expf(-0.5f * z[i] * z[i]);
            }
            break;
        case ASH_ACT_SOFTPLUS:
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float v = a * z[i], e = expf(-fabsf(v));
                y[i] = (v > 0.0f ? z[i] : 0.0f) + log1pf(e) / a;
                d[i] = (v > 0.0f ? 1.0f : e) / (1.0f + e);
                if (v != v) y[i] = d[i] = v;
            }
            break;
        case ASH_ACT_SINE:
#pragma unroll
            for (int i = 0; i < N; ++i) {
                float s, c;
                sincosf(a * z[i], &s, &c);
                y[i] = s;
                d[i] = a * c;
            }
            break;
        default:
#pragma unroll
            for (int i = 0; i < N; ++i) {
                y[i] = z[i];
                d[i] = 1.0f;
            }
    }
}

template <int N>
__device__ inline void curve(int kind, float a, const float (&z)[N], float (&d)[N], float (&dd)[N]) {
    switch (kind) {
        case ASH_ACT_SILU:
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float p = sigmoid(z[i]);
                d[i] = p * (1.0f + z[i] * (1.0f - p));
                dd[i] = p * (1.0f - p) * (2.0f + z[i] * (1.0f - 2.0f * p));
            }
            break;
        case ASH_ACT_GELU:
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float density = 0.39894228f * expf(-0.5f * z[i] * z[i]);
                d[i] = 0.5f * erfcf(-0.70710678f * z[i]) + z[i] * density;
                dd[i] = (2.0f - z[i] * z[i]) * density;
            }
            break;
        case ASH_ACT_SOFTPLUS:
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float v = a * z[i], e = expf(-fabsf(v)), r = 1.0f / (1.0f + e);
                d[i] = v > 0.0f ? r : e * r;
                dd[i] = a * e * r * r;
            }
            break;
        case ASH_ACT_SINE:
#pragma unroll
            for (int i = 0; i < N; ++i) {
                float s, c;
                sincosf(a * z[i], &s, &c);
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

template <typename T> __device__ inline void write8(T* out, int64_t left, const float (&v)[8]) {
    Values<T, 8> r;
#pragma unroll
    for (int i = 0; i < 8; ++i) r.v[i] = static_cast<T>(v[i]);
    if (left >= 8) {
        __builtin_memcpy(out, &r, sizeof(r));
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (i < left) out[i] = r.v[i];
        }
    }
}

template <typename T> __device__ inline void read8(const T* in, int64_t left, float (&v)[8]) {
    const Values<T, 8> r = read<T, 8>(in, left);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = as_float(r.v[i]);
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

template <typename T, int BR, int BC> struct Shared {
    static constexpr int kRowBytes = Form<T>::kStep / Form<T>::kChunk * 16;
    static constexpr int kP = Form<T>::kParts * BR * kRowBytes;
    static constexpr int kQ = Form<T>::kParts * BC * kRowBytes;
    static constexpr int kStride = BC + 4;       // floats between rows of the result
    static constexpr int kOut = BR * kStride * 4;
    static constexpr int kBytes = 2 * (kP + kQ) > kOut ? 2 * (kP + kQ) : kOut;
};

template <typename T, int BR, int BC>
struct Tile {
    static constexpr int kWaveCols = BC >= 128 ? 2 : (BR >= 128 ? 1 : 2);
    static constexpr int kWaveRows = 4 / kWaveCols;
    static constexpr int kR = BR / kWaveRows / 16, kC = BC / kWaveCols / 16;
};

template <typename T, typename TO, int BR, int BC, int KIND>
__global__ __launch_bounds__(kThreads) void product_kernel(const Product a) {
    using S = Shared<T, BR, BC>;
    using W = Tile<T, BR, BC>;
    constexpr bool kGrad = KIND == kLinearGradInput || KIND == kLinearGradWeight;
    constexpr int kStep = Form<T>::kStep;
    __shared__ __attribute__((aligned(16))) char lds[S::kBytes];

    const int64_t tiles = a.row_tiles * a.col_tiles;
    int64_t tile, row_tile, col_tile;
    if (!tile_of(a, tiles * (KIND == kLinearGradWeight ? a.parts * a.pairs : 1), tile)) return;
    int64_t k0 = 0, k_end = a.k;
    bool second = false, sums = false;
    int64_t part = 0;
    if constexpr (KIND == kLinearGradWeight) {
        part = tile / tiles;
        tile = tile % tiles;
        second = part >= a.parts;
        k0 = (second ? part - a.parts : part) * a.part_rows;
        k_end = k0 + a.part_rows < a.k ? k0 + a.part_rows : a.k;
        row_tile = tile % a.row_tiles;
        col_tile = tile / a.row_tiles;
        sums = a.job.bias_out != nullptr && col_tile == 0 && second == a.second_has_bias;
    } else {
        banded(a, tile, row_tile, col_tile);
    }
    constexpr int kRowsOut = KIND == kLinearSecond ? BR / 2 : BR;
    const int64_t row0 = row_tile * kRowsOut, col0 = col_tile * BC;

    using LoadP = std::conditional_t<KIND == kLinearGradWeight, Across<T, BR, true>, Along<T, BR, kGrad>>;
    using LoadQ = std::conditional_t<kGrad, Across<T, BC, false>, Along<T, BC, false>>;
    LoadP p;
    LoadQ q;
    p.template start<KIND == kLinearSecond>(second ? a.p2 : a.p, row0, a.other, a.other_stride);
    q.template start<false>(second ? a.q2 : a.q, col0, nullptr, 0);

    const int wave = threadIdx.x >> 6;
    const int wave_row = wave / W::kWaveCols * W::kR * 16, wave_col = wave % W::kWaveCols * W::kC * 16;
    f32x4 acc[W::kR][W::kC], rows_sum[W::kR];
#pragma unroll
    for (int r = 0; r < W::kR; ++r) {
        rows_sum[r] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
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
            for (int c = 0; c < W::kC; ++c) fq[c] = fetch<T, BC>(now + S::kP, wave_col + c * 16, inner);
#pragma unroll
            for (int r = 0; r < W::kR; ++r) {
                const Fragment<T> fp = fetch<T, BR>(now, wave_row + r * 16, inner);
#pragma unroll
                for (int c = 0; c < W::kC; ++c) acc[r][c] = mma(fq[c], fp, acc[r][c]);
                if constexpr (KIND == kLinearGradWeight) {
                    if (sums) rows_sum[r] = sum_rows(fp, rows_sum[r]);
                }
            }
        }
        if (step + 1 < steps) {
            p.store(next);
            q.store(next + S::kP);
        }
    }

    const int lane = threadIdx.x & 63;
    if constexpr (KIND == kLinearGradWeight) {
        // a part's sums, in float32; reduce_kernel joins the parts
        float* out = static_cast<float*>(a.job.scratch) + part * (a.p.rows * a.q.rows + a.p.rows);
        float* bias = out + a.p.rows * a.q.rows;
#pragma unroll
        for (int r = 0; r < W::kR; ++r) {
            const int64_t row = row0 + wave_row + r * 16 + (lane & 15);
            if (row >= a.p.rows) continue;
#pragma unroll
            for (int c = 0; c < W::kC; ++c) {
                const int64_t col = col0 + wave_col + c * 16 + (lane >> 4) * 4;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (col + i < a.q.rows) out[row * a.q.rows + col + i] = acc[r][c][i];
                }
            }
            if (sums && wave_col == 0 && lane < 16) bias[row] = rows_sum[r][0];
        }
        return;
    } else {
        // the tile goes through LDS once more, so that a thread has eight columns of a row:
        // operands and results then come and go in whole lines
        __syncthreads();
        float* sums_of = reinterpret_cast<float*>(lds);
#pragma unroll
        for (int r = 0; r < W::kR; ++r) {
#pragma unroll
            for (int c = 0; c < W::kC; ++c) {
                *reinterpret_cast<f32x4*>(sums_of + (wave_row + r * 16 + (lane & 15)) * S::kStride + wave_col +
                                          c * 16 + (lane >> 4) * 4) = acc[r][c];
            }
        }
        __syncthreads();
        constexpr int kAcross = BC / 8, kDown = kThreads / kAcross;
        const LinearJob& j = a.job;
        const int at = threadIdx.x % kAcross * 8;
        const int64_t col = col0 + at, left = a.q.rows - col;
        if (left <= 0) return;
        float bias[8], scale[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            bias[i] = 0.0f;
            scale[i] = 1.0f;
        }
        if (j.bias != nullptr) read8(static_cast<const TO*>(j.bias) + col, left, bias);
        if constexpr (Form<T>::kScaled) read8(j.weight_scales + col, left, scale);
#pragma unroll 1
        for (int r = threadIdx.x / kAcross; r < kRowsOut; r += kDown) {
            const int64_t row = row0 + r;
            if (row >= a.p.rows) break;
            float z[8], y[8], d[8];
            const float row_scale = Form<T>::kScaled ? j.input_scales[row] : 1.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                z[i] = sums_of[r * S::kStride + at + i];
                if constexpr (Form<T>::kScaled) z[i] *= row_scale * scale[i];
                z[i] += bias[i];
            }
            const int64_t o = row * a.q.rows + col;
            if constexpr (KIND == kLinearSecond) {
                // t: the derivative of <second input, gradient of the input> by gz
                float t[8], g[8], dd[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) t[i] = sums_of[(kRowsOut + r) * S::kStride + at + i];
                if (j.addend != nullptr) {
                    float more[8];
                    read8(static_cast<const TO*>(j.addend) + row * j.addend_stride + col, left, more);
#pragma unroll
                    for (int i = 0; i < 8; ++i) t[i] += more[i];
                }
                read8(static_cast<const TO*>(j.grad) + o, left, g);
                curve(j.activation, j.act_scale, z, d, dd);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    y[i] = t[i] * d[i];
                    dd[i] *= t[i] * g[i];
                }
                if (j.out != nullptr) write8(static_cast<TO*>(j.out) + o, left, y);
                if (j.curvature_out != nullptr) write8(static_cast<TO*>(j.curvature_out) + o, left, dd);
            } else {
                activate(j.activation, j.act_scale, z, y, d);
                if (j.residual != nullptr) {
                    float more[8];
                    read8(static_cast<const TO*>(j.residual) + row * j.residual_stride + col, left, more);
#pragma unroll
                    for (int i = 0; i < 8; ++i) y[i] += more[i];
                }
                write8(static_cast<TO*>(j.out) + o, left, y);
                if (j.slope_out != nullptr) write8(static_cast<TO*>(j.slope_out) + o, left, d);
            }
        }
    }
}

// Few rows: 16 columns for 16 rows a workgroup, whose eight wavefronts share out k and
// join their sums in LDS.  Operands go from memory straight into the matrix instructions:
// every value of the weight is read once and used once, so there is nothing to keep.
constexpr int kFewThreads = 512;
constexpr int kFewWaves = kFewThreads / 64;
constexpr int kAhead = 4;   // steps whose operands are on their way at a time

template <typename T> __device__ inline Fragment<T> direct(const T* p, int64_t left) {
    const Values<T, Form<T>::kLane> v = read<T, Form<T>::kLane>(p, left);
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

template <typename T, typename TO>
__global__ __launch_bounds__(kFewThreads) void few_rows_kernel(const Product a) {
    constexpr int kEach = Form<T>::kLane * 4;   // values of k a step
    __shared__ float sums[kFewWaves][16][20];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4;
    const int64_t col0 = static_cast<int64_t>(blockIdx.x) * 16, row0 = static_cast<int64_t>(blockIdx.y) * 16;
    const int64_t row = row0 + (lane & 15), col = col0 + (lane & 15);
    const bool has_row = row < a.p.rows, has_col = col < a.q.rows;
    const T* p = static_cast<const T*>(a.p.p) + (has_row ? row : 0) * a.p.stride;
    const T* q = static_cast<const T*>(a.q.p) + (has_col ? col : 0) * a.q.stride;
    f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int64_t k0 = static_cast<int64_t>(wave) * kEach; k0 < a.k; k0 += kAhead * kFewWaves * kEach) {
        Fragment<T> fp[kAhead], fq[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const int64_t k = k0 + i * kFewWaves * kEach + g * Form<T>::kLane;
            fq[i] = direct(q + k, has_col ? a.k - k : 0);
            fp[i] = direct(p + k, has_row ? a.k - k : 0);
        }
#pragma unroll
        for (int i = 0; i < kAhead; ++i) acc = mma(fq[i], fp[i], acc);
    }
    *reinterpret_cast<f32x4*>(&sums[wave][lane & 15][g * 4]) = acc;
    __syncthreads();
    if (threadIdx.x >= 256) return;
    const int r = threadIdx.x >> 4, c = threadIdx.x & 15;
    const int64_t out_row = row0 + r, out_col = col0 + c;
    if (out_row >= a.p.rows || out_col >= a.q.rows) return;
    float z[1] = {0.0f}, y[1], d[1];
#pragma unroll
    for (int i = 0; i < kFewWaves; ++i) z[0] += sums[i][r][c];
    const LinearJob& j = a.job;
    if constexpr (Form<T>::kScaled) z[0] *= j.input_scales[out_row] * j.weight_scales[out_col];
    if (j.bias != nullptr) z[0] += as_float(static_cast<const TO*>(j.bias)[out_col]);
    activate(j.activation, j.act_scale, z, y, d);
    if (j.residual != nullptr) y[0] += as_float(static_cast<const TO*>(j.residual)[out_row * j.residual_stride + out_col]);
    const int64_t o = out_row * a.q.rows + out_col;
    static_cast<TO*>(j.out)[o] = static_cast<TO>(y[0]);
    if (j.slope_out != nullptr) static_cast<TO*>(j.slope_out)[o] = static_cast<TO>(d[0]);
}

// Joins the parts of a weight's gradient, in their order.
constexpr int kJoin = 32;   // values a workgroup, eight threads each
template <typename T>
__global__ __launch_bounds__(kThreads) void join_kernel(const float* parts, int64_t values, int64_t bias_values,
                                                        int64_t n_parts, int64_t bias_first, int64_t bias_parts,
                                                        T* weight, T* bias) {
    __shared__ float sums[kThreads / kJoin][kJoin];
    const int64_t at = static_cast<int64_t>(blockIdx.x) * kJoin + threadIdx.x % kJoin;
    const int group = threadIdx.x / kJoin;
    constexpr int kGroups = kThreads / kJoin;
    const int64_t stride = values + bias_values;
    const bool of_bias = at >= values;
    const int64_t first = of_bias ? bias_first : 0, n = of_bias ? bias_parts : n_parts;
    float sum = 0.0f;
    if (at < stride && (of_bias ? bias != nullptr : weight != nullptr)) {
        const int64_t each = (n + kGroups - 1) / kGroups;
        const int64_t from = first + group * each, to = group * each + each < n ? from + each : first + n;
#pragma unroll 8
        for (int64_t part = from; part < to; ++part) sum += parts[part * stride + at];
    }
    sums[group][threadIdx.x % kJoin] = sum;
    __syncthreads();
    if (group != 0 || at >= stride) return;
#pragma unroll
    for (int i = 1; i < kGroups; ++i) sum += sums[i][threadIdx.x % kJoin];
    if (of_bias) {
        if (bias != nullptr) bias[at - values] = static_cast<T>(sum);
    } else if (weight != nullptr) {
        weight[at] = static_cast<T>(sum);
    }
}

// ------------------------------------------------------------------------ launches
constexpr int64_t kFewRows = 64;

int64_t tiles_of(int64_t n, int size) { return (n + size - 1) / size; }

template <typename T, typename TO, int BR, int BC, int KIND>
int launch(Product a, hipStream_t s) {
    a.row_tiles = tiles_of(a.p.rows, KIND == kLinearSecond ? BR / 2 : BR);
    a.col_tiles = tiles_of(a.q.rows, BC);
    const int64_t tiles = a.row_tiles * a.col_tiles * (KIND == kLinearGradWeight ? a.parts * a.pairs : 1);
    const int64_t groups = (tiles + kXcds - 1) / kXcds * kXcds;
    if (groups > 0x7FFFFFFFll) ASH_FAIL("linear: too many rows");
    product_kernel<T, TO, BR, BC, KIND><<<static_cast<unsigned>(groups), kThreads, 0, s>>>(a);
    ASH_LAUNCH_CHECK();
    return 0;
}

template <typename T, typename TO, int KIND>
int launch_by_size(const Product& a, hipStream_t s) {
    if constexpr (KIND == kLinearForward) {
        if (a.p.rows <= kFewRows) {
            few_rows_kernel<T, TO><<<dim3(static_cast<unsigned>(tiles_of(a.q.rows, 16)),
                                          static_cast<unsigned>(tiles_of(a.p.rows, 16))),
                                     kFewThreads, 0, s>>>(a);
            ASH_LAUNCH_CHECK();
            return 0;
        }
    }
    if (a.q.rows <= 32) return launch<T, TO, 128, 32, KIND>(a, s);
    if constexpr (KIND == kLinearGradWeight) {   // the parts fill the chip whatever the tile
        if (a.p.rows <= 64) return launch<T, TO, 64, 64, KIND>(a, s);
        if constexpr (Form<T>::kParts == 1) {
            if (a.q.rows > 64) return launch<T, TO, 128, 128, KIND>(a, s);
        }
        return launch<T, TO, 128, 64, KIND>(a, s);
    }
    if (tiles_of(a.p.rows, 128) * tiles_of(a.q.rows, 64) < 256) return launch<T, TO, 64, 64, KIND>(a, s);
    if constexpr (Form<T>::kParts == 1) {
        if (a.q.rows > 64) return launch<T, TO, 128, 128, KIND>(a, s);
    }
    return launch<T, TO, 128, 64, KIND>(a, s);
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
            a.p = {j.input, nullptr, j.input_stride, j.rows};
            a.q = {j.weight, nullptr, j.in, j.cols};
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
                a.p = {j.input, nullptr, j.input_stride, j.rows};
                a.q = {j.weight, nullptr, j.in, j.cols};
                a.k = j.in;
                a.other = j.second_input;
                a.other_stride = j.second_stride;
                return launch_by_size<T, T, kLinearSecond>(a, s);
            case kLinearGradInput:
                a.p = {j.grad, j.slope, j.cols, j.rows};
                a.q = {j.weight, nullptr, j.in, j.in};
                a.k = j.cols;
                return launch_by_size<T, T, kLinearGradInput>(a, s);
            case kLinearGradWeight: {
                a.p = {j.grad, j.slope, j.cols, j.cols};
                a.q = {j.input, nullptr, j.input_stride, j.in};
                a.p2 = {j.second_grad, j.second_slope, j.cols, j.cols};
                a.q2 = {j.second_factor, nullptr, j.second_stride, j.in};
                a.k = j.rows;
                a.pairs = j.second_grad != nullptr ? 2 : 1;
                a.parts = j.splits;
                a.second_has_bias = j.second_has_bias;
                const int64_t steps = tiles_of(j.rows, Form<T>::kStep);
                a.part_rows = tiles_of(steps, j.splits) * Form<T>::kStep;
                if (j.rows > 0 && launch_by_size<T, T, kLinearGradWeight>(a, s) != 0) return 1;
                const int64_t values = j.cols * j.in, parts = j.rows > 0 ? a.parts * a.pairs : 0;
                const int64_t groups = tiles_of(values + j.cols, kJoin);
                join_kernel<T><<<static_cast<unsigned>(groups), kThreads, 0, s>>>(
                        static_cast<const float*>(j.scratch), values, j.cols, parts,
                        a.second_has_bias ? a.parts : 0, j.rows > 0 ? a.parts : 0, static_cast<T*>(j.out),
                        static_cast<T*>(j.bias_out));
                ASH_LAUNCH_CHECK();
                return 0;
            }
            default:
                break;
        }
    }
    ASH_FAIL("linear: no such product of this type");
}

}  // namespace ash
