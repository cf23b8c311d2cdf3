// Weights in 4 bits with a scale per group of 32, 64 or 128 consecutive elements of a row, and products with them.
//
//   s = max |w| of the group / 7, rounded to fp32 and then to the scales' type
//   q = the integer nearest w / s, ties to even, in -7 .. 7;  q s stands for w
//
// A row holds whole groups: behind its last element the codes are zero.  Two codes a byte, the lower half is the even
// element, two's complement.  Codes are exact (nearest_int()).  A group that holds a value that is not finite gets
// scale NaN and codes 0.
//
// Included by prime_hip.hip inside its anonymous namespace; not a translation unit of its own.

// t / d for t < 2^31 by a multiplication: the index arithmetic of a lane would otherwise cost more than its eight elements.
struct FastDiv {
    uint32_t mul, shift, d;
    explicit FastDiv(uint32_t by) : mul(0), shift(0), d(by) {
        while ((uint64_t(1) << shift) < by) ++shift;
        mul = static_cast<uint32_t>((((uint64_t(1) << shift) - by) << 32) / by + 1);
    }
    __device__ __forceinline__ uint32_t quotient(uint32_t t) const { return (__umulhi(t, mul) + t) >> shift; }
};

__device__ __forceinline__ float load_scale(const float* p) { return *p; }
__device__ __forceinline__ float load_scale(const __bf16* p) { return static_cast<float>(*p); }

struct PackArgs {
    const void* weight;
    int64_t stride;             // elements from row to row of the weight
    uint8_t* packed;            // dense rows of groups * group / 2 bytes
    void* scales;               // dense rows of `groups`
    uint32_t vectors;           // eights of this launch: rows * groups * group / 8
    int k;
    int lanes;                  // eights of a group: 4, 8 or 16
    FastDiv per_row;            // eights of a row
};

// A lane takes eight elements, a group's lanes sit side by side in a wavefront.
template <typename T, typename ST>
__global__ __launch_bounds__(256) void group4_pack_kernel(PackArgs a) {
    const uint32_t t = blockIdx.x * 256u + threadIdx.x;
    const bool live = t < a.vectors;
    const uint32_t row = a.per_row.quotient(live ? t : 0u);
    const uint32_t v = (live ? t : 0u) - row * a.per_row.d;
    float w[8];
    load8(static_cast<const T*>(a.weight) + row * a.stride, static_cast<int>(v * 8), a.k, w);
    uint32_t top = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(w[e]) & 0x7fffffffu);
    for (int m = a.lanes >> 1; m >= 1; m >>= 1) top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), m, 64)));
    if (!live) return;
    const bool bad = top >= 0x7f800000u;
    const ST stored = bad ? static_cast<ST>(__builtin_nanf("")) : static_cast<ST>(__uint_as_float(top) / 7.0f);
    float s = static_cast<float>(stored);
    uint32_t codes = 0;
    if (s > 0.0f && s < __builtin_inff()) {
        const float up = s < 0x1p-90f ? 0x1p64f : 1.0f;      // keeps the reciprocal and a residual inside fp32's range
        s *= up;
        const float r = 1.0f / s;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float q = __builtin_amdgcn_fmed3f(nearest_int(w[e] * up, s, r), -7.0f, 7.0f);
            codes |= (static_cast<uint32_t>(static_cast<int>(q)) & 15u) << (4 * e);
        }
    }
    reinterpret_cast<U32U*>(a.packed)[t].v = codes;
    if (v % static_cast<uint32_t>(a.lanes) == 0) static_cast<ST*>(a.scales)[t / static_cast<uint32_t>(a.lanes)] = stored;
}

struct UnpackArgs {
    const uint8_t* packed;
    const void* scales;
    void* out;                  // dense rows of k
    int64_t p_stride;           // bytes from row to row of the codes
    int64_t s_stride;           // elements from row to row of the scales
    uint32_t vectors;
    int k;
    int lane_shift;             // log2 of a group's eights
    FastDiv per_row;            // eights of a row of the output
};

// Code e of a word of eight, as an integer.
__device__ __forceinline__ int code4(uint32_t word, int e) { return static_cast<int>(word << (28 - 4 * e)) >> 28; }

template <typename T, typename ST>
__global__ __launch_bounds__(256) void group4_unpack_kernel(UnpackArgs a) {
    const uint32_t t = blockIdx.x * 256u + threadIdx.x;
    if (t >= a.vectors) return;
    const uint32_t row = a.per_row.quotient(t), v = t - row * a.per_row.d;
    const uint32_t word = reinterpret_cast<const U32U*>(a.packed + row * a.p_stride)[v].v;
    const float s = load_scale(static_cast<const ST*>(a.scales) + row * a.s_stride + (v >> a.lane_shift));
    float o[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = static_cast<float>(code4(word, e)) * s;
    store8(static_cast<T*>(a.out) + static_cast<int64_t>(row) * a.k, static_cast<int>(v * 8), a.k, o);
}

// ---- products of a few rows with 4-bit weights, on the matrix cores ----
//
//   y[m][n] = x_scale[m] * sum over groups g of scale[n][g] * sum over k in g of q[n][k] x[m][k]
//
// Rows of x are the A operand of 16 x 16 x 32 matrix instructions (16 x 16 x 64 for int8), 16 outputs n the B
// operand: a lane holds eight consecutive k of one n, which is one 32-bit word of codes, so the codes go from memory to the
// matrix cores through registers alone, eight instructions a word:
//   bf16   a code's four bits, its sign bit flipped, in the middle of the mantissa of 16.0: that is 24 + q.  The 24 is taken off
//          by a product of the same rows with -24, on the matrix cores too, which is where the sums start from
//   fp16   the same
//   fp32   a row is the sum of three bf16 rows exactly (8 bits of the mantissa each), so three products
//   int8   a code in the upper half of a byte is 16 q; sums are exact integers, the 16 is taken off at the end
// A wavefront takes 128 columns of 16 outputs at a time: lane (n, quarter) loads 16 bytes of row n.  With groups of 128 any
// order of k within them does; with smaller ones the words are transposed between the quarters (four instructions for
// four words), so that an instruction's 32 columns lie in one group and its sums can be scaled on their own.
// The wavefronts of a workgroup split the columns; their sums meet in LDS.  The rows of x are brought to LDS once a workgroup,
// in the order in which the codes come out of their words.

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

struct MatvecArgs {
    const void* x;
    const float* x_scales;      // one a row with int8 rows, else null
    const uint8_t* packed;
    const void* scales;
    void* out;                  // dense rows of n
    int64_t x_stride, p_stride, s_stride;
    int rows;
    int n;
    int k;
    int row_bytes;              // codes of a row that exist: whole groups
    int groups;
    int scale_bf16;
    int out_type;               // PRIME_F32, PRIME_BF16 or PRIME_F16
    int chunk_blocks;           // blocks of 128 columns of x that LDS holds at a time
    int tiles;                  // workgroups along n
};

// Sums of one step: fp32, or exact integers.
template <typename XT> struct Sum { typedef f32x4 type; };
template <> struct Sum<int8_t> { typedef i32x4 type; };

// How eight columns of a row of x are held in LDS: 16-bit values in the order 0 4 1 5 2 6 3 7, bytes in the order
// 0 2 4 6 1 3 5 7; fp32 as three bf16 planes, each the leading bits of what the ones before leave.
template <typename XT> struct Held { typedef u32x4 type; static constexpr int kPlanes = 1; };
template <> struct Held<float> { typedef u32x4 type; static constexpr int kPlanes = 3; };
template <> struct Held<int8_t> { typedef u32x2 type; static constexpr int kPlanes = 1; };

__device__ __forceinline__ uint32_t pair16(uint32_t lo, uint32_t hi) { return (lo & 0xffffu) | hi << 16; }

template <typename XT>
__device__ __forceinline__ void hold8(const XT* __restrict__ row, int i, int n, typename Held<XT>::type (&out)[Held<XT>::kPlanes]) {
    if constexpr (sizeof(XT) == 1) {
        uint32_t lo = 0, hi = 0;
        if (i + 8 <= n) {
            const U64U t = *reinterpret_cast<const U64U*>(row + i);
            lo = t.lo;
            hi = t.hi;
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (i + e < n) (e < 4 ? lo : hi) |= static_cast<uint32_t>(static_cast<uint8_t>(row[i + e])) << (8 * (e & 3));
        }
        out[0] = u32x2{__builtin_amdgcn_perm(hi, lo, 0x06040200u), __builtin_amdgcn_perm(hi, lo, 0x07050301u)};
    } else if constexpr (sizeof(XT) == 2) {
        uint16_t v[8];
        if (i + 8 <= n) {
            const typename Eight<XT>::type t = *reinterpret_cast<const typename Eight<XT>::type*>(row + i);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = __builtin_bit_cast(uint16_t, static_cast<XT>(t[e]));
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = i + e < n ? __builtin_bit_cast(uint16_t, row[i + e]) : uint16_t(0);
        }
        out[0] = u32x4{pair16(v[0], v[4]), pair16(v[1], v[5]), pair16(v[2], v[6]), pair16(v[3], v[7])};
    } else {
        float v[8];
        load8(row, i, n, v);
#pragma unroll
        for (int p = 0; p < 3; ++p) {
            uint32_t b[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                b[e] = __float_as_uint(v[e]) >> 16;
                v[e] -= __uint_as_float(b[e] << 16);      // exact: the bits that are left
            }
            out[p] = u32x4{pair16(b[0], b[4]), pair16(b[1], b[5]), pair16(b[2], b[6]), pair16(b[3], b[7])};
        }
    }
}

// new[j] of quarter q = old[q] of quarter j
__device__ __forceinline__ void transpose_quarters(u32x4& w) {
    const auto a = __builtin_amdgcn_permlane32_swap(w[0], w[2], false, false);
    const auto b = __builtin_amdgcn_permlane32_swap(w[1], w[3], false, false);
    const auto c = __builtin_amdgcn_permlane16_swap(a[0], b[0], false, false);
    const auto d = __builtin_amdgcn_permlane16_swap(a[1], b[1], false, false);
    w = u32x4{c[0], c[1], d[0], d[1]};
}

// Eight codes of a word as 24 + q in 16 bits, in the order 0 4 1 5 2 6 3 7.
template <bool BF16>
__device__ __forceinline__ u32x4 widen_word(uint32_t w) {
    if constexpr (BF16) {
        constexpr uint32_t kMask = 0x00780078u, kBase = 0x41c041c0u;      // 16.0 with the code's sign bit flipped in
        return u32x4{((w << 3) & kMask) ^ kBase, ((w >> 1) & kMask) ^ kBase, ((w >> 5) & kMask) ^ kBase, ((w >> 9) & kMask) ^ kBase};
    } else {
        constexpr uint32_t kMask = 0x03c003c0u, kBase = 0x4e004e00u;
        return u32x4{((w << 6) & kMask) ^ kBase, ((w << 2) & kMask) ^ kBase, ((w >> 2) & kMask) ^ kBase, ((w >> 6) & kMask) ^ kBase};
    }
}
constexpr uint32_t kOffsetBf16 = 0xc1c0c1c0u, kOffsetF16 = 0xce00ce00u;      // -24 twice

template <typename XT>
__device__ __forceinline__ f32x4 product(u32x4 rows, u32x4 codes, f32x4 c) {
    if constexpr (std::is_same<XT, _Float16>::value)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, rows), __builtin_bit_cast(f16x8, codes), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, rows), __builtin_bit_cast(bf16x8, codes), c, 0, 0, 0);
}

// Which row of x a row of the A operand is: with up to 4 rows every fourth (a lane's first of four sums is then the one that
// counts, the others are not used), else all 16.  Rows that do not exist repeat the last one; their sums are dropped.
template <int IR> __device__ __forceinline__ int row_of(int v) { return IR == 1 ? v >> 2 : v; }

template <typename XT, int GS, int IR, int NT, int WK, int XBYTES>
__global__ __launch_bounds__(WK * 64) void matvec4_kernel(MatvecArgs a) {
    constexpr int kThreadsHere = WK * 64;
    constexpr int kPlanes = Held<XT>::kPlanes;
    constexpr int NG = 1 << (7 - GS);             // groups of a block of 128 columns
    constexpr int U = 4 / NT;                     // blocks a wavefront has in flight together
    typedef typename Held<XT>::type held_t;
    constexpr bool kInt = sizeof(XT) == 1;
    __shared__ __align__(16) uint8_t lds[XBYTES];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, quarter = lane >> 4;
    const int tile = blockIdx.x % a.tiles, row0 = blockIdx.x / a.tiles * (IR == 1 ? 4 : 16);
    const int rows = min(a.rows - row0, IR == 1 ? 4 : 16);
    const int blocks = (a.k + 127) >> 7;
    const int row_stride = a.chunk_blocks * 16 * static_cast<int>(sizeof(held_t)) + 16;      // 16 bytes more: rows start on other banks
    const int plane_stride = rows * row_stride;
    const int my_row = min(row_of<IR>(lane & 15), rows - 1) * row_stride + quarter * 4 * static_cast<int>(sizeof(held_t));
    const uint8_t* codes[NT];
    int64_t scale_at[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int n = min((tile * NT + t) * 16 + (lane & 15), a.n - 1);
        codes[t] = a.packed + n * a.p_stride + quarter * 16;
        scale_at[t] = n * a.s_stride;
    }
    auto fetch = [&](int b, u32x4 (&w)[NT], float (&s)[NT][NG]) {
        const bool here = b < blocks && b * 64 + quarter * 16 < a.row_bytes;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            typedef u32x4 __attribute__((aligned(1))) u32x4u;
            w[t] = here ? *reinterpret_cast<const u32x4u*>(codes[t] + static_cast<int64_t>(b) * 64) : u32x4{0, 0, 0, 0};
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                const int at = b * NG + g;
                s[t][g] = 0.0f;
                if (at < a.groups) {
                    if (a.scale_bf16) s[t][g] = load_scale(static_cast<const __bf16*>(a.scales) + scale_at[t] + at);
                    else s[t][g] = load_scale(static_cast<const float*>(a.scales) + scale_at[t] + at);
                }
            }
        }
    };
    float y[NT][IR];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < IR; ++i) y[t][i] = 0.0f;
    u32x4 w[U][NT], w2[U][NT];
    float s[U][NT][NG], s2[U][NT][NG];
#pragma unroll
    for (int u = 0; u < U; ++u) fetch(wave + u * WK, w[u], s[u]);
    const XT* x = static_cast<const XT*>(a.x) + static_cast<int64_t>(row0) * a.x_stride;
    for (int first = 0; first < blocks; first += a.chunk_blocks) {
        const int held = min(a.chunk_blocks, blocks - first);
        if (first) {
            __syncthreads();
            // a chunk that is no whole number of turns leaves its successor's first codes unasked for
            if (a.chunk_blocks % (WK * U)) {
#pragma unroll
                for (int u = 0; u < U; ++u) fetch(first + wave + u * WK, w[u], s[u]);
            }
        }
        // rows of x to LDS: eight columns a lane, put where the lane that multiplies them will look
        for (int i = threadIdx.x; i < rows * held * 16; i += kThreadsHere) {
            const int m = i / (held * 16), c = i - m * (held * 16);
            held_t v[kPlanes];
            hold8(x + m * a.x_stride, first * 128 + c * 8, a.k, v);
            const int in = c & 15, to = (c & ~15) | (GS == 7 ? in : (in & 3) * 4 + (in >> 2));
#pragma unroll
            for (int p = 0; p < kPlanes; ++p) *reinterpret_cast<held_t*>(lds + p * plane_stride + m * row_stride + to * static_cast<int>(sizeof(held_t))) = v[p];
        }
        __syncthreads();
        for (int at = wave; at < held; at += WK * U) {
#pragma unroll
            for (int u = 0; u < U; ++u) fetch(first + at + (U + u) * WK, w2[u], s2[u]);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (at + u * WK >= held) break;      // the same for the whole wavefront
                const uint8_t* mine = lds + my_row + (at + u * WK) * (16 * static_cast<int>(sizeof(held_t)));
                if constexpr (kInt) {
                    u32x4 xa[2];
#pragma unroll
                    for (int j = 0; j < 2; ++j) xa[j] = *reinterpret_cast<const u32x4*>(mine + 16 * j);
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        u32x4 v = w[u][t];
                        if constexpr (GS < 7) transpose_quarters(v);
                        i32x4 acc[NG];
#pragma unroll
                        for (int g = 0; g < NG; ++g) acc[g] = i32x4{0, 0, 0, 0};
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            const u32x4 b{(v[2 * j] << 4) & 0xf0f0f0f0u, v[2 * j] & 0xf0f0f0f0u, (v[2 * j + 1] << 4) & 0xf0f0f0f0u, v[2 * j + 1] & 0xf0f0f0f0u};
                            if constexpr (GS == 5) {
                                const u32x2 a0{xa[j][0], xa[j][1]}, a1{xa[j][2], xa[j][3]}, b0{b[0], b[1]}, b1{b[2], b[3]};
                                acc[2 * j] = __builtin_amdgcn_mfma_i32_16x16x32_i8(__builtin_bit_cast(long, a0), __builtin_bit_cast(long, b0), acc[2 * j], 0, 0, 0);
                                acc[2 * j + 1] = __builtin_amdgcn_mfma_i32_16x16x32_i8(__builtin_bit_cast(long, a1), __builtin_bit_cast(long, b1), acc[2 * j + 1], 0, 0, 0);
                            } else {
                                const int g = GS == 6 ? j : 0;
                                acc[g] = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, xa[j]), __builtin_bit_cast(i32x4, b), acc[g], 0, 0, 0);
                            }
                        }
#pragma unroll
                        for (int g = 0; g < NG; ++g)
#pragma unroll
                            for (int i = 0; i < IR; ++i) y[t][i] = fmaf(static_cast<float>(acc[g][i]), s[u][t][g], y[t][i]);
                    }
                } else {
                    constexpr bool kBf16 = !std::is_same<XT, _Float16>::value;
                    constexpr uint32_t kOff = kBf16 ? kOffsetBf16 : kOffsetF16;
                    u32x4 xa[kPlanes][4];
                    f32x4 start[NG];
#pragma unroll
                    for (int g = 0; g < NG; ++g) start[g] = f32x4{0, 0, 0, 0};
#pragma unroll
                    for (int p = 0; p < kPlanes; ++p)
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            xa[p][j] = *reinterpret_cast<const u32x4*>(mine + p * plane_stride + 16 * j);
                            start[j >> (GS - 5)] = product<XT>(xa[p][j], u32x4{kOff, kOff, kOff, kOff}, start[j >> (GS - 5)]);
                        }
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        u32x4 v = w[u][t];
                        if constexpr (GS < 7) transpose_quarters(v);
                        f32x4 acc[NG];
#pragma unroll
                        for (int g = 0; g < NG; ++g) acc[g] = start[g];
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const u32x4 b = widen_word<kBf16>(v[j]);
#pragma unroll
                            for (int p = 0; p < kPlanes; ++p) acc[j >> (GS - 5)] = product<XT>(xa[p][j], b, acc[j >> (GS - 5)]);
                        }
#pragma unroll
                        for (int g = 0; g < NG; ++g)
#pragma unroll
                            for (int i = 0; i < IR; ++i) y[t][i] = fmaf(acc[g][i], s[u][t][g], y[t][i]);
                    }
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    w[u][t] = w2[u][t];
#pragma unroll
                    for (int g = 0; g < NG; ++g) s[u][t][g] = s2[u][t][g];
                }
        }
    }
    // the wavefronts' sums, added in their order
    float* part = reinterpret_cast<float*>(lds);
    static_assert(WK * NT * IR * 64 * 4 <= XBYTES, "the sums fit where the rows were");
    __syncthreads();
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < IR; ++i) part[((wave * NT + t) * IR + i) * 64 + lane] = y[t][i];
    __syncthreads();
    for (int i = threadIdx.x; i < NT * IR * 64; i += kThreadsHere) {
        float v = part[i];
#pragma unroll
        for (int q = 1; q < WK; ++q) v += part[q * NT * IR * 64 + i];
        const int l = i & 63, r = (i >> 6) % IR, t = (i >> 6) / IR;
        const int m = (l >> 4) * IR + r, n = (tile * NT + t) * 16 + (l & 15);
        if (m >= rows || n >= a.n) continue;
        if constexpr (kInt) v *= a.x_scales[row0 + m] * 0.0625f;
        const int64_t at = static_cast<int64_t>(row0 + m) * a.n + n;
        if (a.out_type == PRIME_F32) static_cast<float*>(a.out)[at] = v;
        else if (a.out_type == PRIME_BF16) static_cast<__bf16*>(a.out)[at] = static_cast<__bf16>(v);
        else static_cast<_Float16*>(a.out)[at] = static_cast<_Float16>(v);
    }
}
