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

struct __attribute__((packed)) U16U { uint16_t v; };

__device__ __forceinline__ float load_scale(const float* p) { return *p; }
__device__ __forceinline__ float load_scale(const __bf16* p) { return static_cast<float>(*p); }

// Elements of a lane: 16 bytes of the matrix, so that a wavefront's access covers 1 KiB without gaps (fp32 elements eight a lane, in
// two accesses that each touch every second 16 bytes: 22528 x 8192 packed in 164 us and widened in 189).
template <typename T> constexpr int kUnit = 16 / static_cast<int>(sizeof(T));
template <typename T> struct Unit;
template <> struct Unit<float> { typedef float type __attribute__((ext_vector_type(4), aligned(4))); };
template <> struct Unit<__bf16> { typedef Eight<__bf16>::type type; };
template <> struct Unit<_Float16> { typedef Eight<_Float16>::type type; };

template <typename T, bool ONCE>
__device__ __forceinline__ typename Unit<T>::type take_unit(const T* __restrict__ row, int i, int n) {
    typename Unit<T>::type t;
    if (i + kUnit<T> <= n) {
        const typename Unit<T>::type* p = reinterpret_cast<const typename Unit<T>::type*>(row + i);
        if constexpr (ONCE) t = __builtin_nontemporal_load(p);
        else t = *p;
    } else {
#pragma unroll
        for (int e = 0; e < kUnit<T>; ++e) t[e] = i + e < n ? row[i + e] : static_cast<T>(0.0f);
    }
    return t;
}

struct PackArgs {
    const void* weight;
    int64_t stride;             // elements from row to row of the weight
    uint8_t* packed;            // dense rows of groups * group / 2 bytes
    void* scales;               // dense rows of `groups`
    uint32_t units;             // of this launch: rows * groups * group / kUnit
    int k;
    int lanes;                  // units of a group: 4, 8, 16 or 32
    int lane_shift;
    FastDiv per_row;            // units of a row
};

// The largest magnitude of a unit, as the bits of a float; a NaN compares above all numbers.  16-bit elements two at a time, as whole numbers.
template <typename T>
__device__ __forceinline__ uint32_t largest_bits(const typename Unit<T>::type& v) {
    if constexpr (sizeof(T) == 4) {
        return max(max(__float_as_uint(v[0]) & 0x7fffffffu, __float_as_uint(v[1]) & 0x7fffffffu),
                   max(__float_as_uint(v[2]) & 0x7fffffffu, __float_as_uint(v[3]) & 0x7fffffffu));
    } else {
        typedef uint16_t __attribute__((ext_vector_type(2))) u16x2;
        typedef uint32_t __attribute__((ext_vector_type(4))) words;
        T one[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) one[e] = v[e];
        words w;
        __builtin_memcpy(&w, one, 16);
        u16x2 top = __builtin_bit_cast(u16x2, w[0] & 0x7fff7fffu);
#pragma unroll
        for (int i = 1; i < 4; ++i) top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2, w[i] & 0x7fff7fffu));
        const uint16_t m = top[0] > top[1] ? top[0] : top[1];
        return __float_as_uint(static_cast<float>(__builtin_bit_cast(T, m)));
    }
}

// One unit of the matrix (number t, the v-th of its row) to codes, and its group's scale.
template <typename T, typename ST>
__device__ __forceinline__ void pack_unit(const PackArgs& a, uint32_t t, uint32_t v, const typename Unit<T>::type& raw) {
    constexpr int E = kUnit<T>;
    uint32_t top = largest_bits<T>(raw);
    // the largest of the group's lanes, in all of them
    auto turned = [](uint32_t x, auto n) {
        return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(static_cast<int>(x), static_cast<int>(x), decltype(n)::value, 0xf, 0xf, false));
    };
    top = max(top, turned(top, std::integral_constant<int, 0xb1>{}));                       // quad_perm 1 0 3 2
    top = max(top, turned(top, std::integral_constant<int, 0x4e>{}));                       // quad_perm 2 3 0 1
    if (a.lanes > 4) top = max(top, turned(top, std::integral_constant<int, 0x141>{}));     // row_half_mirror: the other four of eight
    if (a.lanes > 8) top = max(top, turned(top, std::integral_constant<int, 0x140>{}));     // row_mirror: the other eight
    if (E == 4 && a.lanes > 16) {
        const auto r = __builtin_amdgcn_permlane16_swap(top, top, false, false);            // the neighbouring row of 16
        top = max(static_cast<uint32_t>(r[0]), static_cast<uint32_t>(r[1]));
    }
    if (t >= a.units) return;
    float w[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] = e < E ? static_cast<float>(raw[e % E]) : 0.0f;
    const float largest = __uint_as_float(top);
    ST stored;
    uint32_t codes = 0;
    if (largest > 0x1p-80f && largest < 0x1p126f) {
        // largest / 7, correctly rounded: the product with 1/7, put right by what it leaves (Markstein's division)
        const float q = largest * (1.0f / 7.0f);
        stored = static_cast<ST>(__builtin_fmaf(__builtin_fmaf(-7.0f, q, largest), 1.0f / 7.0f, q));
        const float s = static_cast<float>(stored);
        float f[8];
        round8<8>(w, s, __builtin_amdgcn_rcpf(s), f);      // the scale's own rounding puts a quotient up to 7.03: nearest 7
        const uint32_t even = low_bytes(__float_as_uint(f[0]), __float_as_uint(f[2]), __float_as_uint(f[4]), __float_as_uint(f[6])) & 0x0f0f0f0fu;
        const uint32_t odd = low_bytes(__float_as_uint(f[1]), __float_as_uint(f[3]), __float_as_uint(f[5]), __float_as_uint(f[7]));
        codes = even | (odd << 4 & 0xf0f0f0f0u);
    } else {
        // zeros, what is not finite, and magnitudes so small or large that a step above would leave fp32's normal numbers
        stored = top >= 0x7f800000u ? static_cast<ST>(__builtin_nanf("")) : static_cast<ST>(largest / 7.0f);
        float s = static_cast<float>(stored);
        if (s > 0.0f && s < __builtin_inff()) {
            const float by = s < 1.0f ? 0x1p64f : 0x1p-64f;
            s *= by;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                // a subnormal scale is rounded coarsely: quotients beyond 7 are taken to 7
                const float k = __builtin_amdgcn_fmed3f(nearest_int(w[e] * by, s, 1.0f / s), -7.0f, 7.0f);
                codes |= (static_cast<uint32_t>(static_cast<int>(k)) & 15u) << (4 * e);
            }
        }
    }
    if constexpr (E == 8) reinterpret_cast<U32U*>(a.packed)[t].v = codes;
    else reinterpret_cast<U16U*>(a.packed)[t].v = static_cast<uint16_t>(codes);
    if ((v & (a.lanes - 1)) == 0) static_cast<ST*>(a.scales)[t >> a.lane_shift] = stored;
}

constexpr int kPackEach = 2;         // units of a lane, all on their way together

// A group's lanes sit side by side in a wavefront.
template <typename T, typename ST, bool ONCE>
__global__ __launch_bounds__(256) void group4_pack_kernel(PackArgs a) {
    typename Unit<T>::type raw[kPackEach];
    uint32_t col[kPackEach];
#pragma unroll
    for (int i = 0; i < kPackEach; ++i) {
        const uint32_t t = (blockIdx.x * kPackEach + i) * 256u + threadIdx.x, in = t < a.units ? t : 0u;
        const uint32_t row = a.per_row.quotient(in);
        col[i] = in - row * a.per_row.d;
        raw[i] = take_unit<T, ONCE>(static_cast<const T*>(a.weight) + row * a.stride, static_cast<int>(col[i] * kUnit<T>), a.k);
    }
#pragma unroll
    for (int i = 0; i < kPackEach; ++i) pack_unit<T, ST>(a, (blockIdx.x * kPackEach + i) * 256u + threadIdx.x, col[i], raw[i]);
}

struct UnpackArgs {
    const uint8_t* packed;
    const void* scales;
    void* out;                  // dense rows of k
    int64_t p_stride;           // bytes from row to row of the codes
    int64_t s_stride;           // elements from row to row of the scales
    uint32_t units;
    int k;
    int lane_shift;             // log2 of a group's units
    FastDiv per_row;            // units of a row of the output
};

constexpr int kUnpackEach = 2;       // units of a lane, all on their way together

// Code e of a word of eight, as an integer.
__device__ __forceinline__ int code4(uint32_t word, int e) { return static_cast<int>(word << (28 - 4 * e)) >> 28; }

template <typename T, typename ST>
__global__ __launch_bounds__(256) void group4_unpack_kernel(UnpackArgs a) {
    constexpr int E = kUnit<T>;
    uint32_t row[kUnpackEach], v[kUnpackEach], word[kUnpackEach];
    float s[kUnpackEach];
#pragma unroll
    for (int i = 0; i < kUnpackEach; ++i) {
        const uint32_t t = min((blockIdx.x * kUnpackEach + i) * 256u + threadIdx.x, a.units - 1);
        row[i] = a.per_row.quotient(t);
        v[i] = t - row[i] * a.per_row.d;
        const uint8_t* p = a.packed + row[i] * a.p_stride;
        if constexpr (E == 8) word[i] = reinterpret_cast<const U32U*>(p)[v[i]].v;
        else word[i] = reinterpret_cast<const U16U*>(p)[v[i]].v;
        s[i] = load_scale(static_cast<const ST*>(a.scales) + row[i] * a.s_stride + (v[i] >> a.lane_shift));
    }
#pragma unroll
    for (int i = 0; i < kUnpackEach; ++i) {
        if ((blockIdx.x * kUnpackEach + i) * 256u + threadIdx.x >= a.units) return;
        T* out = static_cast<T*>(a.out) + static_cast<int64_t>(row[i]) * a.k;
        const int at = static_cast<int>(v[i] * E);
        typename Unit<T>::type o;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            float p = static_cast<float>(code4(word[i], e)) * s[i];
            if constexpr (std::is_same<T, _Float16>::value) asm("" : "+v"(p));      // keeps the product's own rounding: else it is fused with the conversion
            o[e] = static_cast<T>(p);
        }
        if (at + E <= a.k) {
            *reinterpret_cast<typename Unit<T>::type*>(out + at) = o;
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (at + e < a.k) out[at + e] = o[e];
        }
    }
}

// ---- products of a few rows with 4-bit weights, on the matrix cores ----
//
//   y[m][n] = x_scale[m] * sum over groups g of scale[n][g] * sum over k in g of q[n][k] x[m][k]
//
// Rows of x are the A operand of 16 x 16 matrix instructions, 16 outputs n the B operand.  A wavefront takes 128 columns of 16
// outputs at a time: lane (n, quarter) loads 16 bytes of row n, so codes go from memory to the matrix cores through registers
// alone.  With groups of 128 any order of k within them does; with smaller ones the words are transposed between the
// quarters (four instructions for four words), so that an instruction's columns lie in one group and its sums can be scaled on
// their own.  The rows are brought into the order in which codes come out of their words.
//
// Two kernels, one for up to four rows, which is bound by the codes' way from memory, and one for more.  In both a product with a code is exact:
// int8 rows meet codes as bytes, and a group's sums are whole numbers; floating rows meet codes as 16-bit floating-point
// numbers (widen_word()), and their sums are fp32, of the terms themselves: what a column adds to the error goes with its own term, and
// a code of 0 makes it nothing.

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
    int64_t x_stride;           // elements
    uint32_t p_stride, s_stride; // bytes, from row to row of the codes and of the scales
    int rows;
    int n;
    int k;
    int row_bytes;              // codes of a row that exist: whole groups
    int groups;
    int out_type;               // PRIME_F32, PRIME_BF16 or PRIME_F16
    int chunk_quads;            // stretches of 512 columns of x that LDS holds at a time
    int tiles;                  // 16 outputs each
    int sets;                   // rounds of tiles a row tile takes: ceil(tiles / tiles a workgroup takes at a time)
    int split_shift;            // log2 of the wavefronts that share a tile's columns
};

// new[j] of quarter q = old[q] of quarter j
__device__ __forceinline__ void transpose_quarters(u32x4& w) {
    const auto a = __builtin_amdgcn_permlane32_swap(w[0], w[2], false, false);
    const auto b = __builtin_amdgcn_permlane32_swap(w[1], w[3], false, false);
    const auto c = __builtin_amdgcn_permlane16_swap(a[0], b[0], false, false);
    const auto d = __builtin_amdgcn_permlane16_swap(a[1], b[1], false, false);
    w = u32x4{c[0], c[1], d[0], d[1]};
}

// Eight codes of a word as 16-bit numbers with their sign, in the order 0 4 1 5 2 6 3 7: bf16 holds q / 16, fp16 q, both exactly.  (Beside an
// offset, as 24 + q, a word takes eight instructions instead of thirteen and nine.  But then a column passes through the sums at up to 24 times
// its size whatever its code is, and what a large one leaves there as rounding hides the others, and beyond 2^116 as infinity all of them.  64 x
// 8192 x 22528 took 74 us so, with the offset's own sums read from LDS, and takes 70.)
template <bool BF16>
__device__ __forceinline__ u32x4 widen_word(uint32_t w) {
    if constexpr (BF16) {
        uint32_t odd = w >> 4;
        asm("" : "+v"(odd));                                // keeps the one shift: its bytes are then operands as they are
        float f[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f[2 * i] = __builtin_amdgcn_cvt_off_f32_i4(w >> (8 * i) & 0xff);
            f[2 * i + 1] = __builtin_amdgcn_cvt_off_f32_i4(odd >> (8 * i) & 0xff);
        }
        auto pair = [&](int e) { return __builtin_amdgcn_perm(__float_as_uint(f[e + 4]), __float_as_uint(f[e]), 0x07060302u); };
        return u32x4{pair(0), pair(1), pair(2), pair(3)};
    } else {
        typedef _Float16 __attribute__((ext_vector_type(2))) half2;
        // 1024 + u or 1024 + 16 u with u = q + 8, then q
        auto low = [](uint32_t v) {
            const half2 h = __builtin_bit_cast(half2, (v & 0x000f000fu) ^ 0x64086408u) + half2{static_cast<_Float16>(-1032.0f), static_cast<_Float16>(-1032.0f)};
            return __builtin_bit_cast(uint32_t, h);
        };
        auto high = [](uint32_t v) {
            const half2 by{static_cast<_Float16>(0.0625f), static_cast<_Float16>(0.0625f)}, off{static_cast<_Float16>(-72.0f), static_cast<_Float16>(-72.0f)};
            return __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(__builtin_bit_cast(half2, (v & 0x00f000f0u) ^ 0x64806480u), by, off));
        };
        const uint32_t v = w >> 8;
        return u32x4{low(w), high(w), low(v), high(v)};
    }
}
// The codes in the lower or upper halves of a word's bytes as bytes with their sign: 16 q in an instruction or two, or q in two more.
template <bool SIXTEEN>
__device__ __forceinline__ uint32_t low_codes(uint32_t w) {
    if constexpr (SIXTEEN) return (w << 4) & 0xf0f0f0f0u;
    else return (((w & 0x0f0f0f0fu) ^ 0x08080808u) + 0x78787878u) ^ 0x80808080u;      // q + 8, q + 128: no byte carries
}
template <bool SIXTEEN>
__device__ __forceinline__ uint32_t high_codes(uint32_t w) {
    if constexpr (SIXTEEN) return w & 0xf0f0f0f0u;
    else return low_codes<false>(w >> 4);
}
// What products with widened codes are to be multiplied by.
template <typename XT> constexpr float kWidenedUnit = std::is_same<XT, _Float16>::value ? 1.0f : 16.0f;
template <typename XT>
__device__ __forceinline__ f32x4 product(u32x4 rows, u32x4 codes, f32x4 c) {
    if constexpr (std::is_same<XT, _Float16>::value)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, rows), __builtin_bit_cast(f16x8, codes), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, rows), __builtin_bit_cast(bf16x8, codes), c, 0, 0, 0);
}

// Scales of the groups of 512 columns of one output, as they are stored.
template <typename ST, int GS> struct QuadScales {
    static constexpr int kCount = 4 << (7 - GS);
    typedef ST vec __attribute__((ext_vector_type(kCount), aligned(sizeof(ST))));
    vec v;
    __device__ __forceinline__ void load(const ST* p) { v = *reinterpret_cast<const vec*>(p); }
    __device__ __forceinline__ void load_some(const ST* p, int there) {
#pragma unroll
        for (int i = 0; i < kCount; ++i) v[i] = i < there ? p[i] : static_cast<ST>(0.0f);
    }
    __device__ __forceinline__ float at(int i) const { return static_cast<float>(v[i]); }
};

__device__ __forceinline__ void store_product(const MatvecArgs& a, int64_t at, float v) {
    if (a.out_type == PRIME_F32) static_cast<float*>(a.out)[at] = v;
    else if (a.out_type == PRIME_BF16) static_cast<__bf16*>(a.out)[at] = static_cast<__bf16>(v);
    else static_cast<_Float16*>(a.out)[at] = static_cast<_Float16>(v);
}

template <typename XT> constexpr int kPlanes = sizeof(XT) == 4 ? 3 : 1;

__device__ __forceinline__ uint32_t pair16(uint32_t lo, uint32_t hi) { return (lo & 0xffffu) | hi << 16; }

// Eight columns of a row as the A operand wants them: 16-bit values in the order 0 4 1 5 2 6 3 7 (fp32 in three bf16 planes, each the
// leading eight bits of what the ones before leave: together the value, but for what lies below bf16's smallest step, 2^-133), bytes in
// the order 0 2 4 6 1 3 5 7.
template <typename XT> struct Frag { typedef u32x4 type; };
template <> struct Frag<int8_t> { typedef u32x2 type; };

template <typename XT>
__device__ __forceinline__ void rows8(const XT* __restrict__ row, int64_t i, int n, typename Frag<XT>::type (&out)[kPlanes<XT>]) {
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
        typename Eight<XT>::type t;
        if (i < n) {
            t = take8(row, static_cast<int>(i), n);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) t[e] = static_cast<XT>(0.0f);
        }
        typedef XT __attribute__((ext_vector_type(8))) eight;
        const u32x4 b = __builtin_bit_cast(u32x4, static_cast<eight>(t));
        // 0 4, 1 5, 2 6, 3 7
        out[0] = u32x4{__builtin_amdgcn_perm(b[2], b[0], 0x05040100u), __builtin_amdgcn_perm(b[2], b[0], 0x07060302u),
                       __builtin_amdgcn_perm(b[3], b[1], 0x05040100u), __builtin_amdgcn_perm(b[3], b[1], 0x07060302u)};
    } else {
        float v[8];
        if (i < n) {
            load8(row, static_cast<int>(i), n, v);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = 0.0f;
        }
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

// ---- up to four rows ----
// The rows stay in LDS and the codes pass by.  Rows are taken as they are; the three planes of an fp32 row are three rows of the A operand, so
// that one matrix instruction takes them all, and are added at a group's end, the smallest first.  (Floating rows were fixed point under
// the largest of 128 columns before, four int8 digits each: 1 x 8192 x 128000 bf16 took 93 us instead of 100 in a row of calls, 4 x 8192 x 22528
// 35 instead of 30.  But columns far below that largest were lost, also where its code is 0.)
//
// Bound by memory from a few thousand outputs up: 1 x 8192 x 128000 int8 92 us (5.9 TB/s; with the products taken out and the loads left
// in 97, with loads that cover whole lines instead of 64 bytes of 16 rows 90), bf16 107 to 114 (92 without the products; 61 % of each SIMD's
// cycles are vector and 15 % matrix instructions).  Words of a group in sums of their own, so that no product waits for the one before, cost
// 2 % there.  Small products are a launch and two trips to memory: 1 x 2048 x 2048 4.0 us, 1 x 4096 x 4096 4.8 us.

// Bytes of a row's 128 columns in LDS: [quarter][word of a lane][plane][eight columns], so that the lanes of a quarter, which read the planes
// of one word side by side, read consecutive bytes.  Rows lie 16 (fp32: 64) bytes off the banks' period.
template <typename XT> constexpr int kFewBlock = 128 * static_cast<int>(sizeof(typename Frag<XT>::type)) / 8 * kPlanes<XT>;
template <typename XT> constexpr int kFewPad = sizeof(XT) == 4 ? 64 : 16;

template <typename XT, typename ST, int GS>
__global__ __launch_bounds__(512) void matvec4_few_kernel(MatvecArgs a) {
    constexpr bool kInt = sizeof(XT) == 1;
    constexpr int NG = 1 << (7 - GS);
    constexpr int kBlock = kFewBlock<XT>, P = kPlanes<XT>, kWord = static_cast<int>(sizeof(typename Frag<XT>::type)) * P;
    extern __shared__ __align__(16) uint8_t few_lds[];
    __shared__ float part[2][8 * 64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), quarter = lane >> 4, v16 = lane & 15;
    const int split = 1 << a.split_shift, kpart = wave & (split - 1);
    const int side = static_cast<int>(blockDim.x >> 6) >> a.split_shift;                    // tiles at a time
    const int stride = gridDim.x, set0 = blockIdx.x, rows = a.rows;
    const int quads = (a.k + 511) >> 9;
    const int row_stride = a.chunk_quads * 4 * kBlock + kFewPad<XT>;
    // a lane's row of the A operand: plane v16 & 3 of row v16 >> 2 (one plane: the row, four times).  Rows and planes that do not exist repeat
    // the last one; their sums are dropped
    const int my_row = min(v16 >> 2, rows - 1);
    const uint8_t* mine = few_lds + my_row * row_stride + quarter * (4 * kWord) + (P > 1 ? min(v16 & 3, P - 1) * 16 : 0);
    const uint8_t* scales = static_cast<const uint8_t*>(a.scales);
    u32x4 w[4], w2[4];
    QuadScales<ST, GS> s, s2;
    auto fetch = [&](int set, int q, u32x4 (&to)[4], QuadScales<ST, GS>& sc) {
        const uint32_t n = min((set * side + (wave >> a.split_shift)) * 16 + v16, a.n - 1);
        typedef u32x4 __attribute__((aligned(1))) u32x4u;
        const uint8_t* p = a.packed + (static_cast<uint64_t>(n) * a.p_stride + static_cast<uint32_t>(q * 256 + quarter * 16));
        const ST* sp = reinterpret_cast<const ST*>(scales + static_cast<uint64_t>(n) * a.s_stride) + q * (4 * NG);
        if ((q + 1) * 256 <= a.row_bytes) {
#pragma unroll
            for (int u = 0; u < 4; ++u) to[u] = *reinterpret_cast<const u32x4u*>(p + 64 * u);
            sc.load(sp);
        } else {
#pragma unroll
            for (int u = 0; u < 4; ++u)
                to[u] = q * 256 + u * 64 + quarter * 16 < a.row_bytes ? *reinterpret_cast<const u32x4u*>(p + 64 * u) : u32x4{0, 0, 0, 0};
            sc.load_some(sp, a.groups - q * (4 * NG));
        }
    };
    const XT* x = static_cast<const XT*>(a.x);
    // Where a wavefront starts in its tile's columns: tiles side by side start at different ones, else all rows of
    // a matrix whose row length is a power of two would be read at the same offset at a time, from the same memory channels.
    const bool whole = a.chunk_quads >= quads;
    const int own = (quads - kpart + split - 1) >> a.split_shift;
    auto start = [&](int set) { return whole ? kpart + ((set * side + (wave >> a.split_shift)) % own << a.split_shift) : kpart; };
    int at = start(set0);
    fetch(set0, at, w, s);
    int turn = 0;
    for (int set = set0; set < a.sets; set += stride, turn ^= 1) {
        float y = 0.0f;
        for (int first = 0; first < quads; first += a.chunk_quads) {
            const int held = min(a.chunk_quads, quads - first);
            if (set == set0 || held < quads) {
                if (set != set0 || first) __syncthreads();
                // rows of x to LDS: eight columns a lane, put where the lane that multiplies them will look
                for (int i = threadIdx.x; i < rows * held * 64; i += blockDim.x) {
                    const int m = i / (held * 64), c = i - m * (held * 64);
                    typename Frag<XT>::type v[P];
                    rows8(x + m * a.x_stride, static_cast<int64_t>(first) * 512 + c * 8, a.k, v);
                    // eighth `in` of a block: with groups of 128 a quarter's four lie side by side, else they are a quarter apart
                    const int in = c & 15, q = GS == 7 ? in >> 2 : in & 3, j = GS == 7 ? in & 3 : in >> 2;
                    uint8_t* to = few_lds + m * row_stride + (c >> 4) * kBlock + (q * 4 + j) * kWord;
#pragma unroll
                    for (int p = 0; p < P; ++p) reinterpret_cast<typename Frag<XT>::type*>(to)[p] = v[p];
                }
                __syncthreads();
            }
            for (int i = kpart; i < held; i += split) {
                const int q = at - first;
                const bool more = first + i + split < quads;
                const int next_set = more ? set : min(set + stride, a.sets - 1);
                at = !more ? start(next_set) : at + split < quads ? at + split : kpart;
                fetch(next_set, at, w2, s2);
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    u32x4 c = w[u];
                    if constexpr (GS < 7) transpose_quarters(c);
                    if constexpr (kInt) {
                        // the codes count 16 times, which is taken off a group's sum, exactly, before it meets the scales: at the
                        // end, sums could leave fp32 that the rows' scales bring back, and the rows' smallest scales would lose bits
                        i32x4 acc[NG];
#pragma unroll
                        for (int g = 0; g < NG; ++g) acc[g] = i32x4{0, 0, 0, 0};
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            const u32x4 xa = *reinterpret_cast<const u32x4*>(mine + (q * 4 + u) * kBlock + j * 16);
                            const u32x4 b{low_codes<true>(c[2 * j]), high_codes<true>(c[2 * j]), low_codes<true>(c[2 * j + 1]), high_codes<true>(c[2 * j + 1])};
                            if constexpr (GS == 5) {
                                const u32x2 a0{xa[0], xa[1]}, a1{xa[2], xa[3]}, b0{b[0], b[1]}, b1{b[2], b[3]};
                                acc[2 * j] = __builtin_amdgcn_mfma_i32_16x16x32_i8(__builtin_bit_cast(long, a0), __builtin_bit_cast(long, b0), acc[2 * j], 0, 0, 0);
                                acc[2 * j + 1] = __builtin_amdgcn_mfma_i32_16x16x32_i8(__builtin_bit_cast(long, a1), __builtin_bit_cast(long, b1), acc[2 * j + 1], 0, 0, 0);
                            } else {
                                const int g = GS == 6 ? j : 0;
                                acc[g] = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, xa), __builtin_bit_cast(i32x4, b), acc[g], 0, 0, 0);
                            }
                        }
#pragma unroll
                        for (int g = 0; g < NG; ++g) y = fmaf(static_cast<float>(acc[g][0]) * 0.0625f, s.at(u * NG + g), y);
                    } else {
                        f32x4 acc[NG];
#pragma unroll
                        for (int g = 0; g < NG; ++g) acc[g] = f32x4{0, 0, 0, 0};
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const u32x4 xa = *reinterpret_cast<const u32x4*>(mine + (q * 4 + u) * kBlock + j * kWord);
                            acc[j * NG / 4] = product<XT>(xa, widen_word<!std::is_same<XT, _Float16>::value>(c[j]), acc[j * NG / 4]);
                        }
#pragma unroll
                        for (int g = 0; g < NG; ++g) y = fmaf(P > 1 ? (acc[g][2] + acc[g][1]) + acc[g][0] : acc[g][0], s.at(u * NG + g), y);
                    }
                }
#pragma unroll
                for (int u = 0; u < 4; ++u) w[u] = w2[u];
                s = s2;
            }
        }
        const int n = (set * side + (wave >> a.split_shift)) * 16 + v16;
        if (split > 1) {
            // the wavefronts' sums, added in their order; two buffers in turn, so that one barrier a set is enough
            part[turn][wave * 64 + lane] = y;
            __syncthreads();
            if (kpart) continue;
            for (int p = 1; p < split; ++p) y += part[turn][(wave + p) * 64 + lane];
        }
        if (quarter < rows && n < a.n) store_product(a, static_cast<int64_t>(quarter) * a.n + n, y * (kInt ? a.x_scales[quarter] : kWidenedUnit<XT>));
    }
}

// ---- more rows: 16, 32 or 64 at a time ----
// Here the matrix cores' work grows with the rows: fp32 rows are three bf16 rows.  The rows stay where they are and the codes pass by: the
// eight wavefronts of a workgroup split the columns, each holds its share of the rows in registers for all of the workgroup's outputs, and
// only codes and scales are loaded in the loop, a round of outputs ahead.  The wavefronts' sums of a round meet in LDS.  Rows too
// long for the registers take several visits, whose sums LDS keeps.
// 16 x 8192 x 22528 bf16 35 us, 64 rows 70 us (fp32 46 and 117, int8 64 rows 63).  Up to 16 rows are bound by the loads' way through few, large
// rounds and by the products (without the products 27 us, without the loads 24), 64 rows by the products and the sums' way through LDS
// (without the products 41 us, without the loads 67, without the sums' way 61; of each SIMD's cycles 41 % are vector and 16 % matrix
// instructions).  Measured before the codes were widened with their sign, when 64 rows took 74 us, and neither kept: three rounds in flight in
// registers of their own (74 to 78 us, products of 2048 columns twice the time), workgroups that begin at different columns (73 to 75).  One
// barrier a round was worth 3 us.  The first form kept the rows in LDS, with a barrier for every 256 columns: each stretch waited for
// its loads, 64 x 8192 x 22528 91 us, 7 x 5604 x 11263 fp16 37 us against 18 (now 16).

typedef float f32x2 __attribute__((ext_vector_type(2)));
// f(0), f(1), ... with the index a constant: registers are indexed by it.
template <int N, typename F, int... I>
__device__ __forceinline__ void each_of(F&& f, std::integer_sequence<int, I...>) { (f(std::integral_constant<int, I>{}), ...); }
template <int N, typename F>
__device__ __forceinline__ void each(F&& f) { each_of<N>(static_cast<F&&>(f), std::make_integer_sequence<int, N>{}); }

// MT tiles of 16 rows; B blocks of 128 columns a wavefront; NT tiles of 16 outputs a round.
template <typename XT, typename ST, int GS, int MT, int B, int NT>
__global__ __launch_bounds__(512) void matvec4_many_kernel(MatvecArgs a) {
    constexpr bool kInt = sizeof(XT) == 1;
    constexpr int P = kPlanes<XT>, NG = 1 << (7 - GS), kRows = 16 * MT;
    constexpr int RUN = B < 2 ? B : 2;                       // blocks side by side: whole lines of codes
    constexpr int kPart = NT * MT * 256;                     // values of a round
    typedef typename Frag<XT>::type frag;
    typedef ST __attribute__((ext_vector_type(RUN * NG), aligned(sizeof(ST)))) run_scales;
    // two buffers in turn need one barrier a round; what 64 KiB do not hold twice has one and two
    constexpr int kBuffers = kPart > 1024 ? 1 : 2;
    __shared__ __align__(16) float part_of[kBuffers][8 * kPart];
    int turn = 0;
    extern __shared__ __align__(16) float kept[];            // [own round][value], for rows that take several visits
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), quarter = lane >> 4, v16 = lane & 15;
    const int per_row_tile = gridDim.x / ((a.rows + kRows - 1) / kRows);
    const int row0 = blockIdx.x / per_row_tile * kRows, set0 = blockIdx.x % per_row_tile;
    const int rows = min(a.rows - row0, kRows);
    const int blocks = (a.k + 127) >> 7, visits = (blocks + 8 * B - 1) / (8 * B);
    const XT* x = static_cast<const XT*>(a.x) + static_cast<int64_t>(row0) * a.x_stride;
    const uint8_t* scales = static_cast<const uint8_t*>(a.scales);
    auto block_of = [&](int visit, int u) { return visit * 8 * B + u / RUN * (8 * RUN) + wave * RUN + u % RUN; };
    auto fetch = [&](int visit, int set, u32x4 (&w)[NT][B], run_scales (&s)[NT][B / RUN]) {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const uint32_t n = min((set * NT + t) * 16 + v16, a.n - 1);
            const uint8_t* codes = a.packed + (static_cast<uint64_t>(n) * a.p_stride + quarter * 16);
            const ST* sp = reinterpret_cast<const ST*>(scales + static_cast<uint64_t>(n) * a.s_stride);
#pragma unroll
            for (int r = 0; r < B / RUN; ++r) {
                typedef u32x4 __attribute__((aligned(1))) u32x4u;
                const int b = block_of(visit, r * RUN);
                if ((b + RUN) * 64 <= a.row_bytes) {
#pragma unroll
                    for (int u = 0; u < RUN; ++u) w[t][r * RUN + u] = *reinterpret_cast<const u32x4u*>(codes + static_cast<int64_t>(b + u) * 64);
                    s[t][r] = *reinterpret_cast<const run_scales*>(sp + static_cast<int64_t>(b) * NG);
                } else {
                    // behind the row's end codes and scales are zero
#pragma unroll
                    for (int u = 0; u < RUN; ++u)
                        w[t][r * RUN + u] = (b + u) * 64 + quarter * 16 < a.row_bytes ? *reinterpret_cast<const u32x4u*>(codes + static_cast<int64_t>(b + u) * 64) : u32x4{0, 0, 0, 0};
#pragma unroll
                    for (int g = 0; g < RUN * NG; ++g) s[t][r][g] = b * NG + g < a.groups ? sp[static_cast<int64_t>(b) * NG + g] : static_cast<ST>(0.0f);
                }
            }
        }
    };
    u32x4 w[NT][B], w2[NT][B];
    run_scales s[NT][B / RUN], s2[NT][B / RUN];
    fetch(0, set0, w, s);
    for (int visit = 0; visit < visits; ++visit) {
        // this wavefront's columns of the rows; rows that do not exist repeat the last one, their sums are dropped
        frag xa[B][P][MT][4];
        each<B>([&](auto uc) {
            constexpr int u = decltype(uc)::value;
            const int64_t b = block_of(visit, u);
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    frag f[P];
                    rows8(x + static_cast<int64_t>(min(m * 16 + v16, rows - 1)) * a.x_stride, b * 128 + (GS == 7 ? quarter * 4 + j : j * 4 + quarter) * 8, a.k, f);
#pragma unroll
                    for (int p = 0; p < P; ++p) xa[u][p][m][j] = f[p];
                }
        });
        int own = 0;
        for (int set = set0; set < a.sets; set += per_row_tile, ++own) {
            const bool more = set + per_row_tile < a.sets;
            fetch(more ? visit : min(visit + 1, visits - 1), more ? set + per_row_tile : set0, w2, s2);
            float* part = part_of[turn & (kBuffers - 1)];
            ++turn;
            float y[NT][MT][4];
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int m = 0; m < MT; ++m)
#pragma unroll
                    for (int i = 0; i < 4; ++i) y[t][m][i] = 0.0f;
            each<B>([&](auto uc) {
                constexpr int u = decltype(uc)::value;
                if (block_of(visit, u) >= blocks) return;      // the same for the whole wavefront
                each<NT>([&](auto tc) {
                    constexpr int t = decltype(tc)::value;
                    u32x4 v = w[t][u];
                    if constexpr (GS < 7) transpose_quarters(v);
                    each<NG>([&](auto gc) {
                        constexpr int g = decltype(gc)::value, kSteps = 4 / NG;      // words of a lane in a group
                        const float f = static_cast<float>(s[t][u / RUN][u % RUN * NG + g]);
                        if constexpr (kInt) {
                            // 16 q costs a product more for each of 4 MT sums, q four instructions more for each word: 64 rows in groups of 32 take 78 us
                            // with q (8192 x 22528, fp32 scales) and 84 with 16 q
                            constexpr bool kSixteen = MT <= kSteps;
                            i32x4 acc[MT];
#pragma unroll
                            for (int m = 0; m < MT; ++m) acc[m] = i32x4{0, 0, 0, 0};
                            if constexpr (GS == 5) {
                                const u32x2 cb{low_codes<kSixteen>(v[g]), high_codes<kSixteen>(v[g])};
#pragma unroll
                                for (int m = 0; m < MT; ++m)
                                    acc[m] = __builtin_amdgcn_mfma_i32_16x16x32_i8(__builtin_bit_cast(long, xa[u][0][m][g]), __builtin_bit_cast(long, cb), acc[m], 0, 0, 0);
                            } else {
                                each<kSteps / 2>([&](auto jc) {
                                    constexpr int j = g * kSteps + 2 * decltype(jc)::value;
                                    const u32x4 cb{low_codes<kSixteen>(v[j]), high_codes<kSixteen>(v[j]), low_codes<kSixteen>(v[j + 1]), high_codes<kSixteen>(v[j + 1])};
#pragma unroll
                                    for (int m = 0; m < MT; ++m) {
                                        const frag lo = xa[u][0][m][j], hi = xa[u][0][m][j + 1];
                                        acc[m] = __builtin_amdgcn_mfma_i32_16x16x64_i8(i32x4{static_cast<int>(lo[0]), static_cast<int>(lo[1]), static_cast<int>(hi[0]), static_cast<int>(hi[1])},
                                                                                       __builtin_bit_cast(i32x4, cb), acc[m], 0, 0, 0);
                                    }
                                });
                            }
#pragma unroll
                            for (int m = 0; m < MT; ++m)
#pragma unroll
                                for (int i = 0; i < 4; ++i) y[t][m][i] = fmaf(static_cast<float>(acc[m][i]) * (kSixteen ? 0.0625f : 1.0f), f, y[t][m][i]);
                        } else {
                            f32x4 acc[MT];
#pragma unroll
                            for (int m = 0; m < MT; ++m) acc[m] = f32x4{0, 0, 0, 0};
                            each<kSteps>([&](auto jc) {
                                constexpr int j = g * kSteps + decltype(jc)::value;
                                const u32x4 cb = widen_word<!std::is_same<XT, _Float16>::value>(v[j]);
#pragma unroll
                                for (int p = 0; p < P; ++p)
#pragma unroll
                                    for (int m = 0; m < MT; ++m) acc[m] = product<XT>(xa[u][p][m][j], cb, acc[m]);
                            });
#pragma unroll
                            for (int m = 0; m < MT; ++m)
#pragma unroll
                                for (int i = 0; i < 4; ++i) y[t][m][i] = fmaf(acc[m][i], f, y[t][m][i]);
                        }
                    });
                });
            });
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int m = 0; m < MT; ++m)
                    *reinterpret_cast<f32x4*>(part + wave * kPart + ((t * MT + m) * 64 + lane) * 4) = f32x4{y[t][m][0], y[t][m][1], y[t][m][2], y[t][m][3]};
            __syncthreads();
            // the wavefronts' sums, added in their order, to those of the visits before
            for (int i = threadIdx.x; i < kPart / 2; i += 512) {
                f32x2 v = reinterpret_cast<const f32x2*>(part)[i];
#pragma unroll
                for (int q = 1; q < 8; ++q) v += reinterpret_cast<const f32x2*>(part)[q * (kPart / 2) + i];
                if (visits > 1) {
                    f32x2* keep = reinterpret_cast<f32x2*>(kept) + own * (kPart / 2) + i;
                    if (visit) v += *keep;
                    if (visit + 1 < visits) {
                        *keep = v;
                        continue;
                    }
                }
                const int l = i >> 1 & 63, m = (i >> 7) % MT, t = (i >> 7) / MT;
                const int row = m * 16 + (l >> 4) * 4 + (i & 1) * 2, n = (set * NT + t) * 16 + (l & 15);
                if (n >= a.n) continue;
                const int64_t at = static_cast<int64_t>(row0 + row) * a.n + n;
#pragma unroll
                for (int r = 0; r < 2; ++r)
                    if (row + r < rows) store_product(a, at + static_cast<int64_t>(r) * a.n, v[r] * (kInt ? a.x_scales[row0 + row + r] : kWidenedUnit<XT>));
            }
            if constexpr (kBuffers == 1) __syncthreads();
#pragma unroll
            for (int t = 0; t < NT; ++t) {
#pragma unroll
                for (int u = 0; u < B; ++u) w[t][u] = w2[t][u];
#pragma unroll
                for (int r = 0; r < B / RUN; ++r) s[t][r] = s2[t][r];
            }
        }
    }
}
