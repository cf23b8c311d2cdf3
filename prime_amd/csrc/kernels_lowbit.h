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

struct MatvecArgs {
    const void* x;
    const float* x_scales;      // one a row with int8 rows, else null
    const uint8_t* packed;
    const void* scales;
    void* out;                  // dense rows of n
    int64_t x_stride, p_stride, s_stride;
    int rows;
    int64_t n;
    int k;
    int group_shift;
};

template <typename T> __device__ __forceinline__ float to_float(T v) { return static_cast<float>(v); }

// A wavefront per output, four rows at a time; a group's lanes join their sums before its scale is applied.
template <typename XT, typename ST, typename OT>
__global__ __launch_bounds__(256) void matvec4_kernel(MatvecArgs a) {
    const int64_t n = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
    if (n >= a.n) return;
    const int lane = threadIdx.x & 63;
    const U32U* codes = reinterpret_cast<const U32U*>(a.packed + n * a.p_stride);
    const ST* scales = static_cast<const ST*>(a.scales) + n * a.s_stride;
    for (int m0 = 0; m0 < a.rows; m0 += 4) {
        float acc[4] = {0, 0, 0, 0};
        for (int64_t base = 0; base < a.k; base += 512) {
            const int64_t i = base + lane * 8;
            const uint32_t word = i < a.k ? codes[i >> 3].v : 0u;
            const float s = i < a.k && (lane * 8 & ((1 << a.group_shift) - 1)) == 0 ? load_scale(scales + (i >> a.group_shift)) : 0.0f;
            for (int m = 0; m < 4 && m0 + m < a.rows; ++m) {
                const XT* row = static_cast<const XT*>(a.x) + static_cast<int64_t>(m0 + m) * a.x_stride;
                float part = 0.0f;
                for (int e = 0; e < 8 && i + e < a.k; ++e) part = fmaf(static_cast<float>(code4(word, e)), to_float(row[i + e]), part);
                for (int d = 1 << (a.group_shift - 4); d >= 1; d >>= 1) part += __shfl_xor(part, d, 64);
                if ((lane * 8 & ((1 << a.group_shift) - 1)) == 0 && i < a.k) acc[m] = fmaf(part, s, acc[m]);
            }
        }
        for (int m = 0; m < 4 && m0 + m < a.rows; ++m) {
            const float y = wave_sum_all(acc[m]);
            if (lane == 0) static_cast<OT*>(a.out)[static_cast<int64_t>(m0 + m) * a.n + n] = static_cast<OT>(a.x_scales ? y * a.x_scales[m0 + m] : y);
        }
    }
}
