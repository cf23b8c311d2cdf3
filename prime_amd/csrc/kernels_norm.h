// Root-mean-square norm of rows with the residual's addition and an 8-bit output with one scale per row, and
// the gradients of its input and weight.
//
//   h = x + r rounded to the rows' type (the stream as later blocks read it), or x itself
//   z = fl32(h w),  a = max |z|,  s = fl32(a / top)          top = 127 (int8) or 448 (e4m3)
//   code = the integer (e4m3 number) nearest z / s, ties to even
//   inv = 1 / sqrt(sum h^2 / dim + eps),  scale = s inv      so that code * scale stands for h inv w
//
// The root mean square cancels out of the codes, so the sum of squares and the maximum are taken in one visit and
// nothing waits for the other.  Codes are exact: see nearest_int().  Sums of squares are fp64 (a square of an fp32
// value overflows fp32; at 8 bytes of traffic an element the fp64 additions cost nothing).
// A row that holds a value that is not finite, or whose product with the weight is not, gets scale NaN and codes 0.
//
// Bound by memory: 16384 x 4096 bf16 with residual 74 us (6.35 TB/s; a plain copy reaches 6.8), its gradient with that of the sum 89 us
// (6.0 TB/s, of which 4 us the second launch that adds up the weight's gradient).  A row is one visit: from registers, a
// workgroup a row from 1025 elements up (four rows a workgroup below), and a workgroup that ends after its row, so that no wavefront
// waits for its own stores.  Eight roundings to codes share one test for borders: one at a time they took 96 us instead of 82.
//
// Included by prime_hip.hip inside its anonymous namespace; not a translation unit of its own.

// Eight consecutive elements of a row, at element alignment (a row of odd length starts anywhere).
template <typename T> struct Eight;
template <> struct Eight<float> { typedef float type __attribute__((ext_vector_type(8), aligned(4))); };
template <> struct Eight<__bf16> { typedef __bf16 type __attribute__((ext_vector_type(8), aligned(2))); };
template <> struct Eight<_Float16> { typedef _Float16 type __attribute__((ext_vector_type(8), aligned(2))); };
struct __attribute__((packed, aligned(1))) U64U { uint32_t lo, hi; };

// Elements i .. i + 7 of a row of n as they are, zero behind its end.  ONCE: nobody reads them again soon (a hinted load
// leaves room in the caches for what is).
template <typename T, bool ONCE = false>
__device__ __forceinline__ typename Eight<T>::type take8(const T* __restrict__ row, int i, int n) {
    typename Eight<T>::type t;
    if (i + 8 <= n) {
        const typename Eight<T>::type* p = reinterpret_cast<const typename Eight<T>::type*>(row + i);
        if constexpr (ONCE) t = __builtin_nontemporal_load(p);
        else t = *p;
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) t[e] = i + e < n ? row[i + e] : static_cast<T>(0.0f);
    }
    return t;
}

// The same as floats.
template <typename T>
__device__ __forceinline__ void load8(const T* __restrict__ row, int i, int n, float (&v)[8]) {
    const typename Eight<T>::type t = take8(row, i, n);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = static_cast<float>(t[e]);
}

// The `lane`-th eight elements of a row, dealt to lanes as the memory likes it: 16-bit elements eight side by side; fp32 elements
// four side by side, twice (a wavefront's two loads then cover whole lines of 1 KiB each, where eight side by side
// would have each load touch every second 16 bytes of 2 KiB).
template <typename T>
__device__ __forceinline__ void place8(int lane, int (&at)[2]) {
    if constexpr (sizeof(T) == 4) {
        at[0] = (lane >> 6) * 512 + (lane & 63) * 4;
        at[1] = at[0] + 256;
    } else {
        at[0] = lane * 8;
        at[1] = at[0] + 4;
    }
}
typedef float __attribute__((ext_vector_type(4), aligned(4))) four_floats;
struct __attribute__((packed, aligned(1))) U32Any { uint32_t v; };

template <bool ONCE, typename T>
__device__ __forceinline__ typename Eight<T>::type row_take8(const T* __restrict__ row, int lane, int n) {
    if constexpr (sizeof(T) == 4) {
        typename Eight<T>::type t;
        int at[2];
        place8<T>(lane, at);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            if (at[h] + 4 <= n) {
                const four_floats* p = reinterpret_cast<const four_floats*>(row + at[h]);
                four_floats v;
                if constexpr (ONCE) v = __builtin_nontemporal_load(p);
                else v = *p;
#pragma unroll
                for (int e = 0; e < 4; ++e) t[4 * h + e] = v[e];
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) t[4 * h + e] = at[h] + e < n ? row[at[h] + e] : 0.0f;
            }
        }
        return t;
    } else {
        return take8<T, ONCE>(row, lane * 8, n);
    }
}
// A norm's weight for the elements that row_take8<XT> gives: read again by every row.
template <typename XT, typename WT>
__device__ __forceinline__ void weight8(const WT* __restrict__ weight, int lane, int n, float (&w)[8]) {
    if constexpr (sizeof(XT) == 4 || sizeof(WT) == 2) {
        const typename Eight<WT>::type t = row_take8<false>(weight, lane, n);
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e] = static_cast<float>(t[e]);
    } else {
        load8(weight, lane * 8, n, w);
    }
}

template <typename T>
__device__ __forceinline__ void row_store8(T* __restrict__ row, int lane, int n, const float (&v)[8]) {
    if constexpr (sizeof(T) == 4) {
        int at[2];
        place8<T>(lane, at);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            if (at[h] + 4 <= n) {
                *reinterpret_cast<four_floats*>(row + at[h]) = four_floats{v[4 * h], v[4 * h + 1], v[4 * h + 2], v[4 * h + 3]};
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (at[h] + e < n) row[at[h] + e] = v[4 * h + e];
            }
        }
    } else {
        const int i = lane * 8;
        if (i + 8 <= n) {
            typename Eight<T>::type t;
#pragma unroll
            for (int e = 0; e < 8; ++e) t[e] = static_cast<T>(v[e]);
            *reinterpret_cast<typename Eight<T>::type*>(row + i) = t;
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (i + e < n) row[i + e] = static_cast<T>(v[e]);
        }
    }
}

// Eight consecutive elements.
template <typename T>
__device__ __forceinline__ void store8(T* __restrict__ row, int i, int n, const float (&v)[8]) {
    if (i + 8 <= n) {
        typename Eight<T>::type t;
#pragma unroll
        for (int e = 0; e < 8; ++e) t[e] = static_cast<T>(v[e]);
        *reinterpret_cast<typename Eight<T>::type*>(row + i) = t;
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (i + e < n) row[i + e] = static_cast<T>(v[e]);
    }
}

// The one-byte codes of the elements that row_take8<T> gives, lowest byte first.
template <typename T>
__device__ __forceinline__ void row_store_codes(uint8_t* __restrict__ row, int lane, int n, uint32_t lo, uint32_t hi) {
    int at[2];
    place8<T>(lane, at);
    if (sizeof(T) == 2 && at[1] + 4 <= n) {
        *reinterpret_cast<U64U*>(row + at[0]) = U64U{lo, hi};
        return;
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const uint32_t w = h ? hi : lo;
        if (at[h] + 4 <= n) {
            reinterpret_cast<U32Any*>(row + at[h])->v = w;
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (at[h] + e < n) row[at[h] + e] = static_cast<uint8_t>(w >> (8 * e));
        }
    }
}

// The integer nearest z / unit, ties to even, for |z / unit| < 512, with r = 1 / unit rounded and unit normal.
// t = z r is within 2^-23 |t| of the quotient, less than 2^-14, so away from a border rounding t is right.  Near one the side is
// the sign of z - m unit with m the border, which a fused multiply-add rounds once and therefore never gets wrong.
__device__ __forceinline__ float nearest_int(float z, float unit, float r) {
    const float t = z * r;
    float k = __builtin_rintf(t);
    const float d = t - k;
    if (__builtin_fabsf(d) > 0.5f - 0x1p-14f) {
        const float m = k + __builtin_copysignf(0.5f, d);
        const float side = __builtin_fmaf(-m, unit, z);
        k = side == 0.0f ? __builtin_rintf(m) : m + __builtin_copysignf(0.5f, side);
    }
    return k;
}

// 1.5 * 2^23: adding it rounds to a whole number, ties to even, which the sum's low byte then holds in two's complement.
constexpr float kRoundToInt = 12582912.0f;

// Eight whole numbers z / unit to the nearest, as what they are plus kRoundToInt, for |z / unit| < TOP.  Elements near a border
// are rare, so all eight share one test, and only then each is looked at on its own.  z r is off by at most 2^-22 of it with r
// within one step of 1 / unit, and what is left of it after rounding by another 2^-25.
template <int TOP>
__device__ __forceinline__ void round8(const float (&z)[8], float unit, float r, float (&f)[8]) {
    constexpr float kNearBorder = 0.5f - TOP * 0x1p-21f;
    float d[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        f[e] = __builtin_fmaf(z[e], r, kRoundToInt);
        d[e] = __builtin_fabsf(__builtin_fmaf(z[e], r, kRoundToInt - f[e]));
    }
    if (__builtin_fmaxf(__builtin_fmaxf(__builtin_fmaxf(d[0], d[1]), __builtin_fmaxf(d[2], d[3])), __builtin_fmaxf(__builtin_fmaxf(d[4], d[5]), __builtin_fmaxf(d[6], d[7]))) >
        kNearBorder) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (d[e] > kNearBorder) f[e] = kRoundToInt + nearest_int(z[e], unit, r);
    }
}

// The low bytes of four words.
__device__ __forceinline__ uint32_t low_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    const uint32_t lo = __builtin_amdgcn_perm(b, a, 0x0c0c0400u), hi = __builtin_amdgcn_perm(d, c, 0x0c0c0400u);
    return __builtin_amdgcn_perm(hi, lo, 0x05040100u);
}

// The e4m3 number nearest z / s, as a float: three mantissa bits, so the integer nearest z / (s step) in units of
// step = 2^(e - 3), with e the quotient's exponent, not below -6 (subnormal numbers share the step 2^-9).
__device__ __forceinline__ float value_e4m3(float z, float s, float r) {
    const int e = max(static_cast<int>((__float_as_uint(z * r) >> 23) & 0xff), 127 - 6);
    const float step = __uint_as_float(static_cast<uint32_t>(e - 3) << 23);
    const float inv_step = __uint_as_float(static_cast<uint32_t>(254 - (e - 3)) << 23);
    return __builtin_amdgcn_fmed3f(nearest_int(z, s * step, r * inv_step) * step, -448.0f, 448.0f);
}

// Codes of eight products, packed.  `plain`: no quotient is beyond the largest code (the unit is no subnormal number, whose
// rounding could put one there).
template <bool FP8>
__device__ __forceinline__ void codes8(const float (&z)[8], float s, float r, bool plain, uint32_t& lo, uint32_t& hi) {
    float f[8];
    if constexpr (FP8) {
        // The conversion rounds to the nearest, ties to even, and z r is within two steps of 2^-24 of the quotient: only what lies
        // that near a border, half way between neighbours (a one and 19 zeros below the three bits that stay), is looked at again.
        // Below 2^-6 the borders are those of the numbers 2^-6 higher.
        uint32_t near = 0xffffffffu;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            f[e] = z[e] * r;
            const float m = __builtin_fabsf(f[e]);
            const uint32_t bits = __float_as_uint(m < 0x1p-6f ? m + 0x1p-6f : m);
            near = min(near, (bits & 0xfffffu) - 0x7fff8u);
        }
        if (near <= 16u || !plain) {
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = value_e4m3(z[e], s, r);
        }
        int p = __builtin_amdgcn_cvt_pk_fp8_f32(f[0], f[1], 0, false);
        lo = static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(f[2], f[3], p, true));
        p = __builtin_amdgcn_cvt_pk_fp8_f32(f[4], f[5], 0, false);
        hi = static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(f[6], f[7], p, true));
    } else {
        round8<128>(z, s, r, f);
        if (!plain) {
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = __builtin_amdgcn_fmed3f(f[e], kRoundToInt - 127.0f, kRoundToInt + 127.0f);
        }
        lo = low_bytes(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
        hi = low_bytes(__float_as_uint(f[4]), __float_as_uint(f[5]), __float_as_uint(f[6]), __float_as_uint(f[7]));
    }
}

// Reductions over a wavefront whose result every lane holds: within rows of 16 by data-parallel moves, across them by lane
// swaps; no LDS traffic.  Sums are taken in a fixed tree, in which the two sides of an addition only trade places from lane to lane.
template <int N>
__device__ __forceinline__ uint32_t row_turned(uint32_t v) {
    return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(static_cast<int>(v), static_cast<int>(v), 0x120 + N, 0xf, 0xf, false));     // row_ror:N
}
template <int N> __device__ __forceinline__ float row_turned(float v) { return __uint_as_float(row_turned<N>(__float_as_uint(v))); }
template <int N> __device__ __forceinline__ double row_turned(double v) {
    const long long b = __double_as_longlong(v);
    const uint32_t lo = row_turned<N>(static_cast<uint32_t>(b)), hi = row_turned<N>(static_cast<uint32_t>(b >> 32));
    return __longlong_as_double(static_cast<long long>(hi) << 32 | lo);
}
// f(v of one half, v of the other), likewise for neighbouring rows of 16.
template <typename F> __device__ __forceinline__ uint32_t across_rows(uint32_t v, F&& f) {
    const auto h = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    const uint32_t w = f(static_cast<uint32_t>(h[0]), static_cast<uint32_t>(h[1]));
    const auto r = __builtin_amdgcn_permlane16_swap(w, w, false, false);
    return f(static_cast<uint32_t>(r[0]), static_cast<uint32_t>(r[1]));
}
__device__ __forceinline__ float wave_sum_all(float v) {
    v += row_turned<8>(v);
    v += row_turned<4>(v);
    v += row_turned<2>(v);
    v += row_turned<1>(v);
    return __uint_as_float(across_rows(__float_as_uint(v), [](uint32_t a, uint32_t b) { return __float_as_uint(__uint_as_float(a) + __uint_as_float(b)); }));
}
__device__ __forceinline__ double wave_sum_all(double v) {
    v += row_turned<8>(v);
    v += row_turned<4>(v);
    v += row_turned<2>(v);
    v += row_turned<1>(v);
    auto join = [](uint32_t hi, uint32_t lo) { return __longlong_as_double(static_cast<long long>(hi) << 32 | lo); };
    long long b = __double_as_longlong(v);
    const auto l = __builtin_amdgcn_permlane32_swap(static_cast<uint32_t>(b), static_cast<uint32_t>(b), false, false);
    const auto h = __builtin_amdgcn_permlane32_swap(static_cast<uint32_t>(b >> 32), static_cast<uint32_t>(b >> 32), false, false);
    v = join(h[0], l[0]) + join(h[1], l[1]);
    b = __double_as_longlong(v);
    const auto m = __builtin_amdgcn_permlane16_swap(static_cast<uint32_t>(b), static_cast<uint32_t>(b), false, false);
    const auto n = __builtin_amdgcn_permlane16_swap(static_cast<uint32_t>(b >> 32), static_cast<uint32_t>(b >> 32), false, false);
    return join(n[0], m[0]) + join(n[1], m[1]);
}
__device__ __forceinline__ uint32_t wave_max_all(uint32_t v) {
    v = max(v, row_turned<8>(v));
    v = max(v, row_turned<4>(v));
    v = max(v, row_turned<2>(v));
    v = max(v, row_turned<1>(v));
    return across_rows(v, [](uint32_t a, uint32_t b) { return max(a, b); });
}

struct NormArgs {
    const void* x;
    const void* residual;       // null: none, and hidden is null too
    const void* weight;
    void* hidden;
    uint8_t* codes;
    float* scales;
    float* inv_rms;
    int64_t x_stride, r_stride; // elements from row to row; outputs are dense
    int64_t rows;
    int dim;
    int fp8;
    double eps;
};

// What follows from a row's sum of squares and largest |z| (its bits: a NaN compares above all numbers).
struct RowScale {
    float s, r;                 // unit of the codes and its reciprocal, both of z * up
    float up;                   // 1, or 2^64 where s is so small that its reciprocal or a residual could leave fp32's range
    bool none;                  // nothing to divide by: all codes are zero
};
__device__ __forceinline__ RowScale row_scale(uint32_t top_bits, bool fp8) {
    const float a = __uint_as_float(top_bits);
    RowScale o;
    o.s = a / (fp8 ? 448.0f : 127.0f);
    o.none = !(o.s > 0.0f) || top_bits >= 0x7f800000u;
    o.up = o.s < 0x1p-90f ? 0x1p64f : 1.0f;
    o.s *= o.up;
    o.r = o.none ? 0.0f : 1.0f / o.s;
    return o;
}
__device__ __forceinline__ void store_row_statistics(const NormArgs& a, int64_t row, double sumsq, uint32_t top_bits) {
    const double inv = 1.0 / sqrt(sumsq / static_cast<double>(a.dim) + a.eps);
    const float s = __uint_as_float(top_bits) / (a.fp8 ? 448.0f : 127.0f);
    a.scales[row] = top_bits >= 0x7f800000u ? __builtin_nanf("") : static_cast<float>(static_cast<double>(s) * inv);
    a.inv_rms[row] = static_cast<float>(inv);
}

// One row per TPR lanes (64: four rows a workgroup; else a workgroup), held in registers between the statistics and
// the codes: every byte is read once and written once.  V vectors of eight per lane.
template <typename XT, typename WT, int TPR, int V, bool ONCE>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void rms_norm_row_kernel(NormArgs a) {
    constexpr int kRows = TPR < 256 ? 256 / TPR : 1;
    const int lane = threadIdx.x % TPR;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * kRows + threadIdx.x / TPR;
    const bool live = row < a.rows;
    float z[V][8];
    double sq = 0.0;
    uint32_t top = 0;
    const XT* xr = static_cast<const XT*>(a.x) + row * a.x_stride;
    const WT* wr = static_cast<const WT*>(a.weight);
    if (live) {
        float w[V][8];
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const typename Eight<XT>::type t = row_take8<ONCE>(xr, lane + j * TPR, a.dim);
#pragma unroll
            for (int e = 0; e < 8; ++e) z[j][e] = static_cast<float>(t[e]);
        }
        if (a.residual) {
            const XT* rr = static_cast<const XT*>(a.residual) + row * a.r_stride;
            XT* hr = static_cast<XT*>(a.hidden) + row * a.dim;
            typename Eight<XT>::type r[V];
#pragma unroll
            for (int j = 0; j < V; ++j) r[j] = row_take8<ONCE>(rr, lane + j * TPR, a.dim);
#pragma unroll
            for (int j = 0; j < V; ++j) {
#pragma unroll
                for (int e = 0; e < 8; ++e) z[j][e] = static_cast<float>(static_cast<XT>(z[j][e] + static_cast<float>(r[j][e])));
                row_store8(hr, lane + j * TPR, a.dim, z[j]);
            }
        }
#pragma unroll
        for (int j = 0; j < V; ++j) {
            weight8<XT>(wr, lane + j * TPR, a.dim, w[j]);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const double h = z[j][e];
                sq = fma(h, h, sq);
                z[j][e] *= w[j][e];
                top = max(top, __float_as_uint(z[j][e]) & 0x7fffffffu);
            }
        }
    }
    sq = wave_sum_all(sq);
    top = wave_max_all(top);
    if constexpr (TPR > 64) {
        __shared__ double sh_sq[TPR / 64];
        __shared__ uint32_t sh_top[TPR / 64];
        if ((threadIdx.x & 63) == 0) { sh_sq[threadIdx.x >> 6] = sq; sh_top[threadIdx.x >> 6] = top; }
        __syncthreads();
        sq = sh_sq[0];
        top = sh_top[0];
#pragma unroll
        for (int w = 1; w < TPR / 64; ++w) { sq += sh_sq[w]; top = max(top, sh_top[w]); }
    }
    if (!live) return;
    const RowScale q = row_scale(top, a.fp8);
    uint8_t* cr = a.codes + row * a.dim;
#pragma unroll
    for (int j = 0; j < V; ++j) {
        if ((lane + j * TPR) / 64 * 512 >= a.dim) break;      // the same for a wavefront
        uint32_t lo = 0, hi = 0;
        if (!q.none) {
            const bool plain = q.up == 1.0f;
            if (!plain) {
#pragma unroll
                for (int e = 0; e < 8; ++e) z[j][e] *= q.up;
            }
            if (a.fp8) codes8<true>(z[j], q.s, q.r, plain, lo, hi);
            else codes8<false>(z[j], q.s, q.r, plain, lo, hi);
        }
        row_store_codes<XT>(cr, lane + j * TPR, a.dim, lo, hi);
    }
    if (lane == 0) store_row_statistics(a, row, sq, top);
}

// Rows too long for the registers of a workgroup: two visits, the second to what the first has just read or written
// (a lane reads back its own elements only).
template <typename XT, typename WT>
__global__ __launch_bounds__(1024) void rms_norm_loop_kernel(NormArgs a) {
    __shared__ double sh_sq[16];
    __shared__ uint32_t sh_top[16];
    const int64_t row = blockIdx.x;
    const XT* xr = static_cast<const XT*>(a.x) + row * a.x_stride;
    const XT* rr = a.residual ? static_cast<const XT*>(a.residual) + row * a.r_stride : nullptr;
    XT* hr = a.residual ? static_cast<XT*>(a.hidden) + row * a.dim : nullptr;
    const WT* wr = static_cast<const WT*>(a.weight);
    double sq = 0.0;
    uint32_t top = 0;
    const int turns = (a.dim + 8191) / 8192;
    for (int turn = 0; turn < turns; ++turn) {
        const int l = turn * 1024 + threadIdx.x;
        float h[8], w[8];
        const typename Eight<XT>::type x = row_take8<false>(xr, l, a.dim);
        weight8<XT>(wr, l, a.dim, w);
#pragma unroll
        for (int e = 0; e < 8; ++e) h[e] = static_cast<float>(x[e]);
        if (rr) {
            const typename Eight<XT>::type r = row_take8<false>(rr, l, a.dim);
#pragma unroll
            for (int e = 0; e < 8; ++e) h[e] = static_cast<float>(static_cast<XT>(h[e] + static_cast<float>(r[e])));
            row_store8(hr, l, a.dim, h);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const double d = h[e];
            sq = fma(d, d, sq);
            top = max(top, __float_as_uint(h[e] * w[e]) & 0x7fffffffu);
        }
    }
    sq = wave_sum_all(sq);
    top = wave_max_all(top);
    if ((threadIdx.x & 63) == 0) { sh_sq[threadIdx.x >> 6] = sq; sh_top[threadIdx.x >> 6] = top; }
    __syncthreads();
    sq = sh_sq[0];
    top = sh_top[0];
#pragma unroll
    for (int w = 1; w < 16; ++w) { sq += sh_sq[w]; top = max(top, sh_top[w]); }
    const RowScale q = row_scale(top, a.fp8);
    uint8_t* cr = a.codes + row * a.dim;
    const XT* back = hr ? hr : xr;
    for (int turn = 0; turn < turns; ++turn) {
        const int l = turn * 1024 + threadIdx.x;
        uint32_t lo = 0, hi = 0;
        if (!q.none) {
            float z[8], w[8];
            const typename Eight<XT>::type h = row_take8<false>(back, l, a.dim);
            weight8<XT>(wr, l, a.dim, w);
#pragma unroll
            for (int e = 0; e < 8; ++e) z[e] = static_cast<float>(h[e]) * w[e] * q.up;
            if (a.fp8) codes8<true>(z, q.s, q.r, q.up == 1.0f, lo, hi);
            else codes8<false>(z, q.s, q.r, q.up == 1.0f, lo, hi);
        }
        row_store_codes<XT>(cr, l, a.dim, lo, hi);
    }
    if (threadIdx.x == 0) store_row_statistics(a, row, sq, top);
}

// ---- gradients ----
//   u = dy w,  c = inv^2 sum(u h) / dim,  dx = inv (u - h c) + dh,  dw = sum over rows of dy h inv
// with dy the gradient of what the codes stand for (the rounding to codes is passed straight through) and dh that
// of the stored sum.
struct NormGradArgs {
    const void* grad;
    const void* hidden;
    const void* weight;
    const float* inv_rms;
    const void* grad_hidden;    // null: none
    void* grad_x;
    float* partials;            // [groups][dim]: a workgroup's share of dw
    int64_t g_stride, h_stride, gh_stride;
    int64_t rows;
    int dim;
};

// A workgroup of TPR lanes takes rows blockIdx.x, + gridDim.x, ...; a lane keeps its columns' share of dw in registers over
// all of them, so dw costs one store of a row per workgroup.  The next row is on its way while one is worked on.
template <typename XT, typename WT, int TPR, int V, bool ONCE>
__global__ __launch_bounds__(TPR) void rms_norm_grad_kernel(NormGradArgs a) {
    __shared__ float sh[2][TPR / 64];
    typedef typename Eight<XT>::type eight;
    constexpr bool kAhead = TPR < 1024;        // the 128 registers of 1024 lanes do not hold another row
    const int lane = threadIdx.x;
    const XT* grad = static_cast<const XT*>(a.grad);
    const XT* hidden = static_cast<const XT*>(a.hidden);
    const XT* grad_hidden = static_cast<const XT*>(a.grad_hidden);
    eight g0[V], h0[V], d0[V];
    float inv0;
    auto fetch = [&](int64_t row) {
        inv0 = a.inv_rms[row];
#pragma unroll
        for (int j = 0; j < V; ++j) {
            g0[j] = row_take8<ONCE>(grad + row * a.g_stride, lane + j * TPR, a.dim);
            h0[j] = row_take8<ONCE>(hidden + row * a.h_stride, lane + j * TPR, a.dim);
        }
        if (grad_hidden) {
#pragma unroll
            for (int j = 0; j < V; ++j) d0[j] = row_take8<ONCE>(grad_hidden + row * a.gh_stride, lane + j * TPR, a.dim);
        }
    };
#pragma unroll
    for (int j = 0; j < V; ++j)
#pragma unroll
        for (int e = 0; e < 8; ++e) d0[j][e] = static_cast<XT>(0.0f);
    if (kAhead) fetch(blockIdx.x);
    float dw[V][8], w[V][8];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        weight8<XT>(static_cast<const WT*>(a.weight), lane + j * TPR, a.dim, w[j]);
#pragma unroll
        for (int e = 0; e < 8; ++e) dw[j][e] = 0.0f;
    }
    const float over_dim = 1.0f / static_cast<float>(a.dim);
    int turn = 0;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x, turn ^= 1) {
        if (!kAhead) fetch(row);
        const float inv = inv0;
        float g[V][8], h[V][8];
        eight d[V];
        float c = 0.0f;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            d[j] = d0[j];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                g[j][e] = static_cast<float>(g0[j][e]);
                h[j][e] = static_cast<float>(h0[j][e]) * inv;      // the normalised row
            }
        }
        if (kAhead) fetch(row + gridDim.x < a.rows ? row + gridDim.x : row);
#pragma unroll
        for (int j = 0; j < V; ++j)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                dw[j][e] = fmaf(g[j][e], h[j][e], dw[j][e]);
                g[j][e] *= w[j][e];
                c = fmaf(g[j][e], h[j][e], c);
            }
        c = wave_sum_all(c);
        if constexpr (TPR > 64) {
            // two slots in turn: a wavefront may write the next row's before another has read this row's
            if ((lane & 63) == 0) sh[turn][lane >> 6] = c;
            __syncthreads();
            c = sh[turn][0];
#pragma unroll
            for (int q = 1; q < TPR / 64; ++q) c += sh[turn][q];
        }
        c *= over_dim;
#pragma unroll
        for (int j = 0; j < V; ++j) {
#pragma unroll
            for (int e = 0; e < 8; ++e) g[j][e] = fmaf(inv, fmaf(-h[j][e], c, g[j][e]), static_cast<float>(d[j][e]));
            row_store8(static_cast<XT*>(a.grad_x) + row * a.dim, lane + j * TPR, a.dim, g[j]);
        }
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
        float* to = a.partials + static_cast<int64_t>(blockIdx.x) * a.dim;
        if constexpr (sizeof(XT) == 4) row_store8(to, lane + j * TPR, a.dim, dw[j]);
        else store8(to, (lane + j * TPR) * 8, a.dim, dw[j]);
    }
}

// Rows too long for that: the row's c first, ...
template <typename XT, typename WT>
__global__ __launch_bounds__(1024) void rms_norm_grad_dot_kernel(NormGradArgs a, float* dots) {
    __shared__ float sh[16];
    const int64_t row = blockIdx.x;
    const float inv = a.inv_rms[row];
    float c = 0.0f;
    for (int64_t i = static_cast<int64_t>(threadIdx.x) * 8; i < a.dim; i += 8192) {
        float g[8], h[8], w[8];
        load8(static_cast<const XT*>(a.grad) + row * a.g_stride, i, a.dim, g);
        load8(static_cast<const XT*>(a.hidden) + row * a.h_stride, i, a.dim, h);
        load8(static_cast<const WT*>(a.weight), i, a.dim, w);
#pragma unroll
        for (int e = 0; e < 8; ++e) c = fmaf(g[e] * w[e], h[e] * inv, c);
    }
    c = wave_sum_all(c);
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = c;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int q = 1; q < 16; ++q) c += sh[q];
        dots[row] = c / static_cast<float>(a.dim);
    }
}
// ... then stretches of 2048 columns by bands of rows.
template <typename XT, typename WT>
__global__ __launch_bounds__(256) void rms_norm_grad_apply_kernel(NormGradArgs a, const float* dots, int stretches, int bands) {
    const int band = blockIdx.x / stretches;
    const int64_t i = static_cast<int64_t>(blockIdx.x % stretches) * 2048 + threadIdx.x * 8;
    if (i >= a.dim) return;
    float w[8], dw[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    load8(static_cast<const WT*>(a.weight), i, a.dim, w);
    for (int64_t row = band; row < a.rows; row += bands) {
        const float inv = a.inv_rms[row], c = dots[row];
        float g[8], h[8], dh[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        load8(static_cast<const XT*>(a.grad) + row * a.g_stride, i, a.dim, g);
        load8(static_cast<const XT*>(a.hidden) + row * a.h_stride, i, a.dim, h);
        if (a.grad_hidden) load8(static_cast<const XT*>(a.grad_hidden) + row * a.gh_stride, i, a.dim, dh);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            h[e] *= inv;
            dw[e] = fmaf(g[e], h[e], dw[e]);
            g[e] = fmaf(inv, fmaf(-h[e], c, g[e] * w[e]), dh[e]);
        }
        store8(static_cast<XT*>(a.grad_x) + row * a.dim, i, a.dim, g);
    }
    store8(a.partials + static_cast<int64_t>(band) * a.dim, i, a.dim, dw);
}

// dw[i] = the sum of the workgroups' shares: 32 columns a workgroup, each by 32 lanes whose sums are added in their order.
// `first`: this launch's first column.
template <typename WT>
__global__ __launch_bounds__(1024) void column_sum_kernel(const float* __restrict__ partials, int groups, int dim, int64_t first, WT* __restrict__ out) {
    __shared__ double sh[32][33];
    const int c = threadIdx.x & 31, part = threadIdx.x >> 5;
    const int64_t col = first + static_cast<int64_t>(blockIdx.x) * 32 + c;
    double s = 0.0;
    if (col < dim) {
        const float* p = partials + col;
        int g = part;
        // four on their way at a time
        for (; g + 96 < groups; g += 128) {
            const float a = p[static_cast<int64_t>(g) * dim], b = p[static_cast<int64_t>(g + 32) * dim], d = p[static_cast<int64_t>(g + 64) * dim],
                        e = p[static_cast<int64_t>(g + 96) * dim];
            s += (static_cast<double>(a) + b) + (static_cast<double>(d) + e);
        }
        for (; g < groups; g += 32) s += static_cast<double>(p[static_cast<int64_t>(g) * dim]);
    }
    sh[part][c] = s;
    __syncthreads();
    if (part == 0 && col < dim) {
#pragma unroll
        for (int q = 1; q < 32; ++q) s += sh[q][c];
        out[col] = static_cast<WT>(static_cast<float>(s));
    }
}
