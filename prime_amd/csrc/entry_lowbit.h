// C entry points of the low-bit operators (kernels_norm.h, kernels_lowbit.h): argument checks, choice of the kernel,
// launch.
//
// Included by prime_hip.hip behind its other host code; not a translation unit of its own.

namespace {

// Calls f with a value of the element type; false: not a type of this operand.
template <typename F>
bool with_float_type(int type, F&& f) {
    if (type == PRIME_F32) f(float{});
    else if (type == PRIME_BF16) f(__bf16{});
    else if (type == PRIME_F16) f(_Float16{});
    else return false;
    return true;
}
bool is_float_type(int type) { return type == PRIME_F32 || type == PRIME_BF16 || type == PRIME_F16; }
bool is_scale_type(int type) { return type == PRIME_F32 || type == PRIME_BF16; }
int type_bytes(int type) { return type == PRIME_F32 ? 4 : type == PRIME_I8 || type == PRIME_F8E4M3 ? 1 : 2; }
template <typename F>
void with_scale_type(int type, F&& f) {
    if (type == PRIME_F32) f(float{});
    else f(__bf16{});
}
// A norm's weight has the rows' type or fp32.
template <typename XT, typename F>
void with_weight_type(int weight_type, int type, F&& f) {
    if (weight_type == type) f(XT{});
    else f(float{});
}

constexpr int64_t kMaxDim = int64_t(1) << 30;

// A dispatch counts its work-items in 32 bits: 1024 a row at most, and 32 a column of a sum over rows.
constexpr int64_t kRowsPerLaunch = int64_t(1) << 21, kColumnsPerLaunch = int64_t(1) << 26;

// Rows are read with the hint that leaves them out of the caches when a call moves more than the last-level cache holds anyway
// (256 MiB): norm of 16384 x 4096 bf16 with residual (470 MB) 74 us with it and 82 without, its gradient (537 MB) 89 and 98; a quarter of those
// rows (117 and 134 MB) 23.6 and 20.3, 31.1 and 29.4.  Packing gains from half of that up: 16384 x 4096 bf16 (134 MB) 30.5 and 33.8 us,
// 4096 x 4096 fp32 (67 MB) 16.1 and 13.7.
constexpr double kOnceNormBytes = 300e6, kOncePackBytes = 128e6;
template <typename F>
void with_once(bool once, F&& f) {
    if (once) f(std::true_type{});
    else f(std::false_type{});
}

// Lanes of a row: about as few as hold it in two vectors of eight each, so that a row's reductions and barrier are few beside its loads.  67 million
// elements of bf16 with residual, and in brackets with 256 lanes for 64 and twice as many for 256 and 512: rows of 256 elements 169 us (411), 512
// 83 (195), 1024 74 (118), 4096 73 (80), 8192 74 (81); rows of 16384 in registers 96, in the loop 129.
template <typename XT, typename WT, bool ONCE>
void launch_rms_norm(const NormArgs& a, double bytes, hipStream_t st) {
    const int64_t r = a.rows;
    const int quads = static_cast<int>((r + 3) / 4), all = static_cast<int>(r);
    if (a.dim <= 512) launch(kIdRmsNorm, bytes, rms_norm_row_kernel<XT, WT, 64, 1, ONCE>, quads, 256, st, a);
    else if (a.dim <= 1024) launch(kIdRmsNorm, bytes, rms_norm_row_kernel<XT, WT, 64, 2, ONCE>, quads, 256, st, a);
    else if (a.dim <= 2048) launch(kIdRmsNorm, bytes, rms_norm_row_kernel<XT, WT, 256, 1, ONCE>, all, 256, st, a);
    else if (a.dim <= 4096) launch(kIdRmsNorm, bytes, rms_norm_row_kernel<XT, WT, 256, 2, ONCE>, all, 256, st, a);
    else if (a.dim <= 8192) launch(kIdRmsNorm, bytes, rms_norm_row_kernel<XT, WT, 512, 2, ONCE>, all, 512, st, a);
    else if (a.dim <= 16384) launch(kIdRmsNorm, bytes, rms_norm_row_kernel<XT, WT, 1024, 2, ONCE>, all, 1024, st, a);
    else launch(kIdRmsNorm, bytes, rms_norm_loop_kernel<XT, WT>, all, 1024, st, a);
}

// Workgroups (= partial rows of the weight's gradient) of the backward pass, and its scratch.  Lanes as above: 67 million elements of bf16, and in brackets
// with twice as many: rows of 256 elements 246 us (444), 512 102 (169), 1024 79 (105), 2048 75 (104), 4096 71 (90), 8192 76 (72); rows of
// 16384 in registers 72, by two kernels 123.
constexpr int kGradRegisterDim = 16384;      // rows up to this long stay in registers
int grad_lanes(int64_t dim) { return dim <= 1024 ? 64 : dim <= 2048 ? 128 : dim <= 4096 ? 256 : dim <= 8192 ? 512 : 1024; }
int grad_stretches(int64_t dim) { return static_cast<int>((dim + 2047) / 2048); }
int64_t grad_groups(int64_t rows, int64_t dim) {
    int64_t most = dim <= kGradRegisterDim ? static_cast<int64_t>(cu_count()) * std::max(1, 512 / grad_lanes(dim))
                                           : static_cast<int64_t>(cu_count()) * 8 / grad_stretches(dim);
    if (most < 1) most = 1;
    return rows < most ? rows : most;
}
int64_t grad_scratch_bytes(int64_t rows, int64_t dim) {
    return grad_groups(rows, dim) * dim * 4 + (dim > kGradRegisterDim ? rows * 4 : 0);
}

template <typename XT, typename WT, bool ONCE>
void launch_rms_norm_grad(const NormGradArgs& a, int groups, WT* grad_weight, double bytes, hipStream_t st) {
    if (a.rows > 0) {
        if (a.dim <= 512) launch(kIdRmsNormGrad, bytes, rms_norm_grad_kernel<XT, WT, 64, 1, ONCE>, groups, 64, st, a);
        else if (a.dim <= 1024) launch(kIdRmsNormGrad, bytes, rms_norm_grad_kernel<XT, WT, 64, 2, ONCE>, groups, 64, st, a);
        else if (a.dim <= 2048) launch(kIdRmsNormGrad, bytes, rms_norm_grad_kernel<XT, WT, 128, 2, ONCE>, groups, 128, st, a);
        else if (a.dim <= 4096) launch(kIdRmsNormGrad, bytes, rms_norm_grad_kernel<XT, WT, 256, 2, ONCE>, groups, 256, st, a);
        else if (a.dim <= 8192) launch(kIdRmsNormGrad, bytes, rms_norm_grad_kernel<XT, WT, 512, 2, ONCE>, groups, 512, st, a);
        else if (a.dim <= kGradRegisterDim) launch(kIdRmsNormGrad, bytes, rms_norm_grad_kernel<XT, WT, 1024, 2, ONCE>, groups, 1024, st, a);
        else {
            float* dots = a.partials + static_cast<int64_t>(groups) * a.dim;
            for (int64_t at = 0; at < a.rows; at += kRowsPerLaunch) {
                NormGradArgs part = a;
                part.rows = std::min(a.rows - at, kRowsPerLaunch);
                part.grad = static_cast<const XT*>(a.grad) + at * a.g_stride;
                part.hidden = static_cast<const XT*>(a.hidden) + at * a.h_stride;
                part.inv_rms = a.inv_rms + at;
                launch(kIdRmsNormGrad, bytes, rms_norm_grad_dot_kernel<XT, WT>, static_cast<int>(part.rows), 1024, st, part, dots + at);
            }
            const int stretches = grad_stretches(a.dim);
            launch(kIdRmsNormGrad, bytes, rms_norm_grad_apply_kernel<XT, WT>, stretches * groups, 256, st, a, dots, stretches, groups);
        }
    }
    for (int64_t at = 0; at < a.dim; at += kColumnsPerLaunch) {
        const int64_t columns = std::min(a.dim - at, kColumnsPerLaunch);
        launch(kIdColumnSum, 4.0 * groups * columns, column_sum_kernel<WT>, static_cast<int>((columns + 31) / 32), 1024, st, a.partials, groups, a.dim, at, grad_weight);
    }
}

bool bad_group(int group) { return group != 32 && group != 64 && group != 128; }
bool bad_matrix(int64_t n, int64_t k) { return n < 0 || n >= (int64_t(1) << 40) || k < 1 || k > kMaxDim; }
int group_shift(int group) { return group == 32 ? 5 : group == 64 ? 6 : 7; }

// Up to four rows.
template <typename XT, typename ST, int GS>
void launch_matvec_few(MatvecArgs a, double bytes, hipStream_t st) {
    // two workgroups of eight wavefronts beside each other: 4 x 8192 x 22528 fp32 34 us, with 28 KiB 39, with 112 KiB 45; of what 56 KiB do not
    // hold whole and 112 do, bf16 29, 31 and 25
    constexpr int kMostLds = 56 << 10;
    const int held = a.rows, quads = (a.k + 511) / 512, quad_bytes = 4 * kFewBlock<XT>;
    a.tiles = (a.n + 15) / 16;
    // wavefronts that share a tile's columns: enough for 16 wavefronts a compute unit, but not more than it has stretches (1 x 8192 x 22528 int8
    // 21.8 us, for 8 wavefronts 27.9, for 32 24.2)
    const int wanted = cu_count() * 16;
    a.split_shift = 0;
    while (a.split_shift < 3 && (static_cast<int64_t>(a.tiles) << a.split_shift) < wanted && (2 << a.split_shift) <= quads) ++a.split_shift;
    const int waves = (static_cast<int64_t>(a.tiles) << a.split_shift) >= wanted / 2 ? 8 : std::max(4, 1 << a.split_shift);
    // whole rows of x in LDS if they fit, else as many stretches as do, a multiple of what the wavefronts take in a turn
    const int most = (kMostLds / held - kFewPad<XT>) / quad_bytes;
    while (quads > most && (1 << a.split_shift) > most) --a.split_shift;
    a.chunk_quads = quads <= most ? quads : most >> a.split_shift << a.split_shift;
    const int side = waves >> a.split_shift;
    a.sets = (a.tiles + side - 1) / side;
    const int lds = held * (a.chunk_quads * quad_bytes + kFewPad<XT>);
    int grid = a.sets;
    if (quads <= most && a.sets > cu_count()) {
        // workgroups that stay for all their tiles: as many as the device holds
        int fit = 0;
        if (hipOccupancyMaxActiveBlocksPerMultiprocessor(&fit, matvec4_few_kernel<XT, ST, GS>, waves * 64, lds) != hipSuccess || fit < 1) fit = 1;
        grid = std::min(a.sets, cu_count() * fit);
    }
    launch_lds(kIdMatvec4, bytes, matvec4_few_kernel<XT, ST, GS>, grid, waves * 64, lds, st, a);
}

// Times that rows of k columns are taken up by eight wavefronts of `blocks` blocks each.
int visits_of(int k, int blocks) { return ((k + 127) / 128 + 8 * blocks - 1) / (8 * blocks); }

template <typename XT, typename ST, int GS, int MT, int B, int NT>
void launch_matvec_many_as(MatvecArgs a, double bytes, hipStream_t st) {
    constexpr int kRows = 16 * MT, kPart = NT * MT * 256 * 4;
    a.sets = (a.n + 16 * NT - 1) / (16 * NT);
    const int64_t row_tiles = (static_cast<int64_t>(a.rows) + kRows - 1) / kRows;
    const int visits = visits_of(a.k, B);
    // workgroups that stay for all their rounds, one a compute unit, all with as many (within one); with several visits LDS keeps the
    // sums of at most 48 KiB of rounds
    const int64_t most = visits > 1 ? (48 << 10) / kPart : int64_t(1) << 30;
    const int64_t wanted = std::max<int64_t>(1, cu_count() / row_tiles), rounds = std::min<int64_t>(most, (a.sets + wanted - 1) / wanted);
    const int per_row_tile = static_cast<int>((a.sets + rounds - 1) / rounds);
    const int lds = visits > 1 ? static_cast<int>(rounds) * kPart : 0;
    // a dispatch counts its work-items in 32 bits: 2^22 workgroups at a time
    const int64_t step = std::max<int64_t>(1, (int64_t(1) << 22) / per_row_tile);
    const int type = a.out_type, rows = a.rows;
    for (int64_t at = 0; at < row_tiles; at += step) {
        MatvecArgs part = a;
        const int64_t row = at * kRows;
        part.rows = static_cast<int>(std::min<int64_t>(rows - row, step * kRows));
        part.x = static_cast<const XT*>(a.x) + row * a.x_stride;
        if (a.x_scales) part.x_scales = a.x_scales + row;
        part.out = static_cast<uint8_t*>(a.out) + row * a.n * type_bytes(type);
        launch_lds(kIdMatvec4, bytes, matvec4_many_kernel<XT, ST, GS, MT, B, NT>, static_cast<int>(per_row_tile * ((part.rows + kRows - 1) / kRows)), 512, lds,
                   st, part);
    }
}

// Tiles of rows, blocks of columns and tiles of outputs of a wavefront: what 256 registers hold, next to the scales of a round (which
// groups of 32 have four times as many of).  Up to 16 rows take six blocks and half the outputs where that saves a visit: 7 x 5604 x 11263
// fp16 groups of 32 19 us against 23 (16 since codes are widened with their sign); where it does not, four blocks: 16 x 8192 x 22528 bf16 35 us
// (eight blocks do not fit: 40).
template <typename XT, typename ST, int GS>
void launch_matvec_many(const MatvecArgs& a, double bytes, hipStream_t st) {
    constexpr bool k32 = sizeof(XT) == 4, k8 = sizeof(XT) == 1, kWide = GS == 5 && sizeof(ST) == 4 && !k8;
    // more rows in tiles of 16 all the same where each tile finds a compute unit of its own: a wavefront's work is then a
    // quarter as long, and the codes that every tile reads come from the caches: 59 x 6720 x 76 bf16 15 us, and 34 with 64 rows a workgroup
    const bool small = (static_cast<int64_t>(a.rows) + 15) / 16 * ((static_cast<int64_t>(a.n) + 31) / 32) <= cu_count();
    if (a.rows <= 16 || small) {
        if constexpr (k32) launch_matvec_many_as<XT, ST, GS, 1, 2, 2>(a, bytes, st);
        else if (visits_of(a.k, 6) < visits_of(a.k, 4)) launch_matvec_many_as<XT, ST, GS, 1, 6, 1>(a, bytes, st);
        else launch_matvec_many_as<XT, ST, GS, 1, 4, kWide ? 1 : 2>(a, bytes, st);
    } else if (a.rows <= 32 || k32) {
        launch_matvec_many_as<XT, ST, GS, 2, k32 ? 1 : kWide ? 2 : 4, k32 || k8 ? 2 : 1>(a, bytes, st);
    } else if constexpr (!k32) {
        launch_matvec_many_as<XT, ST, GS, 4, 2, k8 ? 2 : 1>(a, bytes, st);
    }
}

template <typename XT>
void launch_matvec(const MatvecArgs& a, int group, int scale_type, double bytes, hipStream_t st) {
    auto go = [&](auto gs) {
        constexpr int GS = decltype(gs)::value;
        with_scale_type(scale_type, [&](auto s) {
            // four rows are what 16 rows of the A operand hold with three planes each: 4 x 4096 x 4096 bf16 6.3 us, by the kernel for more 9.0;
            // 4 x 8192 x 22528 bf16 29.0 and 30.5, fp32 34.3 and 37.2
            if (a.rows <= 4) launch_matvec_few<XT, decltype(s), GS>(a, bytes, st);
            else launch_matvec_many<XT, decltype(s), GS>(a, bytes, st);
        });
    };
    if (group == 32) go(std::integral_constant<int, 5>{});
    else if (group == 64) go(std::integral_constant<int, 6>{});
    else go(std::integral_constant<int, 7>{});
}

}  // namespace

extern "C" {

int prime_rms_norm_quantize(const void* x, int64_t x_stride, const void* residual, int64_t residual_stride, const void* weight, int64_t rows,
                            int64_t dim, int type, int weight_type, int code_type, double eps, void* codes, float* scales, void* hidden,
                            float* inv_rms, prime_stream_t stream) {
    if (rows < 0 || rows > kMaxElems || dim < 1 || dim > kMaxDim || x_stride < 0 || residual_stride < 0)
        return fail(PRIME_EINVAL, "prime_rms_norm_quantize: bad size");
    if (!is_float_type(type) || (weight_type != type && weight_type != PRIME_F32) || (code_type != PRIME_I8 && code_type != PRIME_F8E4M3))
        return fail(PRIME_EINVAL, "prime_rms_norm_quantize: bad type");
    if (!(eps >= 0.0)) return fail(PRIME_EINVAL, "prime_rms_norm_quantize: eps must not be negative");
    if (rows == 0) return 0;
    if (!x || !weight || !codes || !scales || !inv_rms || (residual == nullptr) != (hidden == nullptr))
        return fail(PRIME_EINVAL, "prime_rms_norm_quantize: null operand");
    const double row_bytes = static_cast<double>(dim) * (type_bytes(type) * (residual ? 3 : 1) + 1) + 8.0;
    for (int64_t at = 0; at < rows; at += kRowsPerLaunch) {
        const int64_t part = std::min(rows - at, kRowsPerLaunch);
        with_float_type(type, [&](auto t) {
            using XT = decltype(t);
            NormArgs a{static_cast<const XT*>(x) + at * x_stride, residual ? static_cast<const XT*>(residual) + at * residual_stride : nullptr, weight,
                       hidden ? static_cast<XT*>(hidden) + at * dim : nullptr, static_cast<uint8_t*>(codes) + at * dim, scales + at, inv_rms + at,
                       x_stride, residual_stride, part, static_cast<int>(dim), code_type == PRIME_F8E4M3, eps};
            with_weight_type<XT>(weight_type, type, [&](auto w) {
                with_once(row_bytes * rows >= kOnceNormBytes, [&](auto once) {
                    launch_rms_norm<XT, decltype(w), decltype(once)::value>(a, row_bytes * part, static_cast<hipStream_t>(stream));
                });
            });
        });
        if (int rc = launch_check("rms_norm_row_kernel")) return rc;
    }
    return 0;
}

int64_t prime_rms_norm_backward_scratch_bytes(int64_t rows, int64_t dim) {
    if (rows < 0 || rows > kMaxElems || dim < 1 || dim > kMaxDim) return PRIME_EINVAL;
    return grad_scratch_bytes(rows, dim);
}

int prime_rms_norm_quantize_backward(const void* grad, int64_t grad_stride, const void* hidden, int64_t hidden_stride, const void* weight,
                                     const float* inv_rms, const void* grad_hidden, int64_t grad_hidden_stride, int64_t rows, int64_t dim,
                                     int type, int weight_type, void* grad_x, void* grad_weight, void* scratch, int64_t scratch_bytes,
                                     prime_stream_t stream) {
    if (rows < 0 || rows > kMaxElems || dim < 1 || dim > kMaxDim || grad_stride < 0 || hidden_stride < 0 || grad_hidden_stride < 0)
        return fail(PRIME_EINVAL, "prime_rms_norm_quantize_backward: bad size");
    if (!is_float_type(type) || (weight_type != type && weight_type != PRIME_F32))
        return fail(PRIME_EINVAL, "prime_rms_norm_quantize_backward: bad type");
    if (!weight || !grad_weight || (rows > 0 && (!grad || !hidden || !inv_rms || !grad_x)))
        return fail(PRIME_EINVAL, "prime_rms_norm_quantize_backward: null operand");
    if (rows > 0 && (!scratch || scratch_bytes < grad_scratch_bytes(rows, dim) || !aligned_to(scratch, 4)))
        return fail(PRIME_EWORKSPACE, "prime_rms_norm_quantize_backward: scratch missing, too small or not aligned");
    const double bytes = static_cast<double>(rows) * dim * type_bytes(type) * (grad_hidden ? 4 : 3);
    with_float_type(type, [&](auto t) {
        using XT = decltype(t);
        NormGradArgs a{grad, hidden, weight, inv_rms, grad_hidden, grad_x, static_cast<float*>(scratch), grad_stride, hidden_stride, grad_hidden_stride,
                       rows, static_cast<int>(dim)};
        with_weight_type<XT>(weight_type, type, [&](auto w) {
            with_once(bytes >= kOnceNormBytes, [&](auto once) {
                launch_rms_norm_grad<XT, decltype(w), decltype(once)::value>(a, static_cast<int>(grad_groups(rows, dim)), static_cast<decltype(w)*>(grad_weight),
                                                                             bytes, static_cast<hipStream_t>(stream));
            });
        });
    });
    return launch_check("rms_norm_grad_kernel");
}

int prime_quantize_4bit(const void* weight, int64_t stride, int64_t n, int64_t k, int type, int group, int scale_type, uint8_t* packed,
                        void* scales, prime_stream_t stream) {
    if (bad_matrix(n, k) || stride < 0) return fail(PRIME_EINVAL, "prime_quantize_4bit: bad size");
    if (!is_float_type(type) || !is_scale_type(scale_type)) return fail(PRIME_EINVAL, "prime_quantize_4bit: bad type");
    if (bad_group(group)) return fail(PRIME_EINVAL, "prime_quantize_4bit: group must be 32, 64 or 128");
    if (n == 0) return 0;
    if (!weight || !packed || !scales) return fail(PRIME_EINVAL, "prime_quantize_4bit: null operand");
    const int64_t groups = (k + group - 1) / group, row_codes = groups * group;
    const int64_t step = std::max<int64_t>(1, ((int64_t(1) << 30) - 1) / (row_codes / 4));      // rows a launch: indexes in 31 bits
    for (int64_t at = 0; at < n; at += step) {
        const int64_t rows = std::min(n - at, step);
        with_float_type(type, [&](auto t) {
            using T = decltype(t);
            constexpr int E = kUnit<T>;
            with_scale_type(scale_type, [&](auto s) {
                using ST = decltype(s);
                const int64_t units = rows * (row_codes / E);
                PackArgs a{static_cast<const T*>(weight) + at * stride, stride, packed + at * row_codes / 2, static_cast<ST*>(scales) + at * groups,
                           static_cast<uint32_t>(units), static_cast<int>(k), group / E, group_shift(group) - (E == 8 ? 3 : 2),
                           FastDiv(static_cast<uint32_t>(row_codes / E))};
                with_once(static_cast<double>(n) * k * sizeof(T) >= kOncePackBytes, [&](auto once) {
                    launch(kIdGroupPack, static_cast<double>(rows) * (k * sizeof(T) + row_codes / 2 + groups * sizeof(ST)),
                           group4_pack_kernel<T, ST, decltype(once)::value>, static_cast<int>((units + 256 * kPackEach - 1) / (256 * kPackEach)), 256,
                           static_cast<hipStream_t>(stream), a);
                });
            });
        });
        if (int rc = launch_check("group4_pack_kernel")) return rc;
    }
    return 0;
}

int prime_dequantize_4bit(const uint8_t* packed, int64_t packed_stride, const void* scales, int64_t scale_stride, int64_t n, int64_t k,
                          int group, int scale_type, void* out, int out_type, prime_stream_t stream) {
    if (bad_matrix(n, k) || packed_stride < 0 || scale_stride < 0) return fail(PRIME_EINVAL, "prime_dequantize_4bit: bad size");
    if (!is_float_type(out_type) || !is_scale_type(scale_type)) return fail(PRIME_EINVAL, "prime_dequantize_4bit: bad type");
    if (bad_group(group)) return fail(PRIME_EINVAL, "prime_dequantize_4bit: group must be 32, 64 or 128");
    if (n == 0) return 0;
    if (!packed || !scales || !out) return fail(PRIME_EINVAL, "prime_dequantize_4bit: null operand");
    const int64_t step = std::max<int64_t>(1, ((int64_t(1) << 30) - 1) / ((k + 3) / 4));
    for (int64_t at = 0; at < n; at += step) {
        const int64_t rows = std::min(n - at, step);
        with_float_type(out_type, [&](auto t) {
            using T = decltype(t);
            constexpr int E = kUnit<T>;
            with_scale_type(scale_type, [&](auto s) {
                using ST = decltype(s);
                const int64_t row_units = (k + E - 1) / E, units = rows * row_units;
                UnpackArgs a{packed + at * packed_stride, static_cast<const ST*>(scales) + at * scale_stride, static_cast<T*>(out) + at * k, packed_stride,
                             scale_stride, static_cast<uint32_t>(units), static_cast<int>(k), group_shift(group) - (E == 8 ? 3 : 2),
                             FastDiv(static_cast<uint32_t>(row_units))};
                launch(kIdGroupUnpack, static_cast<double>(rows) * (k * (sizeof(T) + 0.5)), group4_unpack_kernel<T, ST>,
                       static_cast<int>((units + 256 * kUnpackEach - 1) / (256 * kUnpackEach)), 256, static_cast<hipStream_t>(stream), a);
            });
        });
        if (int rc = launch_check("group4_unpack_kernel")) return rc;
    }
    return 0;
}

int prime_matvec_4bit(const void* x, int64_t x_stride, int x_type, const float* x_scales, const uint8_t* packed, int64_t packed_stride,
                      const void* scales, int64_t scale_stride, int64_t rows, int64_t n, int64_t k, int group, int scale_type, void* out,
                      int out_type, prime_stream_t stream) {
    if (bad_matrix(n, k) || n > (int64_t(1) << 26) || rows < 0 || rows >= (int64_t(1) << 31) || x_stride < 0 || packed_stride < 0 || scale_stride < 0)
        return fail(PRIME_EINVAL, "prime_matvec_4bit: bad size");
    if ((!is_float_type(x_type) && x_type != PRIME_I8) || !is_float_type(out_type) || !is_scale_type(scale_type))
        return fail(PRIME_EINVAL, "prime_matvec_4bit: bad type");
    if (bad_group(group)) return fail(PRIME_EINVAL, "prime_matvec_4bit: group must be 32, 64 or 128");
    if (n == 0 || rows == 0) return 0;
    if (!x || !packed || !scales || !out || (x_type == PRIME_I8) != (x_scales != nullptr))
        return fail(PRIME_EINVAL, "prime_matvec_4bit: null operand, or scales without int8 rows");
    const int64_t groups = (k + group - 1) / group;
    const int64_t scale_bytes = scale_stride > 0xffffffffLL ? scale_stride : scale_stride * type_bytes(scale_type);
    if (packed_stride > 0xffffffffLL || scale_bytes > 0xffffffffLL) return fail(PRIME_EINVAL, "prime_matvec_4bit: rows of codes or scales 4 GiB apart");
    MatvecArgs a{x, x_scales, packed, scales, out, x_stride, static_cast<uint32_t>(packed_stride), static_cast<uint32_t>(scale_bytes), static_cast<int>(rows), static_cast<int>(n), static_cast<int>(k),
                 static_cast<int>(groups * group / 2), static_cast<int>(groups), out_type, 0, 0, 0, 0};
    const double bytes = static_cast<double>(n) * k / 2 + static_cast<double>(n) * groups * type_bytes(scale_type) +
                         static_cast<double>(rows) * (k * type_bytes(x_type) + n * type_bytes(out_type));
    auto go = [&](auto t) { launch_matvec<decltype(t)>(a, group, scale_type, bytes, static_cast<hipStream_t>(stream)); };
    if (x_type == PRIME_I8) go(int8_t{});
    else with_float_type(x_type, go);
    return launch_check("matvec4_kernel");
}

}  // extern "C"
