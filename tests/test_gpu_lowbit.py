"""The low-bit operators on the GPU against plain 64-bit implementations on the CPU."""
import random

import pytest
import torch

from prime_amd import lowbit
from tests import lowbit_reference as ref
from tests.gpu_util import announce

pytestmark = pytest.mark.gpu

F32, BF16, F16, I8, E4M3 = torch.float32, torch.bfloat16, torch.float16, torch.int8, torch.float8_e4m3fn
NAMES = {F32: "fp32", BF16: "bf16", F16: "fp16", I8: "int8", E4M3: "e4m3"}


def gen(*key):
    return torch.Generator().manual_seed(random.Random(repr(key)).randrange(1 << 30))


def rows_like_activations(g, rows, dim, dtype):
    x = torch.randn(rows, dim, generator=g) * torch.exp(0.3 * torch.randn(dim, generator=g))
    x[:, :: max(1, dim // 3)] *= 8
    return x.to(dtype)


def check_norm(got, x, r, w, eps, dtype):
    codes, scales, hidden, inv = got
    wc, ws, wh, wi = ref.norm(x, r, w, eps, dtype)
    assert codes.dtype == dtype and scales.dtype == inv.dtype == F32
    if r is not None:
        assert torch.equal(hidden.cpu().double(), wh), "hidden"
    assert torch.equal(codes.cpu().float().double(), wc), "codes"
    # both are the 64-bit value rounded to 32 bits (sums of squares are fp64 on both sides): half a step each
    for name, a, b in (("scales", scales, ws), ("inv_rms", inv, wi)):
        d = (a.cpu().double() - b).abs() - 1.01 * 2.0 ** -24 * b.abs() - 2.0 ** -150
        assert float(d.max()) <= 0, (name, float(d.max()))


DIMS = [1, 2, 7, 8, 9, 63, 65, 511, 512, 513, 1024, 1025, 1999, 2048, 2049, 4096, 4100, 8191, 8200, 16384, 16385, 20011, 70000]


@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("types", [(BF16, F32), (BF16, BF16), (F16, F16), (F16, F32), (F32, F32)], ids=lambda t: f"{NAMES[t[0]]}-{NAMES[t[1]]}")
def test_norm_codes_are_exact(dev, dim, types):
    xt, wt = types
    g = gen("norm", dim, str(types))
    rows = 5 if dim <= 4096 else 2
    x, r = rows_like_activations(g, rows, dim, xt), rows_like_activations(g, rows, dim, xt)
    w = (1 + 0.2 * torch.randn(dim, generator=g)).to(wt)
    for dtype in (I8, E4M3):
        announce(f"norm dim={dim} {types} {dtype}")
        codes, scales, inv = lowbit.rms_norm_quantize(x.to(dev), w.to(dev), 1e-5, dtype)
        check_norm((codes, scales, None, inv), x, None, w, 1e-5, dtype)
        check_norm(lowbit.add_rms_norm_quantize(x.to(dev), r.to(dev), w.to(dev), 1e-6, dtype), x, r, w, 1e-6, dtype)


def test_norm_borders_between_codes_go_to_the_even_neighbour(dev):
    # the largest is 127 (448), so that the unit is 1 and every half is a tie; and one step either side of each
    for dtype, top in ((I8, 127.0), (E4M3, 448.0)):
        if dtype == I8:
            mids = torch.arange(-126.5, 127.0, 1.0)
        else:
            v = torch.arange(127, dtype=torch.uint8).view(E4M3).double()
            mids = ((v[1:] + v[:-1]) / 2).float()
            mids = torch.cat((mids, -mids))
        x = torch.stack([mids, torch.nextafter(mids, torch.full_like(mids, 1e9)), torch.nextafter(mids, torch.full_like(mids, -1e9))])
        x = torch.cat([torch.full((3, 1), top), x], 1)
        for unit in (1.0, 3.0, 2.0 ** -120, 0.7):
            xs = x * unit
            announce(f"borders {dtype} unit={unit}")
            codes, scales, inv = lowbit.rms_norm_quantize(xs.to(dev), torch.ones(xs.shape[1], device=dev), 1e-6, dtype)
            check_norm((codes, scales, None, inv), xs, None, torch.ones(xs.shape[1]), 1e-6, dtype)


def test_norm_rows_of_zeros_tiny_huge_and_not_finite(dev):
    dim = 300
    x = torch.randn(12, dim, generator=gen("special"))
    x[0] = 0
    x[1] *= 1e-42           # below the smallest normal number
    x[2] *= 1e-37
    x[3] *= 1e18            # squares beyond fp32
    x[4] *= 1e36
    x[5, 7] = float("nan")
    x[6, 299] = float("inf")
    x[7, 0] = -float("inf")
    x[8] = 0
    x[8, 5] = 1e-45         # a unit that rounds to zero
    x[9] = 3.0
    w = torch.ones(dim)
    for dtype in (I8, E4M3):
        announce(f"special rows {dtype}")
        codes, scales, inv = (t.cpu() for t in lowbit.rms_norm_quantize(x.to(dev), w.to(dev), 1e-6, dtype))
        fine = [i for i in range(12) if i not in (5, 6, 7)]
        check_norm((codes[fine], scales[fine], None, inv[fine]), x[fine], None, w, 1e-6, dtype)
        assert torch.isnan(scales[[5, 6, 7]]).all() and not codes.float()[[5, 6, 7]].any()
        assert not codes.float()[0].any() and scales[0] == 0 and not codes.float()[8].any()
    # a product that leaves fp32's range in a finite row; a weight of zeros; a sum that overflows its type
    codes, scales, inv = (t.cpu() for t in lowbit.rms_norm_quantize((x[4:5]).to(dev), (w * 1e30).to(dev)))
    assert torch.isnan(scales).all() and not codes.any() and torch.isfinite(inv).all()
    codes, scales, inv = (t.cpu() for t in lowbit.rms_norm_quantize(x[9:10].to(dev), (w * 0).to(dev)))
    assert scales[0] == 0 and not codes.any()
    big = torch.full((2, 64), 60000.0, dtype=F16)
    codes, scales, hidden, inv = (t.cpu() for t in lowbit.add_rms_norm_quantize(big.to(dev), big.to(dev), torch.ones(64, dtype=F16, device=dev)))
    assert torch.isinf(hidden).all() and torch.isnan(scales).all() and not codes.any()


def test_norm_takes_views_leading_dimensions_and_no_rows(dev):
    g = gen("views")
    base = rows_like_activations(g, 12, 400, BF16)
    w = 1 + 0.1 * torch.randn(130, generator=g)
    for view in (lambda t: t[:, 100:230], lambda t: t[::3, 7:137], lambda t: t.view(3, 4, 400)[:, 1:3, 40:170], lambda t: t[:1, :130].expand(6, 130),
                 lambda t: t.t()[:130].t(), lambda t: t[:, :260:2]):
        x = view(base)
        got = lowbit.rms_norm_quantize(view(base.to(dev)), w.to(dev))
        assert got[0].shape == x.shape and got[1].shape == x.shape[:-1]
        check_norm((got[0], got[1], None, got[2]), x, None, w, 1e-6, I8)
    got = lowbit.add_rms_norm_quantize(base.to(dev)[3, :130], base.to(dev)[4, :130], w.to(dev))           # one row without a leading dimension
    check_norm(got, base[3, :130], base[4, :130], w, 1e-6, I8)
    codes, scales, hidden, inv = lowbit.add_rms_norm_quantize(base.to(dev)[:0, :130], base.to(dev)[:0, :130], w.to(dev))
    assert codes.shape == hidden.shape == (0, 130) and scales.shape == inv.shape == (0,)
    gx, gw = lowbit.rms_norm_quantize_backward(hidden, hidden, w.to(dev), inv)
    assert gx.shape == (0, 130) and not gw.any() and gw.shape == (130,)


@pytest.mark.parametrize("rows,dim", [(1, 1), (3, 7), (2, 64), (9, 513), (70, 1024), (5, 1999), (300, 2048), (1, 4096), (77, 4100), (6, 8192), (3, 16383),
                                      (4, 16385), (2, 70000), (5000, 96)])
@pytest.mark.parametrize("types", [(BF16, F32), (BF16, BF16), (F16, F16), (F32, F32)], ids=lambda t: f"{NAMES[t[0]]}-{NAMES[t[1]]}")
def test_norm_gradients(dev, rows, dim, types):
    xt, wt = types
    g = gen("grad", rows, dim, str(types))
    h = rows_like_activations(g, rows, dim, xt)
    w = (1 + 0.2 * torch.randn(dim, generator=g)).to(wt)
    dy, dh = torch.randn(rows, dim, generator=g).to(xt), torch.randn(rows, dim, generator=g).to(xt)
    inv = (h.double().square().mean(-1) + 1e-6).rsqrt().float()
    for extra in (None, dh):
        announce(f"norm gradient {rows} x {dim} {types} {extra is not None}")
        gx, gw = lowbit.rms_norm_quantize_backward(dy.to(dev), h.to(dev), w.to(dev), inv.to(dev), None if extra is None else extra.to(dev))
        wx, ww, bx, bw = ref.norm_backward(dy, h, w, inv, extra)
        assert gx.dtype == xt and gw.dtype == wt
        assert ref.outside(gx.cpu(), wx, bx) <= 0 and ref.outside(gw.cpu(), ww, bw) <= 0
        again = lowbit.rms_norm_quantize_backward(dy.to(dev), h.to(dev), w.to(dev), inv.to(dev), None if extra is None else extra.to(dev))
        assert torch.equal(again[0], gx) and torch.equal(again[1], gw)          # sums in a fixed order


def test_norm_gradients_against_differences(dev):
    # f(x, w) = sum(dy * norm(x) * w) in 64 bits, central differences
    g = gen("differences")
    rows, dim, eps, step = 3, 40, 1e-3, 1e-5
    x, w, dy = (torch.randn(*s, generator=g, dtype=torch.float64).float().double() for s in ((rows, dim), (dim,), (rows, dim)))

    def f(x, w):
        return float((dy * x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) * w).sum())

    inv = torch.rsqrt((x * x).mean(-1) + eps).float()
    gx, gw = lowbit.rms_norm_quantize_backward(dy.float().to(dev), x.float().to(dev), w.float().to(dev), inv.to(dev))
    # differences: step^2 / 6 times the third derivative (a few units) and 1e-16 * |f| / step = 1e-9 of rounding; 32-bit sums: 1e-6
    for i in range(rows):
        for j in range(0, dim, 7):
            e = torch.zeros_like(x)
            e[i, j] = step
            assert abs((f(x + e, w) - f(x - e, w)) / (2 * step) - float(gx[i, j])) < 2e-5
    for j in range(dim):
        e = torch.zeros_like(w)
        e[j] = step
        assert abs((f(x, w + e) - f(x, w - e)) / (2 * step) - float(gw[j])) < 2e-5


def test_norm_gradients_take_views_and_a_repeated_row(dev):
    g = gen("grad views")
    h = rows_like_activations(g, 6, 300, BF16)
    dy = torch.randn(6, 300, generator=g).to(BF16)
    w = 1 + 0.1 * torch.randn(150, generator=g)
    inv = (h[:, 20:170].double().square().mean(-1) + 1e-6).rsqrt().float()
    one = dy[:1, :150].expand(6, 150)
    gx, gw = lowbit.rms_norm_quantize_backward(dy.to(dev)[:1, :150].expand(6, 150), h.to(dev)[:, 20:170], w.to(dev), inv.to(dev), dy.to(dev)[:, 3:153])
    wx, ww, bx, bw = ref.norm_backward(one, h[:, 20:170], w, inv, dy[:, 3:153])
    assert ref.outside(gx.cpu(), wx, bx) <= 0 and ref.outside(gw.cpu(), ww, bw) <= 0


SHAPES = [(1, 1), (1, 32), (3, 31), (5, 33), (2, 127), (16, 128), (17, 129), (33, 256), (7, 1000), (64, 2048), (129, 5000)]


@pytest.mark.parametrize("n,k", SHAPES)
@pytest.mark.parametrize("group", [32, 64, 128])
def test_quantize_4bit_is_exact_and_its_matrix_comes_back(dev, n, k, group):
    g = gen("pack", n, k, group)
    for wt in (F32, BF16, F16):
        for st in (F32, BF16):
            announce(f"4 bits {n} x {k} group {group} {wt} {st}")
            w = (0.02 * torch.randn(n, k, generator=g)).to(wt)
            w[:, ::5] = w[:, ::5] * 3
            if n > 2:
                w[1] = 0
            codes, s = ref.quantize_4bit(w, group, st)
            packed, scales = lowbit.quantize_4bit(w.to(dev), group, st)
            assert scales.dtype == st and torch.equal(scales.cpu(), s) and torch.equal(packed.cpu(), ref.pack(codes))
            values = codes.float() * s.float().repeat_interleave(group, 1)
            for dt in (F32, BF16, F16):
                got = lowbit.dequantize_4bit(packed, scales, k, dt)
                assert got.dtype == dt and torch.equal(got.cpu(), values[:, :k].to(dt))
            assert torch.equal(lowbit.dequantize_4bit(packed, scales).cpu(), values)


def test_quantize_4bit_borders_and_special_groups(dev):
    mids = torch.arange(-6.5, 7.0, 1.0)
    row = torch.cat([torch.tensor([7.0]), mids, torch.nextafter(mids, torch.tensor(99.0)), torch.nextafter(mids, torch.tensor(-99.0))])
    w = torch.zeros(9, 64)
    for i, unit in enumerate((1.0, 3.0, 0.7, 2.0 ** -120, 2.0 ** 100, 2.0 ** -149)):
        w[i, : len(row)] = row * unit
    w[6, 40] = float("nan")
    w[7, 3] = -float("inf")
    for group in (32, 64):
        for st in (F32, BF16):
            fine = [0, 1, 2, 3, 4, 5, 8]
            codes, s = ref.quantize_4bit(w[fine], group, st)
            packed, scales = (t.cpu() for t in lowbit.quantize_4bit(w.to(dev), group, st))
            assert torch.equal(scales[fine], s) and torch.equal(packed[fine], ref.pack(codes))
            assert torch.isnan(scales[6, 40 // group]) and torch.isnan(scales[7, 0]) and not packed[6:8].any()
            if group == 32:
                assert scales[6, 0] == 0 and scales[7, 1] == 0


def test_quantize_4bit_takes_views(dev):
    w = torch.randn(40, 300, generator=gen("w views"))
    for view in (lambda t: t[::2, 5:205], lambda t: t.t()[:150].t(), lambda t: t[:1, :70].expand(5, 70), lambda t: t[:0, :70]):
        codes, s = ref.quantize_4bit(view(w), 64, F32)
        packed, scales = lowbit.quantize_4bit(view(w.to(dev)), 64, F32)
        assert torch.equal(scales.cpu(), s) and torch.equal(packed.cpu(), ref.pack(codes))


def four_bit(g, n, k, group, st):
    groups = -(-k // group)
    codes = torch.randint(-8, 8, (n, groups * group), generator=g, dtype=torch.int8)       # also behind the row's end: not to be read
    return codes, (0.01 * torch.exp(0.5 * torch.randn(n, groups, generator=g))).to(st)


def check_matvec(dev, x, xs, codes, s, k, dt=None):
    got = lowbit.matvec_4bit(x.to(dev), ref.pack(codes).to(dev), s.to(dev), None if xs is None else xs.to(dev), dt)
    assert got.dtype == (dt or (F32 if x.dtype == I8 else x.dtype)) and got.shape == x.shape[:-1] + (codes.shape[0],)
    want, bound = ref.matvec(x, xs, codes, s, k)
    assert ref.outside(got.cpu(), want, bound) <= 0
    return got


@pytest.mark.parametrize("n,k", [(1, 1), (1, 32), (5, 31), (16, 64), (17, 129), (100, 1000), (33, 2048), (15, 5604), (4099, 130), (48, 20000)])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("xt", [BF16, F16, F32, I8], ids=NAMES.get)
def test_matvec_4bit(dev, n, k, group, xt):
    g = gen("matvec", n, k, group, str(xt))
    for rows in ((1, 3, 5, 16) if n * k < 100000 else (1, 8)):
        for st in (F32, BF16):
            announce(f"matvec {rows} x {k} x {n} group {group} {xt} {st}")
            codes, s = four_bit(g, n, k, group, st)
            x = rows_like_activations(g, rows, k, F32)
            xs = None
            if xt == I8:
                x, xs = torch.randint(-127, 128, (rows, k), generator=g).to(I8), torch.rand(rows, generator=g) * 0.05
            check_matvec(dev, x.to(xt), xs, codes, s, k)


@pytest.mark.parametrize("rows", [2, 4, 9, 12, 17, 31, 32, 33, 48, 63, 64, 65, 100, 130, 300])
@pytest.mark.parametrize("xt", [BF16, F16, F32, I8], ids=NAMES.get)
def test_matvec_4bit_rows(dev, rows, xt):
    g = gen("rows", rows, str(xt))
    for n, k, group, st in ((70, 1100, 32, BF16), (40, 640, 64, F32), (129, 900, 128, BF16)):
        announce(f"matvec {rows} x {k} x {n} group {group} {xt}")
        codes, s = four_bit(g, n, k, group, st)
        x = rows_like_activations(g, rows, k, F32)
        xs = None
        if xt == I8:
            x, xs = torch.randint(-127, 128, (rows, k), generator=g).to(I8), torch.rand(rows, generator=g) * 0.05
        for dt in (F32, BF16, F16):
            check_matvec(dev, x.to(xt), xs, codes, s, k, dt)


@pytest.mark.parametrize("rows,n,k", [(24, 4200, 700), (64, 2090, 4300), (70, 2100, 2100), (9, 8300, 6000)])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("xt", [BF16, F16, F32, I8], ids=NAMES.get)
def test_matvec_4bit_many_rows_and_outputs(dev, rows, n, k, group, xt):
    # more tiles of 16 rows by 32 outputs than compute units: the kernels that take 32 and 64 rows at a time, rows in several visits
    g = gen("many", rows, n, k, group, str(xt))
    for st in (F32, BF16):
        announce(f"matvec {rows} x {k} x {n} group {group} {xt} {st}")
        codes, s = four_bit(g, n, k, group, st)
        x, xs = rows_like_activations(g, rows, k, F32), None
        if xt == I8:
            x, xs = torch.randint(-128, 128, (rows, k), generator=g).to(I8), torch.rand(rows, generator=g) * 0.05
        check_matvec(dev, x.to(xt), xs, codes, s, k)


def test_offsets_beyond_32_bits(dev):
    g = gen("far")
    announce("rows far apart")
    base = torch.zeros(40, 1 << 27, dtype=torch.uint8, device=dev)          # 5 GiB: row 32 starts at 2^32
    codes, s = four_bit(g, 40, 96, 32, F32)
    packed = base[:, 1000:1048]
    packed.copy_(ref.pack(codes))
    x = rows_like_activations(g, 6, 96, BF16)
    for rows in (1, 6):
        got = lowbit.matvec_4bit(x[:rows].to(dev), packed, s.to(dev))
        want, bound = ref.matvec(x[:rows], None, codes, s, 96)
        assert ref.outside(got.cpu(), want, bound) <= 0
    assert torch.equal(lowbit.dequantize_4bit(packed, s.to(dev)).cpu(), codes.float() * s.repeat_interleave(32, 1))
    view = base.view(torch.bfloat16)[:, 512:812]
    x = rows_like_activations(g, 40, 300, BF16)
    view.copy_(x)
    w = 1 + 0.1 * torch.randn(300, generator=g)
    codes8, scales, inv = lowbit.rms_norm_quantize(view, w.to(dev))
    check_norm((codes8, scales, None, inv), x, None, w, 1e-6, I8)
    wx, ww, bx, bw = ref.norm_backward(x, x, w, inv.cpu())
    gx, gw = lowbit.rms_norm_quantize_backward(view, view, w.to(dev), inv)
    assert ref.outside(gx.cpu(), wx, bx) <= 0 and ref.outside(gw.cpu(), ww, bw) <= 0
    want4, ws = ref.quantize_4bit(x, 64, BF16)
    got4, gs = lowbit.quantize_4bit(view, 64, BF16)
    assert torch.equal(got4.cpu(), ref.pack(want4)) and torch.equal(gs.cpu(), ws)


def test_large_codes_and_outputs_leave_their_neighbours_alone(dev):
    # outputs are written inside their own tensors only: guards on both sides of every output of the C calls
    from prime_amd import _lib

    lib = _lib.load()
    st = torch.cuda.current_stream(dev).cuda_stream
    g = gen("guards")
    for rows, dim in ((3, 77), (5, 1030), (2, 5001)):
        x, w = rows_like_activations(g, rows, dim, BF16).to(dev), torch.ones(dim, device=dev)
        out = torch.full((rows * dim + 128,), 0x5A, dtype=torch.uint8, device=dev)
        sc = torch.full((2 * rows + 128,), 7.0, device=dev)
        hid = torch.full((rows * dim + 128,), 9.0, dtype=BF16, device=dev)
        rc = lib.prime_rms_norm_quantize(x.data_ptr(), dim, x.data_ptr(), dim, w.data_ptr(), rows, dim, 1, 0, 3, 1e-6, out[64:].data_ptr(),
                                         sc[64:].data_ptr(), hid[64:].data_ptr(), sc[64 + rows:].data_ptr(), st)
        assert rc == 0
        assert (out[:64] == 0x5A).all() and (out[64 + rows * dim:] == 0x5A).all()
        assert (sc[:64] == 7).all() and (sc[64 + 2 * rows:] == 7).all() and (hid[:64] == 9).all() and (hid[64 + rows * dim:] == 9).all()
    for rows, n, k in ((1, 37, 300), (9, 37, 300), (20, 4099, 130), (70, 2061, 200)):
        codes, s = four_bit(g, n, k, 64, F32)
        packed, sd, x = ref.pack(codes).to(dev), s.to(dev), rows_like_activations(g, rows, k, BF16).to(dev)
        y = torch.full((rows * n + 128,), 3.0, device=dev)
        rc = lib.prime_matvec_4bit(x.data_ptr(), k, 1, None, packed.data_ptr(), packed.stride(0), sd.data_ptr(), sd.stride(0), rows, n, k, 64, 0,
                                   y[64:].data_ptr(), 0, st)
        assert rc == 0 and (y[:64] == 3).all() and (y[64 + rows * n:] == 3).all()


def test_outer_weights_in_4_bits(dev):
    from prime_amd.diloco import Diloco

    torch.manual_seed(3)
    model = torch.nn.Sequential(torch.nn.Linear(130, 70), torch.nn.LayerNorm(70), torch.nn.Linear(70, 33, bias=False)).to(dev)
    d = Diloco(0.7, model)
    start = {n: p.detach().cpu().clone() for n, p in model.named_parameters()}
    with torch.no_grad():
        for p in model.parameters():
            p.add_(0.1)                          # inner training: the outer copy stays
    got = d.outer_weights_4bit(model, 64, F32)
    assert set(got) == {"0.weight", "2.weight"}
    for name, (packed, scales) in got.items():
        codes, s = ref.quantize_4bit(start[name], 64, F32)
        assert torch.equal(packed.cpu(), ref.pack(codes)) and torch.equal(scales.cpu(), s)
    x = torch.randn(1, 130, generator=gen("outer"))
    y = lowbit.matvec_4bit(x.to(dev), *got["0.weight"])
    codes, s = ref.quantize_4bit(start["0.weight"], 64, F32)
    want, bound = ref.matvec(x, None, codes, s, 130)
    assert ref.outside(y.cpu(), want, bound) <= 0


def test_matvec_4bit_rows_are_independent_and_each_sees_what_is_not_finite(dev):
    g = gen("special matvec")
    for xt in (BF16, F16, F32):
        for group in (32, 64, 128):
            codes, s = four_bit(g, 50, 300, group, F32)
            x = torch.randn(6, 300, generator=g).to(xt)
            packed, sd = ref.pack(codes).to(dev), s.to(dev)
            clean = lowbit.matvec_4bit(x.to(dev), packed, sd)
            x[1, 299] = float("nan")
            x[3, 0] = float("inf")
            x[4] = 0
            got = lowbit.matvec_4bit(x.to(dev), packed, sd).cpu()
            assert torch.equal(got[[0, 2, 5]], clean.cpu()[[0, 2, 5]])                  # the other rows are left alone
            assert torch.isnan(got[1]).all() and not got[4].any() and not torch.isfinite(got[3][codes[:, 0] != 0]).any()
            # a scale that is not a number spoils its output alone
            s2 = s.clone()
            s2[7, 1] = float("nan")
            got = lowbit.matvec_4bit(x[:1].to(dev), packed, s2.to(dev)).cpu()
            assert torch.isnan(got[0, 7]) and int(torch.isnan(got).sum()) == 1


def test_matvec_4bit_takes_views_and_leading_dimensions(dev):
    g = gen("matvec views")
    codes, s = four_bit(g, 96, 512, 64, BF16)
    packed, sd = ref.pack(codes).to(dev), s.to(dev)
    x = rows_like_activations(g, 12, 700, BF16)
    for view in (lambda t: t[:, 100:612], lambda t: t[::3, 1:513], lambda t: t.view(3, 4, 700)[:, 1:3, :512], lambda t: t[:1, :512].expand(5, 512),
                 lambda t: t[0, :512], lambda t: t[:0, :512]):
        got = lowbit.matvec_4bit(view(x.to(dev)), packed, sd)
        want, bound = ref.matvec(view(x), None, codes, s, 512)
        assert got.shape == view(x).shape[:-1] + (96,) and ref.outside(got.cpu(), want, bound) <= 0
    # a block of rows and of groups of a larger matrix: what a rank of a tensor-parallel model holds
    got = lowbit.matvec_4bit(x.to(dev)[:3, :256], packed[32:64, 64:192], sd[32:64, 2:6])
    want, bound = ref.matvec(x[:3, :256], None, codes[32:64, 128:384], s[32:64, 2:6], 256)
    assert ref.outside(got.cpu(), want, bound) <= 0
    part = lowbit.dequantize_4bit(packed[32:64, 64:192], sd[32:64, 2:6])
    assert torch.equal(part.cpu(), (codes.float() * s.float().repeat_interleave(64, 1))[32:64, 128:384])


def test_a_block_of_a_decoding_step_and_its_graph(dev):
    """norm with residual -> 4-bit product on its codes -> activation -> 4-bit product -> norm: eager, on another stream, and
    captured and replayed on fresh inputs with eager work in between."""
    g = gen("block")
    dim, ffn = 2048, 5632
    w1 = (0.02 * torch.randn(dim, generator=g)).add(1).to(dev)
    up, us = lowbit.quantize_4bit((0.02 * torch.randn(ffn, dim, generator=g)).to(dev), 128)
    down, ds = lowbit.quantize_4bit((0.02 * torch.randn(dim, ffn, generator=g)).to(dev), 64, F32)

    def block(x, r):
        codes, scales, hidden, _ = lowbit.add_rms_norm_quantize(x, r, w1)
        y = lowbit.matvec_4bit(codes, up, us, scales, BF16)
        y = lowbit.matvec_4bit(torch.nn.functional.silu(y), down, ds)
        return lowbit.add_rms_norm_quantize(y, hidden, w1, 1e-6, E4M3) + (y,)

    inputs = [tuple(rows_like_activations(g, 4, dim, BF16).to(dev) for _ in range(2)) for _ in range(4)]
    eager = [block(*i) for i in inputs]
    # the formulas, in 64 bits, from the framework's own intermediate values where a rounding decides
    for (x, r), (codes, scales, hidden, inv, y) in zip(inputs, eager):
        c, s, h, _ = ref.norm(x.cpu(), r.cpu(), w1.cpu(), 1e-6, I8)
        wide = lowbit.dequantize_4bit(up, us).cpu().double()
        v = (c * s.unsqueeze(-1)) @ wide.T
        a, sig = torch.nn.functional.silu(v), torch.sigmoid(v)
        want = a @ lowbit.dequantize_4bit(down, ds).cpu().double().T
        # v is rounded to bf16, which silu passes on by its slope; silu's value is rounded again; the product a third time
        inner = 2.0 ** -8 * ((sig * (1 + v * (1 - sig)) * v).abs() + a.abs()) * 1.05
        bound = inner @ lowbit.dequantize_4bit(down, ds).cpu().double().abs().T
        bound = bound + 2.0 ** -8 * (want.abs() + bound)
        assert float(((y.cpu().double() - want).abs() - bound).max()) <= 0
        check_norm((codes, scales, hidden, inv), y.cpu(), h.to(BF16), w1.cpu(), 1e-6, E4M3)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = block(*inputs[1])
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(other, eager[1]))
    static = tuple(t.clone() for t in inputs[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = block(*static)
    for turn in range(3):
        for i, want in zip(inputs, eager):
            for a, b in zip(static, i):
                a.copy_(b)
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(out, want))
            block(*inputs[turn])


def test_a_training_step_through_an_autograd_function_and_its_graph(dev):
    """The pair of norm and gradient inside a torch.autograd.Function: what a training step does with them, also captured."""

    class Norm(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, residual, weight):
            codes, scales, hidden, inv = lowbit.add_rms_norm_quantize(x, residual, weight, 1e-6)
            ctx.save_for_backward(hidden, weight, inv)
            return codes.float() * scales.unsqueeze(-1), hidden

        @staticmethod
        def backward(ctx, grad, grad_hidden):
            hidden, weight, inv = ctx.saved_tensors
            gx, gw = lowbit.rms_norm_quantize_backward(grad.to(hidden.dtype), hidden, weight, inv, grad_hidden)
            return gx, gx, gw

    g = gen("training")
    x, r = rows_like_activations(g, 50, 1030, F32), rows_like_activations(g, 50, 1030, F32)
    w = 1 + 0.1 * torch.randn(1030, generator=g)
    dy, dh = torch.randn(50, 1030, generator=g), torch.randn(50, 1030, generator=g)
    xd, rd, wd = (t.to(dev).requires_grad_() for t in (x, r, w))
    y, h = Norm.apply(xd, rd, wd)
    torch.autograd.backward((y, h), (dy.to(dev), dh.to(dev)))
    _, _, wh, wi = ref.norm(x, r, w, 1e-6, I8)
    wx, ww, bx, bw = ref.norm_backward(dy, wh.float(), w, wi.float(), dh)
    # inv_rms may be the neighbouring 32-bit number: two steps more, relative to every term
    more = 2.0 ** -22
    assert ref.outside(xd.grad.cpu(), wx, bx + more * (wx.abs() + wi.unsqueeze(-1) * (dy * w).abs() + 4 * dh.abs())) <= 0
    assert torch.equal(xd.grad, rd.grad) and ref.outside(wd.grad.cpu(), ww, bw + more * ww.abs() + more * (dy * wh * wi.unsqueeze(-1)).abs().sum(0)) <= 0
    # the two calls captured, with the framework's own tensors
    static = [t.to(dev).clone() for t in (x, r, w, dy, dh)]

    def step():
        codes, scales, hidden, inv = lowbit.add_rms_norm_quantize(static[0], static[1], static[2])
        return (codes, scales, hidden, inv) + lowbit.rms_norm_quantize_backward(static[3], hidden, static[2], inv, static[4])

    want = [t.clone() for t in step()]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(3):
        for t in out:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
        step()


def test_two_streams_at_once_share_nothing(dev):
    g = gen("streams")
    sets = [(torch.randn(600, 1500, generator=g).to(dev), (torch.randn(600, 1500, generator=g)).to(dev)) for _ in range(2)]
    w = torch.ones(1500, device=dev)
    packed, s = lowbit.quantize_4bit(torch.randn(3000, 1500, generator=g).to(dev), 32)

    def work(x, dy):
        codes, scales, inv = lowbit.rms_norm_quantize(x, w)
        return lowbit.rms_norm_quantize_backward(dy, x, w, inv) + (lowbit.matvec_4bit(codes[:9], packed, s, scales[:9]), lowbit.matvec_4bit(x[:1], packed, s))

    want = [work(*i) for i in sets]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for st in streams:
        st.wait_stream(torch.cuda.current_stream())
    for _ in range(6):
        for k, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[k].append(work(*sets[k]))
    torch.cuda.synchronize()
    for k in range(2):
        for one in got[k]:
            assert all(torch.equal(a, b) for a, b in zip(one, want[k]))


def test_calls_that_record_gradients_are_refused_on_the_gpu(dev):
    x = torch.randn(3, 64, device=dev)
    w = torch.nn.Parameter(torch.ones(64, device=dev))
    with pytest.raises(RuntimeError, match="no gradient"):
        lowbit.rms_norm_quantize(x, w)
    with torch.no_grad():
        lowbit.rms_norm_quantize(x, w)
    # through the dispatcher as well
    with pytest.raises(RuntimeError, match="no gradient"):
        torch.ops.prime_lowbit.rms_norm_quantize(x, w)
    assert torch.equal(torch.ops.prime_lowbit.rms_norm_quantize(x, w.detach())[0], lowbit.rms_norm_quantize(x, w.detach())[0])


def test_norm_and_gradients_of_one_very_long_row(dev):
    # 2^27 columns: 32 work-items a column for the sum over rows are one dispatch more than 32 bits count
    dim = (1 << 27) + 41
    announce("norm gradient 1 x 2^27 + 41")
    g = torch.Generator(device=dev).manual_seed(7)
    h, dy = (torch.randn(1, dim, device=dev, generator=g).to(BF16) for _ in range(2))
    w = torch.rand(dim, device=dev, generator=g) + 0.5
    inv = (h.double().square().mean(-1) + 1e-6).rsqrt().float()
    gx, gw = lowbit.rms_norm_quantize_backward(dy, h, w, inv)
    assert torch.equal(gw, (dy.float() * (h.float() * inv))[0])            # one row: two roundings, the same ones
    wx, _, bx, _ = ref.norm_backward(dy, h, w, inv)
    assert ref.outside(gx, wx, bx) <= 0
    del wx, bx
    codes, scales, got_inv = lowbit.rms_norm_quantize(h, w)
    unit = (h.float() * w).abs().max() / 127
    assert torch.equal(got_inv, inv) and abs(float(scales[0]) - float(unit.double() * inv.double())) <= 2.0 ** -23 * float(scales[0])
    assert torch.equal(codes, torch.round((h.float() * w).double() / unit.double()).clamp(-127, 127).to(I8))


@pytest.mark.parametrize("xt", [F16, F32], ids=NAMES.get)
def test_matvec_4bit_of_the_most_rows(dev, xt):
    # 2^31 - 1 rows, the most a call takes: their number of tiles is rounded up in 64 bits
    rows = (1 << 31) - 1
    announce(f"matvec of 2^31 - 1 rows {xt}")
    codes = torch.arange(-8, 8, dtype=torch.int8).repeat(2).view(1, 32)
    x = torch.arange(1, 33).to(xt)
    got = lowbit.matvec_4bit(x.to(dev).expand(rows, 32), ref.pack(codes).to(dev), torch.ones(1, 1, device=dev), None, F16)
    want = float((x.double() * codes.double()).sum())          # every sum of the products is a whole number, and fp16 holds it
    assert got.shape == (rows, 1) and want == 416
    for part in got.view(-1).split(1 << 28):
        assert bool((part == want).all())


# ---- floating rows: more of them than are taken as a decoding step's few (5 and up), then few ----

FLOATS = [BF16, F16, F32]


def check_matvec_closely(dev, x, codes, s, k):
    got = lowbit.matvec_4bit(x.to(dev), ref.pack(codes).to(dev), s.to(dev), None, F32)
    want, _ = ref.matvec(x, None, codes, s, k)
    assert torch.isfinite(got).all() and ref.outside(got.cpu(), want, ref.matvec_bound(x, codes, s, k)) <= 0
    return got.cpu()


def check_large_columns_under_zero_codes(dev, rows, xt):
    # what a large column leaves where its code is 0 is nothing: neither its rounding nor its range shows in the other columns' sum
    for n, k, group in ((40, 128, 128), (33, 700, 32), (70, 2100, 64)):
        for far in (13, 20, 60) if xt != F16 else (13, 15):
            g = gen("large columns", rows, str(xt), k, group, far)
            announce(f"matvec {rows} x {k} x {n} group {group} {xt}: columns of 2^{far} under zeros")
            codes, s = four_bit(g, n, k, group, F32)
            x = torch.randn(rows, k, generator=g)
            large = torch.randperm(k, generator=g)[: max(1, k // 50)]
            x[:, large] = 2.0 ** far * (0.5 + torch.rand(rows, len(large), generator=g))
            codes[:, large] = 0
            codes[5] = 0                                                    # an output of zeros stays one
            got = check_matvec_closely(dev, x.to(xt), codes, s, k)
            assert not got[:, 5].any()
    # one column of 1e10 (1e4) under a zero, 127 ones under ones
    codes, s = torch.ones(3, 128, dtype=torch.int8), torch.ones(3, 1)
    codes[:, 0] = 0
    x = torch.ones(rows, 128)
    x[:, 0] = 1e10 if xt != F16 else 6e4
    assert bool((lowbit.matvec_4bit(x.to(xt).to(dev), ref.pack(codes).to(dev), s.to(dev), None, F32) == 127).all())


def check_the_range_of_columns(dev, rows, xt):
    # up to 2^120 in magnitude a finite product is finite, whatever the scale takes off afterwards; small columns keep their bits
    for group in (32, 64, 128):
        codes = torch.full((20, 256), 7, dtype=torch.int8)
        codes[1::2] = -8
        for top, scale in ((116.0, 0.5), (120.0, 2.0 ** -20), (15.0, 1.0), (-100.0, 2.0 ** 60), (-108.0, 2.0 ** 80)):
            if xt == F16 and top != 15.0:
                continue
            announce(f"matvec {rows} x 256 x 20 group {group} {xt}: columns of 2^{top}")
            s = torch.full((20, 256 // group), scale)
            x = torch.full((rows, 256), 2.0 ** top)
            want = x.double() @ (codes.double() * scale).T
            got = lowbit.matvec_4bit(x.to(xt).to(dev), ref.pack(codes).to(dev), s.to(dev), None, F32)
            assert torch.equal(got.cpu().double(), want)                    # equal columns: every sum has few bits
            x = torch.randn(rows, 256, generator=gen("range", rows, str(xt), group)).clamp(-3, 3) * 2.0 ** (top - 2)
            mixed, _ = four_bit(gen("range codes", group), 20, 256, group, F32)
            check_matvec_closely(dev, x.to(xt), mixed, s, 256)


def check_whole_numbers(dev, rows, xt, sizes):
    # sixteenths up to 8 and scales of 1/2, 1 and 2: every sum, in every order, is a multiple of 2^-5 below 2^19, so nothing is rounded, and
    # a column that is lost, doubled or met with another's code shows
    for n, k, group in sizes:
        g = gen("whole", rows, str(xt), n, k, group)
        announce(f"matvec {rows} x {k} x {n} group {group} {xt}: whole numbers")
        codes, _ = four_bit(g, n, k, group, F32)
        s = 2.0 ** torch.randint(-1, 2, (n, codes.shape[1] // group), generator=g).float()
        x = torch.randint(-127, 128, (rows, k), generator=g) / 16
        weights = codes[:, :k].double() * s.double().repeat_interleave(group, 1)[:, :k]
        assert float((x.double().abs() @ weights.abs().T).max()) < 2 ** 19
        got = lowbit.matvec_4bit(x.to(xt).to(dev), ref.pack(codes).to(dev), s.to(dev), None, F32)
        assert torch.equal(got.cpu().double(), x.double() @ weights.T)


def check_single_columns(dev, rows, xt):
    # one column that is not 0 in a row, of as many bits as its type has.  16-bit columns: the product has at most 11 + 3 bits and is exact.  fp32: its
    # three parts of 8 bits give products of 11; the first two add up to 19 bits, exactly, and the third addition alone is inexact.  The
    # matrix unit is free to cut off what it does not hold, so that addition is off by less than a whole step of the sum, 2^-23 of it
    # (half a step if it rounds); the factors behind it are powers of two
    for group in (32, 64, 128):
        g = gen("single", rows, str(xt), group)
        codes, _ = four_bit(g, 50, 600, group, F32)
        s = 2.0 ** torch.randint(-1, 2, (50, codes.shape[1] // group), generator=g).float()
        x = torch.zeros(rows, 600, dtype=xt)
        for m in range(rows):
            x[m, int(torch.randint(0, 600, (1,), generator=g))] = torch.randn(1, generator=g).to(xt)[0]
        got = lowbit.matvec_4bit(x.to(dev), ref.pack(codes).to(dev), s.to(dev), None, F32)
        want, _ = ref.matvec(x, None, codes, s, 600)
        assert bool(((got.cpu().double() - want).abs() <= (2.0 ** -23 * want.abs() if xt == F32 else 0.0)).all())


@pytest.mark.parametrize("rows", [5, 16, 20, 40, 64])
@pytest.mark.parametrize("xt", FLOATS, ids=NAMES.get)
def test_matvec_4bit_many_rows_with_large_columns_under_zero_codes(dev, rows, xt):
    check_large_columns_under_zero_codes(dev, rows, xt)


@pytest.mark.parametrize("rows", [5, 40, 64])
@pytest.mark.parametrize("xt", FLOATS, ids=NAMES.get)
def test_matvec_4bit_many_rows_range_of_columns(dev, rows, xt):
    check_the_range_of_columns(dev, rows, xt)


@pytest.mark.parametrize("rows", [5, 16, 30, 64])
@pytest.mark.parametrize("xt", FLOATS, ids=NAMES.get)
def test_matvec_4bit_many_rows_of_whole_numbers(dev, rows, xt):
    check_whole_numbers(dev, rows, xt, ((48, 20000, 32), (48, 20000, 128), (600, 6000, 64), (4200, 2100, 128)))
    check_single_columns(dev, rows, xt)


@pytest.mark.parametrize("rows", [1, 2, 3, 4])
@pytest.mark.parametrize("xt", FLOATS, ids=NAMES.get)
def test_matvec_4bit_few_rows_with_large_columns_under_zero_codes(dev, rows, xt):
    check_large_columns_under_zero_codes(dev, rows, xt)


@pytest.mark.parametrize("rows", [1, 4])
@pytest.mark.parametrize("xt", FLOATS, ids=NAMES.get)
def test_matvec_4bit_few_rows_range_of_columns(dev, rows, xt):
    check_the_range_of_columns(dev, rows, xt)


@pytest.mark.parametrize("rows", [1, 2, 3, 4])
@pytest.mark.parametrize("xt", FLOATS, ids=NAMES.get)
def test_matvec_4bit_few_rows_of_whole_numbers(dev, rows, xt):
    # rows that LDS holds whole and rows that it takes in stretches, columns shared by one to eight wavefronts, one tile a workgroup and several
    check_whole_numbers(dev, rows, xt, ((48, 20000, 32), (48, 20000, 128), (600, 6000, 64), (9000, 2100, 128), (70001, 130, 64)))
    check_single_columns(dev, rows, xt)
    # longer than LDS holds of one 16-bit row
    g = gen("longest", rows, str(xt))
    codes, s = four_bit(g, 40, 30000, 128, F32)
    check_matvec_closely(dev, rows_like_activations(g, rows, 30000, xt), codes, s, 30000)


@pytest.mark.parametrize("rows", [1, 4, 5, 20])
def test_matvec_4bit_columns_of_the_smallest_magnitudes(dev, rows):
    # columns that are subnormal in their type, under a scale that brings the products back; fp32 columns down to bf16's smallest step
    announce(f"matvec {rows} rows of the smallest magnitudes")
    g = gen("smallest", rows)
    codes, _ = four_bit(g, 20, 128, 64, F32)
    for xt, top, scale in ((F16, -24, 1024.0), (BF16, -133, 2.0 ** 100), (F32, -133, 2.0 ** 100)):
        x = torch.randint(-3, 4, (rows, 128), generator=g).double() * 2.0 ** top
        s = torch.full((20, 2), scale)
        got = lowbit.matvec_4bit(x.to(xt).to(dev), ref.pack(codes).to(dev), s.to(dev), None, F32)
        assert torch.equal(got.cpu().double(), x @ (codes.double() * scale).T)


@pytest.mark.parametrize("rows", [1, 4, 5, 20, 40])
def test_matvec_4bit_int8_rows_between_large_and_small_scales(dev, rows):
    # sums of code x scale up to fp32's last power of two and row scales down to its smallest normal number, and the other way round
    for group in (32, 64, 128):
        for scale, x_scale in ((2.0 ** 110, 2.0 ** -126), (2.0 ** -126, 2.0 ** 110), (2.0 ** 110, 1.5 * 2.0 ** -130)):
            announce(f"matvec {rows} x 128 x 20 group {group} int8, scales {scale:g} and {x_scale:g}")
            codes = torch.full((20, 128), 7, dtype=torch.int8)
            codes[1::2] = -8
            x = torch.full((rows, 128), 127, dtype=I8)
            s, xs = torch.full((20, 128 // group), scale), torch.full((rows,), x_scale)
            got = lowbit.matvec_4bit(x.to(dev), ref.pack(codes).to(dev), s.to(dev), xs.to(dev))
            want = (x.double() @ (codes.double() * scale).T) * xs.double().unsqueeze(-1)      # 17 bits at most: exact
            assert torch.equal(got.cpu().double(), want)


def test_compiled_traced_and_transformed_calls_reach_the_ops(dev):
    from torch.autograd import forward_ad
    from torch.fx.experimental.proxy_tensor import make_fx

    g = gen("traced")
    x, r = rows_like_activations(g, 6, 200, F32).to(dev), rows_like_activations(g, 6, 200, F32).to(dev)
    w = (1 + 0.1 * torch.randn(200, generator=g)).to(dev)

    def step(x, r, w):
        codes, scales, hidden, inv = lowbit.add_rms_norm_quantize(x, r, w)
        packed, s = lowbit.quantize_4bit(hidden, 32)
        y = lowbit.matvec_4bit(codes, packed, s, scales)
        return (y, lowbit.dequantize_4bit(packed, s, 200)) + lowbit.rms_norm_quantize_backward(hidden, x, w, inv)

    want = step(x, r, w)
    torch._dynamo.reset()
    got = torch.compile(step, backend="eager", fullgraph=True)(x, r, w)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = make_fx(step)(x, r, w)
    assert sum("prime_lowbit" in str(n.target) for n in graph.graph.nodes) == 5
    assert all(torch.equal(a, b) for a, b in zip(graph(r, x, w), step(r, x, w)))          # not what it was traced with
    # a call for each row, and the calls that would drop a gradient
    for a, b in zip(torch.vmap(lambda t: lowbit.rms_norm_quantize(t, w))(x), lowbit.rms_norm_quantize(x, w)):
        assert torch.equal(a, b)
    with forward_ad.dual_level(), pytest.raises(RuntimeError, match="no gradient"):
        lowbit.rms_norm_quantize(forward_ad.make_dual(x, r), w)
    for transform in (lambda: torch.func.grad(lambda t: lowbit.rms_norm_quantize(t, w)[1].sum())(x),
                      lambda: torch.func.jvp(lambda t: lowbit.rms_norm_quantize(t, w)[1], (x,), (r,))):
        with pytest.raises(RuntimeError, match="no gradient"):
            transform()
    # a view whose memory holds the negated values
    z = torch.complex(x, r).contiguous()
    neg = torch._neg_view(x)
    assert torch.equal(lowbit.rms_norm_quantize(neg, w)[0], lowbit.rms_norm_quantize(-x, w)[0])
    assert torch.equal(lowbit.add_rms_norm_quantize(x, z.conj().imag, w)[2], x - r)


def test_the_pair_in_an_autograd_function_compiles(dev):
    class Norm(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, weight):
            codes, scales, inv = lowbit.rms_norm_quantize(x, weight)
            ctx.save_for_backward(x, weight, inv)
            return codes.float() * scales.unsqueeze(-1)

        @staticmethod
        def backward(ctx, grad):
            return lowbit.rms_norm_quantize_backward(grad, *ctx.saved_tensors)

    g = gen("compiled pair")
    base, w, dy = rows_like_activations(g, 9, 130, F32).to(dev), torch.ones(130, device=dev), torch.randn(9, 130, generator=g).to(dev)
    torch._dynamo.reset()
    results = []
    for fn in (Norm.apply, torch.compile(lambda x, w: Norm.apply(x, w), backend="aot_eager", fullgraph=True)):
        x, weight = base.clone().requires_grad_(), w.clone().requires_grad_()
        y = fn(x, weight)
        y.backward(dy)
        results.append((y.detach(), x.grad, weight.grad))
    assert all(torch.equal(a, b) for a, b in zip(*results))


@pytest.mark.parametrize("rows", [1, 3, 8, 24, 64])
@pytest.mark.parametrize("xt", FLOATS, ids=NAMES.get)
def test_matvec_4bit_of_floating_rows_closely(dev, rows, xt):
    # within the roundings of the terms' own sums: rows in stretches and in several visits, ragged ends, every size of group
    for n, k, group, st in ((48, 20000, 128, BF16), (15, 5604, 32, F32), (600, 6000, 64, BF16), (2090, 4300, 128, F32), (33, 1999, 32, BF16), (4099, 130, 64, F32)):
        g = gen("closely", rows, str(xt), n, k, group)
        announce(f"matvec {rows} x {k} x {n} group {group} {xt}, closely")
        codes, s = four_bit(g, n, k, group, st)
        check_matvec_closely(dev, rows_like_activations(g, rows, k, F32).to(xt), codes, s, k)


def test_calls_make_their_tensors_device_the_current_one(dev, monkeypatch):
    # one device stands in for two: it counts as another one until its guard is entered
    g = gen("another device")
    x, w = rows_like_activations(g, 3, 96, F32).to(dev), torch.ones(96, device=dev)
    inv = torch.ones(3, device=dev)
    packed, s = lowbit.quantize_4bit(x, 32)
    calls = [lambda: lowbit.rms_norm_quantize(x, w), lambda: lowbit.add_rms_norm_quantize(x, x, w), lambda: lowbit.rms_norm_quantize_backward(x, x, w, inv, x),
             lambda: lowbit.quantize_4bit(x, 64), lambda: lowbit.dequantize_4bit(packed, s), lambda: lowbit.matvec_4bit(x, packed, s)]
    want = [torch.utils._pytree.tree_leaves(call()) for call in calls]
    state = {"current": 1, "entered": []}

    class Guard:
        def __init__(self, device):
            self.device = device

        def __enter__(self):
            state["entered"].append(self.device)
            state["current"] = self.device.index

        def __exit__(self, *exc):
            state["current"] = 1
            return False

    with monkeypatch.context() as m:
        m.setattr(lowbit, "_current_device", lambda: state["current"])
        m.setattr(torch.cuda, "device", Guard)
        got = [torch.utils._pytree.tree_leaves(call()) for call in calls]
    assert state["entered"] == [x.device] * len(calls)
    for a, b in zip(got, want):
        assert all(torch.equal(p.view(torch.uint8), q.view(torch.uint8)) for p, q in zip(a, b))
