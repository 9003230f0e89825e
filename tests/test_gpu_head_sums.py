"""How exactly ``scaled_matmul`` forms its sums, beneath the rounding of the result.

A bias of minus the exact sum leaves the result's own error behind, and large products that cancel show which small ones a sum
has dropped.
"""

import pytest

torch = pytest.importorskip("torch")

from tests import head_sums  # noqa: E402

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu


@pytest.fixture(scope="module")
def head():
    import tf_faster_rcnn_amd as pkg
    return pkg.head_utils


def cancelling(rows, columns):
    """One block: 448 * 448 and its negative in columns 0 and 1, and 1 in column 2 + row % 126.  Every sum is 1."""
    a = torch.zeros((rows, 128), device="cuda")
    a[:, :2] = 448.0
    a[torch.arange(rows), 2 + torch.arange(rows) % 126] = 1.0
    b = torch.ones((columns, 128), device="cuda")
    b[:, 0], b[:, 1] = 448.0, -448.0
    return a.to(E4M3), b.to(E4M3)


@pytest.mark.parametrize("scale_dtype", [F32, E8M0])
@pytest.mark.parametrize("out_dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows", [1, 7, 16])
def test_few_rows_drop_no_product(head, rows, out_dtype, scale_dtype):
    """Up to 16 rows are bound by the weights' way from memory: their products keep all their bits whatever the result's type."""
    a, b = cancelling(rows, 40)
    y = head.scaled_matmul(a, torch.ones((rows, 1), device="cuda").to(scale_dtype), b, torch.ones((1, 1), device="cuda").to(scale_dtype),
                           out_dtype=out_dtype)
    assert (y == 1).all()


@pytest.mark.parametrize("scale_dtype", [F32, E8M0])
@pytest.mark.parametrize("out_dtype", [F32, F16, BF16])
@pytest.mark.parametrize("form", [0, 1, 2, 3, 4])
def test_products_are_cut_in_their_eight_only(head, knobs, form, out_dtype, scale_dtype):
    """The documented loss of the tile forms' 16-bit results: the 1 beside 448 * 448 in columns 0 to 7, and nothing else.  An fp32
    result and the split-K form (4) lose nothing."""
    knobs.setenv("FRCNN_PRODUCT_FORM", form)
    rows = 300
    a, b = cancelling(rows, 150)
    y = head.scaled_matmul(a, torch.ones((rows, 1), device="cuda").to(scale_dtype), b, torch.ones((2, 1), device="cuda").to(scale_dtype),
                           out_dtype=out_dtype).float()
    column = 2 + torch.arange(rows, device="cuda") % 126
    exact = column >= 8
    if out_dtype == F32 or form == 4:
        exact[:] = True
    assert (y[exact] == 1).all()
    assert ((y == 0) | (y == 1)).all()


@pytest.mark.parametrize("scale_dtype", [F32, E8M0])
@pytest.mark.parametrize("out_dtype", [F32, BF16])
@pytest.mark.parametrize("form", [0, 1, 2, 3, 4])
def test_sums_of_blocks_are_fp32(head, knobs, form, out_dtype, scale_dtype):
    """P, s and -P in three blocks: s survives while it is more than 2^-24 of P, also where the instruction accumulates."""
    knobs.setenv("FRCNN_PRODUCT_FORM", form)
    rows = 30
    a = torch.zeros((rows, 384), device="cuda")
    b = torch.zeros((20, 384), device="cuda")
    a[:, 0], a[:, 128], a[:, 256] = 448.0, 1.0, 448.0
    b[:, 0], b[:, 128], b[:, 256] = 448.0, 1.0, -448.0
    for t in range(-8, 7):  # P is 1.53 * 2^17
        sa = torch.ones((rows, 3), device="cuda")
        sa[:, 1] = 2.0 ** -t
        y = head.scaled_matmul(a.to(E4M3), sa.to(scale_dtype), b.to(E4M3), torch.ones((1, 3), device="cuda").to(scale_dtype), out_dtype=out_dtype)
        assert (y.float() == 2.0 ** -t).all(), t


def operands(head, rows, units, inner, scale_dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn((rows, inner), generator=g, device="cuda").clamp_min_(-0.3) * torch.exp2(torch.randn((rows, 1), generator=g, device="cuda"))
    w = torch.randn((units, inner), generator=g, device="cuda") * inner ** -0.5
    return (*head.quantize_blocks(x, scale_dtype=scale_dtype), *head.quantize_blocks(w, 128, scale_dtype=scale_dtype))


def rows_of(a, sa, pick):
    return a.view(torch.uint8)[pick].view(E4M3), sa.view(torch.uint8 if sa.dtype == E8M0 else sa.dtype)[pick].view(sa.dtype)


@pytest.mark.parametrize("scale_dtype", [F32, E8M0])
@pytest.mark.parametrize("out_dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows,units,inner", [(1, 4096, 28224), (16, 1000, 25088), (300, 4096, 28224), (300, 105, 4096), (700, 520, 28230), (4800, 4096, 4100),
                                              (2400, 1111, 2050), (64, 300, 130), (33, 129, 300000)])
def test_sums_at_the_heads_sizes(head, rows, units, inner, out_dtype, scale_dtype):
    """Within what the additions that there are may be off by: a lost chunk or a wrong scale in one of 221 blocks is seen."""
    a, sa, b, sb = operands(head, rows, units, inner, scale_dtype, rows + inner)
    bias = 0.1 * torch.randn((units,), generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
    y = head.scaled_matmul(a, sa, b, sb, bias=bias, out_dtype=out_dtype)
    pick = torch.unique(torch.cat([torch.arange(0, rows, max(1, rows // 53), device="cuda"), torch.tensor([rows - 1], device="cuda")]))
    want, l2 = head_sums.product(*rows_of(a, sa, pick), b, sb, bias)
    allowed = head_sums.tolerance(want, l2, inner, out_dtype, out_dtype != F32 and rows > 16)
    worst = ((y[pick].double() - want).abs() / allowed).max().item()
    assert worst <= 1, worst


@pytest.mark.parametrize("form", [0, 1, 2, 3, 4])
@pytest.mark.parametrize("scale_dtype", [F32, E8M0])
@pytest.mark.parametrize("rows,units,inner", [(40, 300, 128), (161, 257, 1000), (700, 1111, 2500), (300, 260, 28224)])
def test_sums_of_every_form(head, knobs, rows, units, inner, scale_dtype, form):
    knobs.setenv("FRCNN_PRODUCT_FORM", form)
    a, sa, b, sb = operands(head, rows, units, inner, scale_dtype, form)
    want, l2 = head_sums.product(a, sa, b, sb)
    for out_dtype in (F32, F16, BF16):
        y = head.scaled_matmul(a, sa, b, sb, out_dtype=out_dtype)
        worst = ((y.double() - want).abs() / head_sums.tolerance(want, l2, inner, out_dtype, out_dtype != F32 and form != 4)).max().item()
        assert worst <= 1, (out_dtype, worst)


@pytest.mark.parametrize("form", [0, 1, 2, 3, 4])
@pytest.mark.parametrize("scale_dtype", [F32, E8M0])
@pytest.mark.parametrize("inner", [4096, 28224, 262144])
def test_error_beneath_the_rounding(head, knobs, inner, scale_dtype, form):
    """A bias of minus the sum leaves its error behind: neither the length of K nor the type of the scales makes it grow.  Also for
    operands of one sign, where every cut has the same one: eight products lose less than 2^-13 of their largest each."""
    knobs.setenv("FRCNN_PRODUCT_FORM", form)
    for positive in (False, True):
        g = torch.Generator(device="cuda").manual_seed(inner)
        x, w = torch.randn((1, inner), generator=g, device="cuda"), torch.randn((200, inner), generator=g, device="cuda") * inner ** -0.5
        if positive:
            x, w = x.abs(), w.abs()
        b, sb = head.quantize_blocks(w, 128, scale_dtype=scale_dtype)
        a, sa = head.quantize_blocks(x.expand(40, inner), scale_dtype=scale_dtype)
        sums, l2 = head_sums.product(*rows_of(a, sa, torch.zeros(1, dtype=torch.long, device="cuda")), b, sb)
        bias = -sums[0].float()
        for out_dtype in (F32, BF16):
            y = head.scaled_matmul(a, sa, b, sb, bias=bias, out_dtype=out_dtype)
            assert torch.equal(y, y[:1].expand_as(y))
            left = (sums + bias.double())[0]
            error = (y[0].double() - left).abs() - torch.finfo(out_dtype).eps / 2 * y[0].double().abs()
            narrow = out_dtype != F32 and form != 4
            if positive:
                # the partial sums are the sum at most, each addition off by 2 U of it; an eight's largest product is its sum at most
                allowed = sums[0] * (2 * head_sums.U * (inner // 128 + 64) + (7 * 2.0 ** -13 if narrow else 0))
            else:
                allowed = head_sums.tolerance(sums, l2, inner, F32, narrow)[0]
            assert (error <= allowed).all(), (out_dtype, positive, (error / allowed).max().item())


def test_parameter_gradients_of_many_images(head):
    """dgamma and dbeta over 155000 pooled images, more than 2^32 elements, against sums in 64 bits.

    dy = 2 relu(x) makes both sums ones of positive terms, of which a lost share is seen.  The kernel's threads (256 at least, 8
    channels each) are about a thousand workgroups' worth, so a chain adds at most 1.25 * N S C / (1024 * 256 * 8) terms, and 200
    join the chains; xhat is off by 160 U of (1 + mean / deviation) and itself."""
    images, positions, channels, groups = 155000, 49, 576, 32
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.empty((images, positions, channels), dtype=BF16, device="cuda")
    for i in range(0, images, 5000):
        x[i:i + 5000].normal_(generator=g)
    dy = x.clamp_min(0).mul_(2)
    gamma, beta = torch.ones(channels, device="cuda"), torch.zeros(channels, device="cuda")
    y, stats = head.group_norm(x, gamma, beta, groups, return_stats=True)
    del y
    _, dgamma, dbeta = head.group_norm_gradients(dy, x, gamma, beta, stats)
    want_gamma, want_beta, size = (torch.zeros(channels, dtype=torch.float64, device="cuda") for _ in range(3))
    for i in range(0, images, 1000):
        v = x[i:i + 1000].double().view(1000, positions, groups, -1)
        mean = v.mean((1, 3), keepdim=True)
        centred = v - mean
        xhat = (centred / torch.sqrt((centred * centred).mean((1, 3), keepdim=True) + 1e-3)).view(1000, positions, channels)
        d = dy[i:i + 1000].double()
        want_gamma += (d * xhat).sum((0, 1))
        want_beta += d.sum((0, 1))
        size += (d * xhat).abs().sum((0, 1))
    depth = 1.25 * images * positions * channels / (1024 * 256 * 8) + 200
    assert depth * head_sums.U < 2e-4  # a thousandth lost is seen
    assert ((dbeta.double() - want_beta).abs() <= depth * head_sums.U * want_beta).all()
    assert ((dgamma.double() - want_gamma).abs() <= (depth + 160) * head_sums.U * size + 160 * head_sums.U * 1.1 * want_beta).all()


@pytest.mark.parametrize("form", [0, 1, 2, 3, 4])
@pytest.mark.parametrize("scale_dtype", [F32, E8M0])
@pytest.mark.parametrize("inner", [384, 640, 1250])
@pytest.mark.parametrize("far", [(100, 30), (-100, -30), (-120, -32), (120, 7), (20, 107), (-126, -1)])
def test_products_of_scales_beyond_fp32(head, knobs, far, inner, scale_dtype, form):
    """Scales whose product is no fp32 number while the result is one, in some rows' second block: a block of zeros gives zero, the
    smallest sum 2^-18 and the largest 2^24.6 what they are worth; other rows and blocks are as ever."""
    knobs.setenv("FRCNN_PRODUCT_FORM", form)
    ea, eb = far
    rows, units = 70, 200
    blocks = -(-inner // 128)
    a, b = torch.ones((rows, inner), device="cuda"), torch.ones((units, inner), device="cuda")
    a[3::5, 128:256], b[:, 128:256] = 0.0, 0.0
    b[:, 128] = 2.0 ** -9
    a[0::5, 128:256] = 2.0 ** -9  # sums of 2^-18
    if ea + eb < 0:
        a[0::5, 128:256], b[:, 128:256] = 448.0, 448.0
    # others: 0 in the far block
    a[1::5, 128:256], a[2::5, 128:256], a[4::5, 128:256] = 0.0, 0.0, 0.0
    a, b = a.to(E4M3), b.to(E4M3)
    step = 1.0 if scale_dtype == E8M0 else 1.375
    sa, sb = torch.ones((rows, blocks), device="cuda"), torch.ones((2, blocks), device="cuda")
    sa[0::5, 1], sa[3::5, 1], sb[:, 1] = step * 2.0 ** ea, step * 2.0 ** ea, step * 2.0 ** eb
    if ea + eb < 0:
        sa[0::5, ::2] = 0.0 if scale_dtype == F32 else 2.0 ** -127
        sa[0::5, 3::2] = sa[0::5, :1]
    sa, sb = sa.to(scale_dtype), sb.to(scale_dtype)
    want, _ = head_sums.product(a, sa, b, sb)
    if ea + eb < 0 and scale_dtype == E8M0:  # the other blocks' 2^-127 are beside the far block's 2^-106 and more
        assert want[0, 0] > 2.0 ** -127
    for out_dtype in (F32, BF16):
        y = head.scaled_matmul(a, sa, b, sb, out_dtype=out_dtype)
        # all terms are positive: the roundings of the sums and of the scales, and the type's own; where the result is subnormal,
        # half of the type's smallest step, and a step of fp32's for each block
        half = torch.finfo(out_dtype).eps / 2
        off = (half + (blocks + 8) * 2 * head_sums.U) * want.abs() + half * 2.0 ** -126 + 2.0 ** -149 * blocks
        assert torch.isfinite(y).all()
        assert ((y.double() - want).abs() <= off).all(), (out_dtype, ((y.double() - want).abs() / off).max().item())


@pytest.mark.parametrize("form", [0, 2, 4])
@pytest.mark.parametrize("out_dtype", [F32, BF16])
def test_scales_that_are_no_numbers(head, knobs, out_dtype, form):
    """Infinite and NaN scales reach what they scale and nothing else; a zero scale makes zeros."""
    knobs.setenv("FRCNN_PRODUCT_FORM", form)
    a, b = torch.ones((40, 300), device="cuda"), torch.ones((260, 300), device="cuda")
    a[7, 128:256] = 0.0
    sa, sb = torch.ones((40, 3), device="cuda"), torch.ones((3, 3), device="cuda")
    sa[5, 1], sa[6, 2], sa[7, 1], sa[8] = float("inf"), float("nan"), float("inf"), 0.0
    sb[1, 0] = float("inf")
    y = head.scaled_matmul(a.to(E4M3), sa, b.to(E4M3), sb, out_dtype=out_dtype).float()
    want = torch.full((40, 260), 300.0, device="cuda")
    want[:, 128:256] = float("inf")
    want[5], want[6], want[7] = float("inf"), float("nan"), float("nan")  # 0 times infinity
    want[8] = 0.0
    want[8, 128:256] = float("nan")
    want = want.to(out_dtype).float()
    assert torch.equal(torch.isnan(y), torch.isnan(want)) and torch.equal(torch.nan_to_num(y, nan=1.0), torch.nan_to_num(want, nan=1.0))


@pytest.mark.parametrize("form", [0, 1, 2, 3, 4])
@pytest.mark.parametrize("out_dtype", [F32, BF16])
def test_e8m0_scales_at_their_ends(head, knobs, out_dtype, form):
    """2^127 twice and 2^-127 twice: zeros stay zeros, the smallest sum leaves the range, the largest vanishes, 1 is beside them."""
    knobs.setenv("FRCNN_PRODUCT_FORM", form)
    a, b = torch.ones((40, 384), device="cuda"), torch.ones((130, 384), device="cuda")
    a[:, 128:256], b[:, 128:256] = 448.0, 448.0
    a[1::2, 256:] = 0.0
    b[:, 256:], b[:, 256] = 0.0, 2.0 ** -9
    sa = torch.tensor([127, 0, 254], dtype=torch.uint8, device="cuda").expand(40, 3).contiguous().view(E8M0)
    sb = torch.tensor([127, 0, 254], dtype=torch.uint8, device="cuda").expand(2, 3).contiguous().view(E8M0)
    y = head.scaled_matmul(a.to(E4M3), sa, b.to(E4M3), sb, out_dtype=out_dtype)
    assert (y[1::2] == 128).all() and (y[::2] == float("inf")).all()
