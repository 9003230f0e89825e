"""The detection head's operators at counts where one launch would have 2^32 threads: the work is done in several."""

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
E8M0 = torch.float8_e8m0fnu


@pytest.fixture(scope="module")
def head():
    import tf_faster_rcnn_amd as pkg
    return pkg.head_utils


def same_in_pieces(call, count, *tensors):
    """The call on all rows gives what calls on a third of them at a time give, which fit one launch each."""
    whole = call(*tensors)
    for i in range(3):
        part = slice(count * i // 3, count * (i + 1) // 3)
        for got, want in zip(whole, call(*[t[part] for t in tensors])):
            got, want = (t.view(torch.uint8) if t.element_size() == 1 else t for t in (got[part], want))
            assert torch.equal(got, want)


@pytest.mark.parametrize("scale_dtype", [F32, E8M0])
def test_quantize_blocks_of_many_rows(head, scale_dtype):
    rows = 2 ** 30 + 70  # 64 rows and 256 threads a workgroup
    x = torch.empty((rows, 1), dtype=BF16, device="cuda").normal_()
    same_in_pieces(lambda v: head.quantize_blocks(v, scale_dtype=scale_dtype), rows, x)


@pytest.mark.parametrize("scale_dtype,out_dtype", [(F32, F32), (E8M0, BF16)])
def test_scaled_matmul_of_many_rows(head, scale_dtype, out_dtype):
    rows = 2 ** 26 + 21  # 16 rows and 1024 threads a workgroup
    a = torch.randint(0, 120, (rows, 16), dtype=torch.uint8, device="cuda")
    a = a.view(torch.float8_e4m3fn)
    scales = torch.randint(100, 140, (rows, 1), dtype=torch.uint8, device="cuda").view(E8M0)
    b, sb = head.quantize_blocks(torch.randn((5, 16), device="cuda"), 128, scale_dtype=scale_dtype)
    scales = scales if scale_dtype == E8M0 else scales.float()
    same_in_pieces(lambda v, s: [head.scaled_matmul(v, s, b, sb, out_dtype=out_dtype)], rows, a, scales)


def test_group_norm_of_many_images(head):
    images = 2 ** 26 + 5  # an image and 64 threads a workgroup
    x = torch.empty((images, 1, 8), dtype=BF16, device="cuda").normal_()
    gamma, beta = torch.randn(8, device="cuda"), torch.randn(8, device="cuda")
    same_in_pieces(lambda v: head.group_norm(v, gamma, beta, 2, return_stats=True), images, x)
    y, stats = head.group_norm(x, gamma, beta, 2, return_stats=True)
    dx, _, dbeta = head.group_norm_gradients(y, x, gamma, beta, stats)
    part = slice(images - 1000, images)
    assert torch.equal(dx[part], head.group_norm_gradients(y[part], x[part], gamma, beta, stats[part])[0])
    # an image adds a term of size 1 to each sum; chains of 2^26 / 2^10 terms at most
    want = sum(p.double().sum((0, 1)) for p in y.split(1 << 22))
    assert ((dbeta.double() - want).abs() <= 2.0 ** 17 * 2.0 ** -24 * sum(p.double().abs().sum((0, 1)) for p in y.split(1 << 22))).all()


def test_group_norm_by_chunks_of_many_images(head, knobs):
    knobs.setenv("FRCNN_NORM_CHUNKED", 1)
    images = 2 ** 23 + 5  # an image and 512 threads a workgroup
    x = torch.empty((images, 1, 8), dtype=BF16, device="cuda").normal_()
    gamma, beta = torch.randn(8, device="cuda"), torch.randn(8, device="cuda")
    same_in_pieces(lambda v: head.group_norm(v, gamma, beta, 2, return_stats=True), images, x)
    import tf_faster_rcnn_amd as pkg
    y, stats = head.group_norm(x[:10], gamma, beta, 2, return_stats=True)
    with pytest.raises(pkg._lib.UnsupportedSizeError, match="threads"):
        head.group_norm_gradients(x, x, gamma, beta, stats[:1].expand(images, 2, 2))


def test_dropout_that_keeps_nothing(head):
    """Where round(rate * 2^32) is 2^32 no word is large enough, not even 2^32 - 1, of which 2^33 elements have a few."""
    x = torch.ones((1 << 33,), dtype=F16, device="cuda")
    for seed in (1, 2, 3):
        y = head.dropout(x, 1 - 2.0 ** -34, seed)
        assert not y.view(torch.int16).any()
    del y
    state = torch.tensor([5, 6], device="cuda")
    for dtype in (F32, F16, BF16):
        bad = torch.full((1027,), float("nan"), dtype=dtype, device="cuda")
        for v in (bad, bad[1:]):
            for args in ((3,), (state,)):
                assert (head.dropout(v, 1 - 2.0 ** -53, *args) == 0).all()
    # words of 2^32 - 1: two in the mean, and a chance of 1e-13 of 20
    kept = sum(int((part != 0).sum()) for part in head.dropout(x, 1 - 2.0 ** -32, 1).split(1 << 30))
    assert kept < 20


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("shape,groups", [((2, 4, 1024), 1), ((3, 50, 64), 8)])
def test_gradients_of_a_dy_between_16_bytes(head, shape, groups, dtype):
    """A contiguous dy at any element's address gives the bits of an aligned one, with groups of more than 512 channels too."""
    x = torch.randn(shape, device="cuda").to(dtype)
    dy = torch.empty(x.numel() + 1, dtype=dtype, device="cuda")[1:].view(shape).normal_()
    gamma, beta = torch.randn(shape[-1], device="cuda"), torch.randn(shape[-1], device="cuda")
    _, stats = head.group_norm(x, gamma, beta, groups, activation="swish", return_stats=True)
    want = head.group_norm_gradients(dy.clone(), x, gamma, beta, stats, activation="swish")
    for got, exp in zip(head.group_norm_gradients(dy, x, gamma, beta, stats, activation="swish"), want):
        assert torch.equal(got, exp)
    leaf = x.clone().requires_grad_()
    head.group_norm(leaf, gamma, beta, groups, activation="swish").backward(dy)
    assert torch.equal(leaf.grad, want[0])


@pytest.mark.parametrize("groups", [2.5, 0.5, 0, -2, 3, 20])
def test_groups_that_do_not_divide(head, groups):
    """Also fractions that divide: 10 channels are no 2.5 groups."""
    with pytest.raises(ValueError, match="multiple"):
        head.group_norm(torch.ones((2, 3, 10), device="cuda"), torch.ones(10, device="cuda"), torch.ones(10, device="cuda"), groups)
