"""How exactly ``scaled_matmul`` forms its sums, beneath the rounding of the result.

A bias of minus the exact sum leaves the result's own error behind, and large products that cancel show which small ones a sum
has dropped.
"""

import pytest

torch = pytest.importorskip("torch")

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
