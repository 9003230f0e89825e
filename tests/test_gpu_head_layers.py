"""The detection head's layers: what they keep of their weights, and who else sees it."""

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def box():
    import tf_faster_rcnn_amd as pkg
    return pkg.box_head


def test_quantized_dense_keeps_no_hold_of_its_sources(box):
    """Weights are taken when they are set: a staging buffer that is filled again, or an optimiser's step, changes nothing."""
    x = torch.randn((5, 300), device="cuda")
    for device in ("cuda", "cpu"):
        kernel, bias = torch.randn((300, 40), device=device), torch.randn(40, device=device)
        dense = box.QuantizedDense(40, activation="relu", out_dtype=torch.float32)
        dense.set_weights([kernel, bias])
        want = dense(x)
        kernel.add_(1.0)
        bias.add_(100.0)
        assert torch.equal(dense(x), want)
