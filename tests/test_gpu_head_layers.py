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


@pytest.mark.parametrize("source", ["cuda", "cpu"])
def test_weights_set_again_reach_who_holds_the_parameters(box, source):
    """An optimiser built on a norm's parameters goes on with them after set_weights."""
    norm = box.GroupNormalization(4)
    x = torch.randn((3, 5, 16), device="cuda")
    norm(x)
    held = norm.get_weights()
    optimiser = torch.optim.SGD(held, lr=1.0)
    norm.set_weights([torch.full((16,), 2.0, device=source), torch.full((16,), 3.0, device=source)])
    assert norm.gamma is held[0] and norm.beta is held[1] and norm.gamma.is_leaf and norm.gamma.requires_grad
    assert (norm.gamma == 2).all() and (norm.beta == 3).all()
    norm(x).sum().backward()
    optimiser.step()
    assert torch.allclose(norm.beta, torch.full_like(norm.beta, 3.0 - 15.0))
    with pytest.raises(ValueError):
        norm.set_weights([torch.ones(8), torch.ones(9)])
    assert norm.gamma is held[0] and norm.beta is held[1]
    norm.set_weights([torch.ones(8), torch.ones(8)])  # of another size: parameters of their own
    assert norm.gamma is not held[0] and norm.gamma.shape == (8,) and held[0].shape == (16,)
    norm.trainable = False
    norm.set_weights([torch.ones(8), torch.zeros(8)])
    assert not norm.gamma.requires_grad


def test_weights_set_again_are_seen_by_a_backward_pass_in_between(box):
    """A graph that saved the old values refuses instead of using the new ones."""
    norm = box.GroupNormalization(4)
    x = torch.randn((3, 5, 16), device="cuda")
    y = norm(x)
    norm.set_weights([torch.full((16,), 2.0), torch.zeros(16)])
    with pytest.raises(RuntimeError, match="inplace"):
        y.sum().backward()


@pytest.mark.parametrize("scale_dtype", [torch.float32, torch.float8_e8m0fnu])
def test_weights_set_again_reach_a_captured_graph(box, scale_dtype):
    x = torch.randn((20, 200), device="cuda")
    dense = box.QuantizedDense(40, scale_dtype=scale_dtype)
    first, second = ([torch.randn((200, 40), device="cuda"), torch.randn(40, device="cuda")] for _ in range(2))
    dense.set_weights(first)
    old = [dense.kernel, dense.kernel_scales, dense.bias]  # alive whatever the layer does
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = dense(x)
    dense.set_weights(second)
    fresh = box.QuantizedDense(40, scale_dtype=scale_dtype)
    fresh.set_weights(second)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, fresh(x)) and torch.equal(y, dense(x))
    dense.set_weights(second[:1])
    assert dense.bias is None and len(old) == 3


def test_weights_set_in_and_out_of_inference_mode(box):
    dense, norm = box.QuantizedDense(40), box.GroupNormalization(4)
    x = torch.randn((20, 200), device="cuda")
    for inside in (True, False, True, True, False):
        with torch.inference_mode(inside):
            weights = [torch.randn((200, 40), device="cuda"), torch.randn(40, device="cuda")]
            dense.set_weights(weights)
            norm.set_weights([weights[1][:16], weights[1][16:32]])
            fresh = box.QuantizedDense(40)
            fresh.set_weights(weights)
            assert torch.equal(dense(x), fresh(x)) and torch.equal(norm.gamma, weights[1][:16])
        norm(torch.randn((2, 3, 16), device="cuda")).sum().backward()
