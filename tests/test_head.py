"""The detection head's operators without a GPU: what they refuse, through Python and through the C ABI."""

import ctypes

import pytest

torch = pytest.importorskip("torch")

import tf_faster_rcnn_amd as pkg  # noqa: E402

lib = pkg._lib.lib()
EINVAL, EUNSUPPORTED = pkg._lib.FRCNN_EINVAL, pkg._lib.FRCNN_EUNSUPPORTED
P = 1 << 20  # an address that no call below may reach


def refused(rc, code=EINVAL, word=b""):
    assert rc == code and word in lib.frcnn_last_error(), (rc, lib.frcnn_last_error())


def test_quantize_blocks_refusals():
    call = lambda **k: lib.frcnn_quantize_blocks(*{**dict(x=P, type=0, ldx=256, rows=4, K=256, block_rows=1, q=P, ldq=256, scales=P, scale_type=0,  # noqa: E731
                                                         row=1, block=4, stream=None), **k}.values())
    refused(call(type=9), word=b"element type")
    refused(call(scale_type=2), word=b"scale type")
    refused(call(block_rows=64), word=b"block_rows")
    refused(call(rows=-1), word=b"negative")
    refused(call(x=None), word=b"null")
    refused(call(scales=None), word=b"null")
    refused(call(ldx=255))
    refused(call(ldq=250, K=250))
    refused(call(q=P + 8), word=b"misaligned")
    refused(call(x=P + 2), word=b"misaligned")
    refused(call(scales=P + 2), word=b"misaligned")
    refused(call(row=-1), word=b"stride")
    refused(call(rows=2 ** 31 - 1, K=2 ** 20, ldx=2 ** 20, ldq=2 ** 20), EUNSUPPORTED)
    assert call(rows=0) == 0 and call(K=0) == 0


def test_scaled_matmul_refusals():
    call = lambda **k: lib.frcnn_scaled_matmul(*{**dict(a=P, lda=256, sa=P, sar=1, sab=4, b=P, ldb=256, sb=P, sbr=1, sbb=1, st=0, bias=None, act=0, M=4,  # noqa: E731
                                                       N=4, K=256, y=P, yt=2, ldy=4, ws=None, wsb=0, stream=None), **k}.values())
    refused(call(st=5), word=b"scale type")
    refused(call(yt=5), word=b"output type")
    refused(call(act=2), word=b"activation")
    refused(call(K=-1), word=b"negative")
    refused(call(y=None), word=b"output")
    refused(call(ldy=3), word=b"output")
    refused(call(bias=P + 1), word=b"bias")
    refused(call(a=None), word=b"null")
    refused(call(lda=250), word=b"16 bytes")
    refused(call(a=P + 8), word=b"16 bytes")
    refused(call(ldb=128), word=b"16 bytes")
    refused(call(sa=P + 2), word=b"scales")
    refused(call(sab=-4), word=b"stride")
    refused(call(K=2 ** 23, lda=2 ** 23, ldb=2 ** 23), EUNSUPPORTED)
    refused(call(lda=2 ** 24), EUNSUPPORTED)
    assert call(M=0) == 0 and call(N=0) == 0


def test_group_norm_refusals():
    f = ctypes.c_float
    call = lambda **k: lib.frcnn_group_norm(*{**dict(x=P, type=0, N=2, S=49, C=64, G=8, gamma=P, beta=P, eps=f(1e-3), act=0, y=P, stats=None, ws=None,  # noqa: E731
                                                    wsb=0, stream=None), **k}.values())
    grad = lambda **k: lib.frcnn_group_norm_grad(*{**dict(dy=P, x=P, type=0, N=2, S=49, C=64, G=8, gamma=P, beta=P, stats=P, act=0, dx=P, dgamma=P,  # noqa: E731
                                                         dbeta=P, ws=P, wsb=1 << 30, stream=None), **k}.values())
    for c in (call, grad):
        refused(c(type=3), word=b"element type")
        refused(c(S=0), word=b"position")
        refused(c(N=-1))
        refused(c(C=65), word=b"multiple")
        refused(c(G=0), word=b"multiple")
        refused(c(act=7), word=b"activation")
        refused(c(x=None), word=b"null")
        refused(c(x=P + 2), word=b"misaligned")
        refused(c(S=1 << 25), EUNSUPPORTED)
        refused(c(C=4096 * 8, G=1), EUNSUPPORTED, b"per group")
        refused(c(C=513, G=1), EUNSUPPORTED, b"per group")
    refused(call(eps=f(-1.0)), word=b"epsilon")
    refused(call(eps=f(float("nan"))), word=b"epsilon")
    refused(call(S=50000), word=b"workspace")
    refused(grad(wsb=0), word=b"workspace")
    refused(grad(ws=P + 16), word=b"workspace")
    refused(grad(dgamma=None), word=b"null")
    assert call(N=0) == 0
    assert lib.frcnn_group_norm_workspace_bytes(0, 2, 49, 64, 8) == 0
    assert lib.frcnn_group_norm_grad_workspace_bytes(0, 2, 49, 64, 8) > 0


def test_dropout_refusals():
    call = lambda **k: lib.frcnn_dropout(*{**dict(x=P, y=P, type=0, count=8, rate=0.5, seed=0, offset=0, state=None, stream=None), **k}.values())  # noqa: E731
    refused(call(type=-1), word=b"element type")
    refused(call(rate=1.0), word=b"rate")
    refused(call(rate=-0.1), word=b"rate")
    refused(call(rate=float("nan")), word=b"rate")
    refused(call(count=-1), word=b"count")
    refused(call(x=None), word=b"null")
    refused(call(y=P + 2), word=b"aligned")
    refused(call(state=P + 4), word=b"aligned")
    assert call(count=0) == 0


def test_python_entry_points_refuse_before_the_gpu():
    h = pkg.head_utils
    with pytest.raises(ValueError, match="x must be one of"):
        h.quantize_blocks(torch.zeros(2, 2, dtype=torch.float64))
    with pytest.raises(ValueError, match="a must be one of"):
        h.scaled_matmul(torch.zeros(2, 2), None, None, None)
    with pytest.raises(ValueError, match="x must be one of"):
        h.group_norm(torch.zeros(2, 2, dtype=torch.int32), None, None, 1)
    with pytest.raises(ValueError, match="x must be one of"):
        h.dropout(torch.zeros(2, dtype=torch.int64), 0.5, 1)
    if not torch.cuda.is_available():
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            h.dropout(torch.zeros(2), 0.5, 1)


def test_layer_configs_and_refusals():
    box = pkg.box_head
    with pytest.raises(ValueError, match="rate"):
        box.Dropout(1.0)
    assert box.Dropout(0.5, seed=3, name="drop").get_config() == {"name": "drop", "trainable": True, "dtype": "float32", "rate": 0.5, "seed": 3}
    cfg = box.GroupNormalization(16, activation="relu", name="gn").get_config()
    assert cfg["groups"] == 16 and cfg["activation"] == "relu" and box.GroupNormalization.from_config(cfg).get_config() == cfg
    dense = box.QuantizedDense(8, activation="relu", name="fc")
    assert box.QuantizedDense.from_config(dense.get_config()).get_config() == dense.get_config()
    with pytest.raises(ValueError, match="no weights"):
        dense(torch.zeros(2, 4))
    with pytest.raises(ValueError, match="kernel must be"):
        dense.set_weights([torch.zeros(4, 9)])
    x = torch.zeros(2)
    assert box.Dropout(0.5)(x) is x and box.Dropout(0.0)(x, training=True) is x


@pytest.mark.parametrize("size", [2 ** 31, 2 ** 32, 2 ** 32 + 5, 2 ** 33 + 128, 2 ** 40])
def test_sizes_beyond_32_bits_are_seen_whole(size):
    """Counts reach the library in 64 bits: none of them is taken for its lower 32."""
    big = -(-size // 128) * 128
    refused(lib.frcnn_quantize_blocks(P, 0, 256, size, 256, 1, P, 256, P, 0, 1, 4, None), EUNSUPPORTED, b"%d" % size)
    refused(lib.frcnn_quantize_blocks(P, 0, big, 4, big, 1, P, big, P, 0, 1, 4, None), EUNSUPPORTED, b"%d" % big)
    refused(lib.frcnn_quantize_blocks(P, 0, big, 128, big, 128, P, big, P, 1, 1, 4, None), EUNSUPPORTED, b"%d" % big)
    for m, n, k in ((size, 4, 256), (4, size, 256), (4, 4, big)):
        ld = max(k, 256)
        refused(lib.frcnn_scaled_matmul(P, ld, P, 1, 4, P, ld, P, 1, 1, 0, None, 0, m, n, k, P, 2, max(n, 4), None, 0, None), EUNSUPPORTED, b"index")
        assert lib.frcnn_scaled_matmul_workspace_bytes(m, n, k) == 0
    f = ctypes.c_float
    for n, s, c, g in ((size, 49, 64, 8), (2, size, 64, 8), (2, 49, big, 8), (2, 50000, big + 64, big + 64)):
        refused(lib.frcnn_group_norm(P, 0, n, s, c, g, P, P, f(1e-3), 0, P, None, P, 1 << 40, None), EUNSUPPORTED, b"index")
        refused(lib.frcnn_group_norm_grad(P, P, 0, n, s, c, g, P, P, P, 0, P, P, P, P, 1 << 40, None), EUNSUPPORTED, b"index")
        assert lib.frcnn_group_norm_workspace_bytes(0, n, s, c, g) == 0 and lib.frcnn_group_norm_grad_workspace_bytes(0, n, s, c, g) == 0
    refused(lib.frcnn_group_norm(P, 0, 2, 49, 64, size, P, P, f(1e-3), 0, P, None, P, 1 << 40, None), EINVAL, b"multiple")


def calls_on(x, gamma):
    """Each operator with `x` in the place of every tensor that has derivatives, and of `gamma` alone."""
    h = pkg.head_utils
    plain, ones = torch.ones(2, 3, 8), torch.ones(8)
    stats = torch.ones(2, 2, 2)
    a = torch.zeros(2, 8, dtype=torch.float8_e4m3fn)
    one = torch.ones(2, 1)
    return {"group_norm": [lambda: h.group_norm(x, ones, ones, 2), lambda: h.group_norm(plain, gamma, ones, 2), lambda: h.group_norm(plain, ones, gamma, 2)],
            "group_norm_gradients": [lambda: h.group_norm_gradients(x, plain, ones, ones, stats), lambda: h.group_norm_gradients(plain, x, ones, ones, stats),
                                     lambda: h.group_norm_gradients(plain, plain, gamma, ones, stats)],
            "dropout": [lambda: h.dropout(x, 0.5, 1)],
            "quantize_blocks": [lambda: h.quantize_blocks(x)],
            "scaled_matmul": [lambda: h.scaled_matmul(a, one, a, one[:1], bias=gamma)]}


@pytest.mark.parametrize("operator", ["group_norm", "group_norm_gradients", "dropout", "quantize_blocks", "scaled_matmul"])
def test_forward_mode_derivatives_and_traces_are_refused(operator):
    """They would come back without a tangent, that is with derivative zero, or as a record of uninitialised memory."""
    from torch.autograd import forward_ad

    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))  # noqa: E731
        for call in calls_on(dual(torch.ones(2, 3, 8)), dual(torch.ones(8)))[operator]:
            with pytest.raises(RuntimeError, match=f"{operator} has no forward-mode"):
                call()
    for at in range(len(calls_on(None, None)[operator])):
        def traced(x, gamma):
            calls_on(x, gamma)[operator][at]()
            return x
        with pytest.raises(RuntimeError, match=f"{operator} cannot be traced"):
            torch.jit.trace(traced, (torch.ones(2, 3, 8), torch.ones(8)))
