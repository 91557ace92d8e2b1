"""The int8, norm and beam entry points reject bad arguments before touching a device, and do nothing,
successfully, for zero rows."""
import ctypes

import pytest

P = ctypes.c_void_p
OK = P(1 << 20)  # never dereferenced: validation fails first
ODD = P((1 << 20) + 4)


def _status(name, *args):
    from mq._lib import lib

    rc = getattr(lib, name)(*args)
    return rc, lib.mq_last_error().decode()


def test_quantize():
    assert _status("mq_quantize_s8", None, 0, 64, None, 64, None, 0, 64, None)[0] == 0
    for args, code, word in (((OK, 5, 64, OK, 64, OK, 4, 64, None), -1, "MQ_F32"), ((OK, 0, 63, OK, 64, OK, 4, 64, None), -1, "stride"),
                             ((OK, 0, 64, OK, 63, OK, 4, 64, None), -1, "stride"), ((OK, 0, 64, OK, 64, None, 4, 64, None), -1, "null"),
                             ((OK, 0, 64, OK, 64, OK, 4, 0, None), -1, "shape"), ((P((1 << 20) + 2), 0, 64, OK, 64, OK, 4, 64, None), -2, "aligned")):
        rc, msg = _status("mq_quantize_s8", *args)
        assert rc == code and word in msg, (args, rc, msg)


def test_products():
    good = [OK, 64, OK, OK, 64, OK, None, OK, 0, 32, 4, 32, 64, 0, None]
    for at, value, code, word in ((0, None, -1, "null"), (1, 63, -1, "stride"), (1, 72, -2, "16"), (3, ODD, -2, "16"), (8, 3, -1, "type"),
                                  (9, 31, -1, "stride"), (10, -1, -1, "shape"), (12, 0, -1, "shape"), (6, P((1 << 20) + 2), -2, "bias"),
                                  (7, P((1 << 20) + 1), -2, "aligned")):
        args = list(good)
        args[at] = value
        rc, msg = _status("mq_gemm_w8a8", *args)
        assert rc == code and word in msg, (at, rc, msg)
    args = list(good)
    args[1] = args[4] = args[12] = 131072
    rc, msg = _status("mq_gemm_w8a8", *args)
    assert rc == -4 and "131071" in msg
    args = list(good)
    args[0] = args[7] = None
    args[10] = 0
    assert _status("mq_gemm_w8a8", *args)[0] == 0
    rc, msg = _status("mq_gate_up_w8a8", OK, 64, OK, OK, 64, OK, OK, 0, 31, 4, 32, 64, None)
    assert rc == -1 and "stride" in msg


def test_norms():
    rc, msg = _status("mq_pre_norm", OK, 0, 64, None, 0, 1e-6, OK, 0, 64, None, 4, 64, None)
    assert rc == -1 and "null" in msg
    rc, msg = _status("mq_pre_norm", OK, 0, 64, OK, 0, 1e-6, OK, 3, 64, None, 4, 64, None)
    assert rc == -1 and "scales" in msg
    rc, msg = _status("mq_pre_norm", OK, 0, 64, OK, 0, 1e-6, OK, 4, 64, None, 4, 64, None)
    assert rc == -1 and "MQ_S8" in msg
    post = [OK, 0, 64, OK, 0, 1e-6, OK, 0, 64, None, 0, 64, 1, 1.0, OK, 64, OK, 0, 1e-6, OK, 0, 64, None, 4, 64, None]
    for at, value, word in ((0, None, "null"), (7, 3, "residual"), (8, 63, "residual"), (15, 63, "out"), (16, None, "next_w")):
        args = list(post)
        args[at] = value
        rc, msg = _status("mq_post_norm", *args)
        assert rc == -1 and word in msg, (at, rc, msg)
    args = list(post)
    args[9], args[12] = OK, 0
    rc, msg = _status("mq_post_norm", *args)
    assert rc == -1 and "rows_per_gate" in msg
    args = list(post)
    args[23] = 0
    assert _status("mq_post_norm", *args)[0] == 0


def test_beams():
    from mq._lib import lib

    assert lib.mq_beam_workspace_size(1, 4, 1000) > 0 and lib.mq_beam_workspace_size(1, 33, 1000) == 0
    good = [OK, 0, 1000, OK, None, -1, OK, OK, OK, None, 2, 4, 1000, OK, 1 << 24, None]
    for at, value, code, word in ((0, None, -1, "null"), (1, 3, -1, "type"), (2, 999, -1, "stride"), (4, OK, -1, "eos"), (5, 1000, -1, "eos"),
                                  (11, 33, -4, "32"), (12, 1 << 30, -4, "large"), (13, ODD, -2, "16"), (14, 100, -1, "small")):
        args = list(good)
        args[at] = value
        if at == 12:
            args[2] = value
        rc, msg = _status("mq_beam_select", *args)
        assert rc == code and word in msg, (at, rc, msg)
    args = list(good)
    args[10] = 0
    assert _status("mq_beam_select", *args)[0] == 0

    states, outer, strides = (P * 2)(OK, OK), (ctypes.c_int64 * 3)(1, 1, 4), (ctypes.c_int64 * 3)(0, 0, 64)
    good = [states, 2, OK, 2, 4, 256, outer, strides, 64, None]
    for at, value, code, word in ((0, None, -1, "null"), (5, 255, -1, "overlap"), (7, (ctypes.c_int64 * 3)(0, 0, 32), -1, "overlap"),
                                  (0, (P * 2)(OK, None), -1, "null state"), (4, 33, -4, "32"), (3, 70000, -4, "65535")):
        args = list(good)
        args[at] = value
        rc, msg = _status("mq_beam_reorder", *args)
        assert rc == code and word in msg, (at, rc, msg)
    args = list(good)
    args[1] = 0
    assert _status("mq_beam_reorder", *args)[0] == 0


def test_reorder_refuses_states_that_share_memory():
    """Two states of one layout, any distance apart: refused exactly where their bytes meet."""
    import itertools

    import torch

    if torch.cuda.is_available():
        pytest.skip("what is not refused would be launched with made-up addresses")
    layouts = (((1, 1, 1), (0, 0, 0), 2, 12), ((1, 1, 3), (0, 0, 8), 4, 32), ((1, 2, 3), (0, 64, 12), 8, 192),
               ((2, 3, 2), (40, 12, 4), 3, 100), ((1, 2, 2), (0, 8, 64), 8, 16))
    for sizes, strides, inner, row in layouts:
        offsets = [sum(i * s for i, s in zip(at, strides + (row,))) for at in itertools.product(*map(range, sizes + (4,)))]
        own = {o + b for o in offsets for b in range(inner)}
        for delta in range(0, max(own) + 3):
            states = (P * 3)(P((1 << 20) + delta), P(1 << 24), P(1 << 20))
            rc, msg = _status("mq_beam_reorder", states, 3, OK, 2, 2, row, (ctypes.c_int64 * 3)(*sizes),
                              (ctypes.c_int64 * 3)(*strides), inner, None)
            meet = any(b + delta in own for b in own)
            assert (rc == -1 and "one another" in msg) if meet else rc == -3, (sizes, strides, inner, row, delta, rc, msg)


def test_sizes_whose_products_pass_64_bits():
    """Refused as too large, not taken for what is left of them after an overflow."""
    from mq._lib import lib

    huge = 1 << 62
    for batch, vocab in ((huge, 1000), (2, huge), (1 << 60, 1 << 60), ((1 << 22) // 4, 1000), (2, (1 << 31) // 4)):
        assert lib.mq_beam_workspace_size(batch, 4, vocab) == 0
        rc, msg = _status("mq_beam_select", OK, 0, vocab, OK, None, -1, OK, OK, OK, None, batch, 4, vocab, OK, 1 << 24, None)
        assert rc == -4 and "large" in msg, (batch, vocab, rc, msg)
    assert lib.mq_beam_workspace_size((1 << 20) - 1, 4, 1000) > 0 and lib.mq_beam_workspace_size(1, 4, 536868000) > 0
    rc, msg = _status("mq_gate_up_w8a8", OK, 64, OK, OK, 64, OK, OK, 0, huge, 4, huge, 64, None)
    assert rc == -4 and "2^30" in msg, (rc, msg)
    rc, msg = _status("mq_gemm_w8a8", OK, 64, OK, OK, 64, OK, None, OK, 0, huge, 4, huge, 64, 0, None)
    assert rc == -4 and "2^30" in msg, (rc, msg)
    states = (P * 2)(OK, P(1 << 24))
    for sizes, strides, row, inner in (((1, 1, 4), (0, 0, 1 << 61), huge, 64), ((1, 1, 1), (0, 0, 0), huge, 64),
                                       ((1, 1, 1), (0, 0, 0), huge, 1 << 61)):
        rc, msg = _status("mq_beam_reorder", states, 2, OK, 2, 4, row, (ctypes.c_int64 * 3)(*sizes),
                          (ctypes.c_int64 * 3)(*strides), inner, None)
        assert rc == -4 and "too large" in msg, (sizes, strides, row, inner, rc, msg)


def test_python_refuses_cpu_tensors():
    import torch

    import mq

    x, w = torch.zeros(2, 16), torch.ones(16)
    for call in (lambda: mq.quantize_s8(x), lambda: mq.pre_norm(x, w), lambda: mq.post_norm(x, w, x),
                 lambda: mq.gemm_w8a8(x.to(torch.int8), w[:2], x.to(torch.int8), w[:2]), lambda: mq.beam_select(x, torch.zeros(1, 2)),
                 lambda: mq.beam_reorder(x, torch.zeros(1, 2, dtype=torch.int32))):
        with pytest.raises(mq.MQError, match="CUDA"):
            call()
