"""CPU: what the training calls refuse before any device work (code 1), and the binding's own checks."""
from __future__ import annotations

import pytest

A, B, C = 1 << 20, 1 << 21, 1 << 22  # 16-byte aligned addresses that nothing may read


@pytest.mark.parametrize("name", ["spaceslug_act8_pack_device", "spaceslug_act8_unpack_device"])
@pytest.mark.parametrize("x,codes,exps,dtype,m,k", [
    (None, A, B, 0, 1, 32), (C, None, B, 0, 1, 32), (C, A, None, 0, 1, 32),  # null pointers
    (C, A, B, 2, 1, 32), (C, A, B, -1, 1, 32),                              # no such element type
    (C, A, B, 0, 0, 32), (C, A, B, 0, 1, 0), (C, A, B, 1, 4, 48),           # empty, k % 32
    (C + 4, A, B, 0, 1, 32), (C + 2, A, B, 1, 1, 32), (C, A + 8, B, 0, 1, 32),  # alignment
    (C, A, B, 0, (1 << 30) + 1, 32), (C, A, B, 0, 1 << 20, 1 << 21)])       # too large
def test_act8_refuses(session, name, x, codes, exps, dtype, m, k):
    f = session.raw(name)
    args = (x, dtype, codes, exps, m, k, None) if "unpack" not in name else (codes, exps, x, dtype, m, k, None)
    assert f(*args) == 1
    assert session._native().spaceslug_last_error()


@pytest.mark.parametrize("name", ["spaceslug_act8_pack_device", "spaceslug_act8_unpack_device"])
@pytest.mark.parametrize("x,codes,exps", [(C, C, B), (C, C + 64 * 96 * 2 - 16, B), (C + 64 * 96 - 16, C, B), (C, A, C + 5),
                                          (C, A, C - 191)])
def test_act8_refuses_overlap(session, name, x, codes, exps):
    """64 x 96 bf16: x 12288 bytes, codes 6144, exps 192; what is written shares a byte with another buffer."""
    f = session.raw(name)
    args = (x, 1, codes, exps, 64, 96, None) if "unpack" not in name else (codes, exps, x, 1, 64, 96, None)
    assert f(*args) == 1
    assert b"overlaps" in session._native().spaceslug_last_error()


def test_handle_calls_refuse_null(session):
    back, grad, loss = (session.raw("spaceslug_q4_weights_" + n) for n in
                        ("lora_backward_act8", "input_gradient", "cross_entropy"))
    assert back(None, A, B, C, 0, 4, None, None, None) == 1
    assert grad(None, A, B, 0, 4, None) == 1
    assert loss(None, A, 0, B, None, C, None, None, 4, None) == 1


def test_binding_names_element_types(session):
    from spaceslug_b200.backend import BackendError
    with pytest.raises(BackendError, match="dtype"):
        session.act8_pack_device(C, A, B, 1, 32, dtype="f16")


def test_capabilities_list_the_training_calls(session):
    assert {"act8_checkpoint", "lora_training_act8", "q4_input_gradient", "q4_cross_entropy"} <= set(session.capabilities())


def test_scratch_hook_bounds(session):
    hook = session.raw("spaceslug_q4_debug_train_scratch")
    assert hook((1 << 30) + 1, 0) == 1 and hook(0, (1 << 32) + 1) == 1
    assert hook(1, 1) == 0 and hook(0, 0) == 0
