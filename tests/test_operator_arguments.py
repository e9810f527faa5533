"""What the gated delta rule and the group norm refuse on the host, before a GPU is touched."""

import ctypes
import os

import pytest
import torch

from griffin_amd import _lib, hip_gated_delta, hip_gated_delta_step, hip_group_norm

F32, BF16 = _lib.RGLRU_F32, _lib.RGLRU_BF16
FAKE = ctypes.c_void_p(256)                     # never dereferenced: the checks come first
OFF = ctypes.c_void_p(258)
ARG, UNSUPPORTED = 1, 2
HUGE = 1 << 40


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(_lib.LIB_PATH):
        from griffin_amd import build

        build.build()
    return _lib.load()


def fwd(lib, sizes=(2, 100, 2, 4, 64, 64), types=(BF16, F32, F32), strides=None, q=FAKE, v=FAKE, ws=FAKE, flags=None):
    strides = None if strides is None else ctypes.cast((ctypes.c_int64 * 9)(*strides), ctypes.c_void_p)
    return lib.rglru_hip_gated_delta_fwd(q, FAKE, v, strides, FAKE, FAKE, None, flags, FAKE, None, ws, 0, 0.125, *sizes, *types, None)


def bwd(lib, sizes=(2, 100, 2, 4, 64, 64), types=(BF16, F32, F32), dout=FAKE, scratch=FAKE):
    return lib.rglru_hip_gated_delta_bwd(FAKE, FAKE, None, FAKE, FAKE, None, dout, None, FAKE, scratch, FAKE, FAKE, FAKE, FAKE, FAKE, None, 0.125,
                                         *sizes, *types, None)


def step(lib, sizes=(2, 2, 4, 64, 64), types=(BF16, F32, F32), state=FAKE):
    return lib.rglru_hip_gated_delta_step(FAKE, FAKE, FAKE, FAKE, FAKE, state, None, FAKE, 0.125, *sizes, *types, None)


DENSE = (100 * 128, 128, 64, 100 * 128, 128, 64, 100 * 256, 256, 64)


@pytest.mark.parametrize("wrong, code, word", [
    (dict(sizes=(0, 100, 2, 4, 64, 64)), ARG, b"positive"),
    (dict(sizes=(2, 0, 2, 4, 64, 64)), ARG, b"positive"),
    (dict(sizes=(2, 100, 2, 4, 64, 0)), ARG, b"positive"),
    (dict(sizes=(2, 100, 2, 3, 64, 64)), ARG, b"evenly"),
    (dict(sizes=(2, 100, 2, 4, 129, 64)), UNSUPPORTED, b"128"),
    (dict(sizes=(2, 1 << 30, 2, 4, 64, 64)), UNSUPPORTED, b"too large"),
    (dict(sizes=(HUGE, 64, 1, 1, 64, 64)), UNSUPPORTED, b"too large"),
    (dict(sizes=(1, 64, 1 << 20, 1 << 20, 64, 64)), UNSUPPORTED, b"wider"),
    (dict(types=(7, F32, F32)), ARG, b"dtype"),
    (dict(types=(BF16, 7, F32)), ARG, b"dtype"),
    (dict(types=(BF16, F32, -1)), ARG, b"dtype"),
    (dict(q=None), ARG, b"null"),
    (dict(v=None), ARG, b"null"),
    (dict(ws=None), ARG, b"null"),
    (dict(q=OFF), UNSUPPORTED, b"aligned"),
    (dict(v=OFF), UNSUPPORTED, b"aligned"),
    (dict(strides=DENSE[:1] + (-128,) + DENSE[2:]), ARG, b"negative"),
    (dict(strides=DENSE[:1] + (1 << 40,) + DENSE[2:]), UNSUPPORTED, b"apart"),
    (dict(strides=DENSE[:1] + (129,) + DENSE[2:]), UNSUPPORTED, b"aligned"),
    (dict(flags=ctypes.c_void_p(1)), ARG, b"FIRST_RESET"),
])
def test_whole_sequences_are_refused(lib, wrong, code, word):
    assert fwd(lib, **wrong) == code
    assert word in lib.rglru_hip_last_error()


@pytest.mark.parametrize("call, code, word", [
    (lambda lib: bwd(lib, sizes=(2, 100, 3, 4, 64, 64)), ARG, b"evenly"),
    (lambda lib: bwd(lib, sizes=(2, 100, 2, 4, 200, 64)), UNSUPPORTED, b"128"),
    (lambda lib: bwd(lib, types=(BF16, F32, 9)), ARG, b"dtype"),
    (lambda lib: bwd(lib, dout=None), ARG, b"null"),
    (lambda lib: bwd(lib, scratch=None), ARG, b"null"),
    (lambda lib: bwd(lib, dout=OFF), UNSUPPORTED, b"aligned"),
    (lambda lib: step(lib, sizes=(0, 2, 4, 64, 64)), ARG, b"positive"),
    (lambda lib: step(lib, sizes=(2, 2, 4, 129, 64)), UNSUPPORTED, b"128"),
    (lambda lib: step(lib, sizes=(2, 3, 4, 64, 64)), ARG, b"evenly"),
    (lambda lib: step(lib, state=None), ARG, b"null"),
    (lambda lib: step(lib, types=(5, F32, F32)), ARG, b"dtype"),
])
def test_gradients_and_steps_are_refused(lib, call, code, word):
    assert call(lib) == code
    assert word in lib.rglru_hip_last_error()


def test_delta_sizes(lib):
    assert lib.rglru_hip_gated_delta_max_key_size() == 128
    size = lambda T, keep, K=128, dtype=BF16: lib.rglru_hip_gated_delta_workspace_bytes(2, T, 4, 8, K, 128, dtype, keep)
    # T, P and a gate record of 136 numbers for each chunk and value head; kept, the states and the solved values as well
    assert size(640, 0) >= 2 * 8 * 10 * (2 * 64 * 64 * 4 + 136 * 4)
    assert size(640, 1) >= size(640, 0) + 2 * 8 * 10 * (128 + 64) * 128 * 4
    assert size(641, 0) > size(640, 0)
    assert size(640, 0, K=127) > size(640, 0, K=128)                            # room for rows of whole vectors
    assert size(0, 0) == size(640, 0, K=129) == size(640, 0, dtype=3) == 0
    scratch = lib.rglru_hip_gated_delta_scratch_bytes
    assert scratch(2, 640, 8, 128, 128, BF16) >= 2 * 8 * 10 * (128 + 64) * 128 * 4
    assert scratch(2, 640, 0, 128, 128, BF16) == scratch(2, 640, 8, 129, 128, BF16) == 0


def norm_fwd(lib, sizes=(2, 3, 8, 2), activation=0, types=(F32, F32), x=FAKE, scratch=FAKE):
    return lib.rglru_hip_group_norm_fwd(x, None, None, FAKE, None, scratch, *sizes, 1e-5, activation, *types, None)


def norm_bwd(lib, sizes=(2, 3, 8, 2), activation=0, types=(F32, F32, F32), stats=FAKE, scratch=FAKE):
    return lib.rglru_hip_group_norm_bwd(FAKE, None, None, stats, FAKE, scratch, FAKE, None, None, *sizes, activation, *types, None)


@pytest.mark.parametrize("call, code, word", [
    (lambda lib: norm_fwd(lib, sizes=(2, 3, 8, 3)), ARG, b"sizes"),
    (lambda lib: norm_fwd(lib, sizes=(0, 3, 8, 2)), ARG, b"sizes"),
    (lambda lib: norm_fwd(lib, sizes=(2, 3, 8, 0)), ARG, b"sizes"),
    (lambda lib: norm_fwd(lib, activation=9), ARG, b"activation"),
    (lambda lib: norm_fwd(lib, types=(4, F32)), ARG, b"dtype"),
    (lambda lib: norm_fwd(lib, types=(F32, 4)), ARG, b"dtype"),
    (lambda lib: norm_fwd(lib, x=None), ARG, b"null"),
    (lambda lib: norm_fwd(lib, scratch=None), ARG, b"null"),
    (lambda lib: norm_fwd(lib, sizes=(2, 1 << 30, 8, 2)), UNSUPPORTED, b"too large"),
    (lambda lib: norm_fwd(lib, sizes=(2, 3, 1 << 24, 2)), UNSUPPORTED, b"too large"),
    (lambda lib: norm_fwd(lib, sizes=(1 << 27, 1, 64, 8)), UNSUPPORTED, b"too large"),
    (lambda lib: norm_fwd(lib, sizes=(1 << 28, 8, 8192, 1)), UNSUPPORTED, b"too large"),
    (lambda lib: norm_bwd(lib, sizes=(1 << 28, 8, 8192, 1)), UNSUPPORTED, b"too large"),
    (lambda lib: norm_bwd(lib, sizes=(2, 3, 8, 5)), ARG, b"sizes"),
    (lambda lib: norm_bwd(lib, stats=None), ARG, b"null"),
    (lambda lib: norm_bwd(lib, types=(F32, F32, 6)), ARG, b"dtype"),
])
def test_group_norms_are_refused(lib, call, code, word):
    assert call(lib) == code
    assert word in lib.rglru_hip_last_error()
    assert lib.rglru_hip_group_norm_scratch_bytes(2, 3, 8, 3, 0) == 0 < lib.rglru_hip_group_norm_scratch_bytes(2, 3, 8, 2, 1)


def operands(B=2, T=5, H=2, HV=4, K=8, V=6, device="cpu"):
    make = lambda *shape: torch.zeros(*shape, device=device)
    return [make(B, T, H, K), make(B, T, H, K), make(B, T, HV, V), make(B, T, HV), make(B, T, HV)]


def test_no_fallback_on_the_cpu():
    with pytest.raises(RuntimeError):
        hip_gated_delta(*operands())
    with pytest.raises(RuntimeError):
        hip_gated_delta(*operands(), active_mask=torch.ones(2, 5, dtype=torch.bool))
    with pytest.raises(RuntimeError):
        hip_gated_delta_step(*(t[:, 0] for t in operands()), torch.zeros(2, 4, 8, 6))
    with pytest.raises(RuntimeError):
        hip_group_norm(torch.zeros(3, 8), 2)


def test_arguments_that_are_wrong_anywhere():
    for name in ("reset_mask", "active_mask"):
        with pytest.raises(ValueError):
            hip_gated_delta(*operands(), **{name: torch.ones(2, 4, dtype=torch.bool)})
    with pytest.raises(ValueError):
        hip_group_norm(torch.zeros(3, 8), 2, activation="relu")


def swapped(index, tensor):
    made = operands(device="cuda")
    made[index] = tensor if isinstance(tensor, torch.Tensor) else tensor(made[index])
    return made


@pytest.mark.gpu
@pytest.mark.parametrize("error, call", [
    (ValueError, lambda: hip_gated_delta(*swapped(1, lambda t: t[..., :4]))),
    (ValueError, lambda: hip_gated_delta(*swapped(2, lambda t: t[:, :, :3]))),
    (ValueError, lambda: hip_gated_delta(*swapped(2, lambda t: t[:, :4]))),
    (ValueError, lambda: hip_gated_delta(*swapped(3, lambda t: t[:, :, :2]))),
    (ValueError, lambda: hip_gated_delta(*swapped(4, lambda t: t[..., None]))),
    (ValueError, lambda: hip_gated_delta(*(t[:0] for t in operands(device="cuda")))),
    (ValueError, lambda: hip_gated_delta(*(t[:, :0] for t in operands(device="cuda")))),
    (ValueError, lambda: hip_gated_delta(*operands(K=129, device="cuda"))),
    (ValueError, lambda: hip_gated_delta(*operands(device="cuda"), torch.zeros(2, 4, 6, 8, device="cuda"))),
    (TypeError, lambda: hip_gated_delta(*swapped(0, lambda t: t.bfloat16()))),
    (TypeError, lambda: hip_gated_delta(*(t.half() for t in operands(device="cuda")))),
    (TypeError, lambda: hip_gated_delta(*swapped(3, lambda t: t.double()))),
    (RuntimeError, lambda: hip_gated_delta(*swapped(2, lambda t: t.cpu()))),
    (RuntimeError, lambda: hip_gated_delta(*operands(device="cuda"), torch.zeros(2, 4, 8, 6))),
    (ValueError, lambda: hip_gated_delta_step(*(t[:, 0] for t in operands(device="cuda")), torch.zeros(2, 4, 6, 8, device="cuda"))),
    (ValueError, lambda: hip_gated_delta_step(*(t[:, 0] for t in operands(device="cuda")), torch.zeros(2, 4, 6, 8, device="cuda").mT)),
    (ValueError, lambda: hip_gated_delta_step(*(t[:, 0] for t in operands(device="cuda")), torch.zeros(2, 4, 8, 6, device="cuda").bfloat16())),
    (ValueError, lambda: hip_gated_delta_step(*(t[:, 0] for t in operands(device="cuda")), torch.zeros(2, 4, 8, 6, device="cuda"),
                                              flags=torch.zeros(3, dtype=torch.uint8, device="cuda"))),
    (RuntimeError, lambda: hip_gated_delta_step(*(t[:, 0] for t in operands(device="cuda")), torch.zeros(2, 4, 8, 6, device="cuda").requires_grad_())),
    (ValueError, lambda: hip_group_norm(torch.zeros(3, 8, device="cuda"), 3)),
    (ValueError, lambda: hip_group_norm(torch.zeros(3, 8, device="cuda"), 0)),
    (ValueError, lambda: hip_group_norm(torch.zeros(8, device="cuda"), 2)),
    (ValueError, lambda: hip_group_norm(torch.zeros(3, 8, device="cuda"), 2, torch.ones(4, device="cuda"))),
    (TypeError, lambda: hip_group_norm(torch.zeros(3, 8, device="cuda").half(), 2)),
    (RuntimeError, lambda: hip_group_norm(torch.zeros(3, 8, device="cuda"), 2, torch.ones(8))),
])
def test_tensors_that_do_not_fit(error, call):
    with pytest.raises(error):
        call()


def test_partial_gradients_of_many_short_rows_do_not_outgrow_them(lib):
    x = 2 * (1 << 20) * 2 * 64                                                  # a million rows of 2 x 64 in bf16
    assert lib.rglru_hip_group_norm_scratch_bytes(1 << 20, 2, 64, 4, 1) <= x // 4


@pytest.mark.parametrize("call", [
    lambda lib: fwd(lib, sizes=(1 << 20, 1, 1, 1, 1, 1024)),                    # 2^24 workgroups of 64 columns
    lambda lib: fwd(lib, sizes=(1 << 24, 1, 1, 1, 8, 8)),                       # ... of a chunk
    lambda lib: bwd(lib, sizes=(1 << 23, 1, 1, 1, 8, 8)),                       # 2^23 of twice the threads
    lambda lib: norm_fwd(lib, sizes=(1 << 24, 1 << 10, 64, 4)),                 # more than any card holds
    lambda lib: norm_bwd(lib, sizes=(1 << 24, 1 << 10, 64, 4)),
])
def test_launches_of_too_many_threads_are_refused(lib, call):
    assert call(lib) == UNSUPPORTED
    assert b"too large" in lib.rglru_hip_last_error()
