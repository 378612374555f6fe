"""Operators on rows of logits (logit_cases.py): on the device (marked gpu), and from the same sources on the host model
of the kernels (CPU suite), there also with the lanes taken in adverse orders."""
import numpy as np
import pytest
import torch

import emu_lib
import logit_cases as cases
from test_emulated_kernels import E   # noqa: F401  (fixture: the host build)

# vocabulary, bf16, padding of the rows: a wave, four waves and sixteen waves per row, sizes around a vector, odd ones
SHAPES = [(1, False, 0), (1, True, 3), (5, True, 0), (7, False, 2), (16, True, 0), (50, False, 0), (257, True, 0),
          (1000, False, 24), (2047, False, 0), (2051, False, 0), (4099, True, 0), (4096, True, 8), (9001, False, 1),
          (30522, True, 0), (30522, False, 6), (70001, False, 0), (140001, True, 0)]
ON_HOST = [s for s in SHAPES if s[0] < 10000]


def device_backend():
    from sfb import sfb

    def dev(a, bf16=False):
        t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
        return t.to(torch.bfloat16) if bf16 else t
    return sfb, dev


def host_backend(E, **how):
    emu_lib.configure(**how)
    return E, emu_lib.tensor


def top_of(vocab):
    return min(vocab, 20)


@pytest.mark.gpu
@pytest.mark.parametrize("vocab,bf16,pad", SHAPES)
def test_token_logprobs_on_the_device(vocab, bf16, pad):
    cases.logprobs(*device_backend(), vocab, bf16, pad, n=1, k=top_of(vocab), repeat=2)
    cases.logprobs(*device_backend(), vocab, bf16, pad, n=5, k=min(vocab, 64), scale=0.7, seed=3)
    cases.logprobs(*device_backend(), vocab, bf16, pad, n=1, k=1, scale=1.6, seed=4, entropy=False)
    cases.logprobs(*device_backend(), vocab, bf16, pad, n=20, k=min(vocab, 7), seed=6)


@pytest.mark.gpu
@pytest.mark.parametrize("vocab,bf16,pad", SHAPES)
def test_token_logprobs_backward_on_the_device(vocab, bf16, pad):
    cases.logprobs_backward(*device_backend(), vocab, bf16, pad, n=1)
    cases.logprobs_backward(*device_backend(), vocab, bf16, pad, n=7, scale=0.6, entropy=False, in_place=True)


@pytest.mark.gpu
@pytest.mark.parametrize("vocab,bf16,pad", SHAPES)
def test_distillation_on_the_device(vocab, bf16, pad):
    cases.distillation(*device_backend(), vocab, bf16, pad, slots=1)
    cases.distillation(*device_backend(), vocab, bf16, pad, slots=37, teacher_bf16=True, in_place=True, seed=11)
    cases.distillation(*device_backend(), vocab, bf16, pad, slots=256, scale=1.5, seed=12)


CUT = [(9001, False, 1), (30522, True, 0), (70001, False, 0), (140001, True, 0)]   # rows long enough to be cut


@pytest.mark.gpu
@pytest.mark.parametrize("vocab,bf16,pad", CUT)
def test_few_long_rows_cut_over_the_device(vocab, bf16, pad):
    S, dev = device_backend()
    ws = torch.zeros(S.LOGIT_WORKSPACE_BYTES, dtype=torch.uint8, device="cuda")
    for n, k in ((1, 20), (5, 64), (3, 0), (1, 1)):
        cases.logprobs(S, dev, vocab, bf16, pad, n=n, k=k, workspace=ws, repeat=3, seed=20 + k)
        for kind in ("normal", "masked", "nan"):   # one row: the most parts
            cases.logprobs(S, dev, vocab, bf16, pad, n=n, k=k, workspace=ws, kinds=[kind], seed=40 + k)
    torch.cuda.synchronize()
    assert int(ws[:1024].view(torch.int32).abs().sum()) == 0, "arrival counters must be left at zero"


@pytest.mark.gpu
def test_teacher_to_student_on_the_device():
    cases.teacher_to_student(*device_backend())


@pytest.mark.gpu
def test_refusals_on_the_device():
    cases.refusals(*device_backend())


@pytest.mark.parametrize("vocab,bf16,pad", ON_HOST)
def test_token_logprobs_on_the_host_model(E, vocab, bf16, pad):   # noqa: F811
    cases.logprobs(*host_backend(E), vocab, bf16, pad, n=1, k=top_of(vocab))
    cases.logprobs(*host_backend(E), vocab, bf16, pad, n=5, k=min(vocab, 64), scale=0.7, seed=3)
    cases.logprobs(*host_backend(E), vocab, bf16, pad, n=20, k=min(vocab, 7), seed=6)


@pytest.mark.parametrize("vocab,bf16,pad", ON_HOST)
def test_token_logprobs_backward_on_the_host_model(E, vocab, bf16, pad):   # noqa: F811
    cases.logprobs_backward(*host_backend(E), vocab, bf16, pad, n=1)
    cases.logprobs_backward(*host_backend(E), vocab, bf16, pad, n=7, scale=0.6, entropy=False, in_place=True)


@pytest.mark.parametrize("vocab,bf16,pad", ON_HOST)
def test_distillation_on_the_host_model(E, vocab, bf16, pad):   # noqa: F811
    cases.distillation(*host_backend(E), vocab, bf16, pad, slots=1)
    cases.distillation(*host_backend(E), vocab, bf16, pad, slots=37, teacher_bf16=True, in_place=True, seed=11)


@pytest.mark.parametrize("vocab,bf16,order", [(8200, False, 0), (9001, False, 14), (16400, True, 1), (25003, True, 21)])
def test_few_long_rows_cut_on_the_host_model(E, vocab, bf16, order):   # noqa: F811
    S, dev = host_backend(E, order=order)
    ws = dev(np.zeros(S.LOGIT_WORKSPACE_BYTES, np.uint8))
    cases.logprobs(S, dev, vocab, bf16, 3, n=5, k=9, workspace=ws, kinds=["normal", "masked", "rising", "nan", "all lowest", "empty"], repeat=2)
    cases.logprobs(S, dev, vocab, bf16, 0, n=1, k=64, workspace=ws, kinds=["ties"], seed=8)
    assert not ws[:1024].any(), "arrival counters must be left at zero"


@pytest.mark.parametrize("order", [1, 14, 21])
def test_logit_ops_with_lanes_in_adverse_orders(E, order):   # noqa: F811
    back = host_backend(E, order=order)
    cases.logprobs(*back, 2500, False, 1, n=5, k=40)
    cases.logprobs_backward(*back, 2500, False, 1, n=5, in_place=True)
    cases.distillation(*back, 4200, True, 3, slots=70, in_place=True)
    cases.distillation(*back, 900, False, 0, slots=70, in_place=True)


def test_teacher_to_student_on_the_host_model(E):   # noqa: F811
    cases.teacher_to_student(*host_backend(E))


def test_refusals_on_the_host_model(E):   # noqa: F811
    cases.refusals(*host_backend(E))
