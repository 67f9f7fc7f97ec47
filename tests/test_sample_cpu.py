"""CPU: the sampler's argument checks (C ABI and Python), which return before
any device work."""
import ctypes as C

import pytest
import torch

INVALID = 1  # cudaErrorInvalidValue


def test_launch_refusals(native):
    fn = native.lib().ornith_moe_b200_sample_launch
    names = ('logits', 'temperature', 'top_k', 'top_p', 'min_p', 'uniform', 'tokens', 'logprobs', 'flags')
    at = {name: C.c_void_p((1 << 30) + (i << 26)) for i, name in enumerate(names)}

    def call(stride=1000, type=0, m=4, vocab=1000, **changed):
        p = {**at, **changed}
        return fn(p['logits'], stride, type, *[p[n] for n in names[1:]], m, vocab, None)

    assert fn(None, 0, 0, *[None] * 8, 0, 1, None) == 0          # no rows: no pointer is looked at
    assert call(m=-1) == INVALID
    assert call(vocab=0) == INVALID and call(vocab=(1 << 19) + 1, stride=1 << 20) == INVALID
    assert call(type=3) == INVALID and call(type=-1) == INVALID
    assert call(stride=999) == INVALID                           # overlapping rows
    for needed in ('logits', 'uniform', 'tokens', 'flags'):
        assert call(**{needed: None}) == INVALID, needed
    for name in names:
        assert call(**{name: C.c_void_p(at[name].value + 1)}) == INVALID, name   # off its type's alignment
    assert call(type=2, logits=C.c_void_p(at['logits'].value + 2)) == INVALID
    for name in names[:6]:                                       # written over an input
        for written in ('tokens', 'logprobs', 'flags'):
            assert call(**{written: at[name]}) == INVALID, (written, name)
    assert call(tokens=at['logprobs']) == INVALID and call(flags=at['logprobs']) == INVALID
    assert call(flags=C.c_void_p(at['tokens'].value + 12)) == INVALID


def test_python_refuses_cpu_tensors(native):
    with pytest.raises(ValueError):
        native.sample_launch(torch.zeros((2, 16)), None, None, None, None, torch.zeros(2),
                             torch.zeros(2, dtype=torch.int32), None, torch.zeros(1, dtype=torch.int32))


def test_rows_that_wrap_the_address_space(native):
    """Rows times stride beyond 64 bits must not pass for a small tensor."""
    fn = native.lib().ornith_moe_b200_sample_launch
    at = [C.c_void_p((1 << 30) + (i << 32)) for i in range(9)]
    for m, stride, type_ in (((1 << 24) + 1, 1 << 40, 0), ((1 << 22) + 1, 1 << 40, 2), ((1 << 30) + 1, 1 << 33, 1),
                             ((1 << 31) - 1, 1 << 40, 2)):
        assert fn(at[0], stride, type_, *at[1:], m, 1000, None) == INVALID, (m, stride)
