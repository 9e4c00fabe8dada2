"""Refusals of the packed-prompt operators: argument errors come back as
CLEF_EINVAL before anything reaches a device, so they are checked without one."""

from __future__ import annotations

import ctypes

import pytest

from deciax_b200 import _lib
from deciax_b200.build import build

BF16, F32 = _lib.DTYPE_BF16, _lib.DTYPE_F32
P = 4096  # a pointer that no refused call follows


@pytest.fixture(scope="module")
def lib():
    build()
    return _lib.load()


def sections(*values):
    return (ctypes.c_int32 * len(values))(*values)


def rope(lib, **kw):
    a = dict(dtype=BF16, q=P, ldq=512, hsq=128, k=P, ldk=256, hsk=128, qo=P, ldqo=512, hsqo=128, ko=P, ldko=256, hsko=128, pos=P, ldp=10,
             axes=1, sections=None, interleaved=0, tokens=10, hq=4, hkv=2, d=128, rot=64, theta=1e4, qw=P, kw=P, eps=1e-6)
    assert set(kw) <= set(a)
    a.update(kw)
    return lib.clef_op_qk_norm_rope_axes(*a.values(), None)


ROPE_REFUSED = [
    dict(dtype=2), dict(tokens=-1), dict(hq=-1), dict(hq=0, hkv=0), dict(d=0), dict(d=257, rot=64), dict(rot=0), dict(rot=63), dict(rot=130),
    dict(theta=0.5), dict(theta=float("nan")), dict(axes=0), dict(axes=9, sections=sections(*[4] * 9)), dict(axes=2),
    dict(axes=2, sections=sections(16, 15)), dict(axes=2, sections=sections(33, -1)), dict(axes=3, sections=sections(8, 8, 16), interleaved=1),
    dict(axes=2, sections=sections(16, 16), ldp=9), dict(q=None), dict(qo=None), dict(k=None), dict(ko=None), dict(pos=None),
    dict(hsq=127), dict(hsko=64), dict(ldk=100), dict(ldqo=0),
]


@pytest.mark.parametrize("kw", ROPE_REFUSED, ids=lambda kw: "-".join(f"{k}" for k in kw))
def test_rope_axes_refusals(lib, kw):
    assert rope(lib, **kw) == _lib.CLEF_EINVAL
    with pytest.raises(ValueError):
        _lib.check(rope(lib, **kw))


def test_rope_axes_without_tokens_is_a_no_op(lib):
    assert rope(lib, tokens=0, q=None, k=None) == _lib.CLEF_OK


def attention(lib, **kw):
    a = dict(dtype=BF16, q=P, ldq=512, hsq=128, k=P, ldk=256, hsk=128, v=P, ldv=256, hsv=128, gate=P, ldg=512, hsg=128, out=P, ldo=512,
             hso=128, cu=P, n_seqs=2, tokens=10, hq=4, hkv=2, d=128, softcap=0.0, window=0)
    assert set(kw) <= set(a)
    a.update(kw)
    return lib.clef_op_attention_packed(*a.values(), None)


ATTENTION_REFUSED = [
    dict(dtype=-1), dict(n_seqs=-1), dict(tokens=-1), dict(tokens=65535 * 128 + 1), dict(hq=0), dict(hkv=0), dict(hkv=3), dict(hq=65536, hkv=1),
    dict(d=0), dict(d=264), dict(softcap=-1.0), dict(softcap=float("nan")), dict(softcap=float("inf")), dict(window=-1), dict(q=None),
    dict(k=None), dict(v=None), dict(out=None), dict(cu=None), dict(hsq=64), dict(ldk=127), dict(ldv=-256), dict(hsg=0), dict(hso=8),
]


@pytest.mark.parametrize("kw", ATTENTION_REFUSED, ids=lambda kw: "-".join(f"{k}" for k in kw))
def test_attention_packed_refusals(lib, kw):
    assert attention(lib, **kw) == _lib.CLEF_EINVAL


@pytest.mark.parametrize("kw", [dict(n_seqs=0), dict(tokens=0)])
def test_attention_packed_without_rows_is_a_no_op(lib, kw):
    assert attention(lib, q=None, cu=None, **kw) == _lib.CLEF_OK


def logprobs(lib, **kw):
    a = dict(dtype=BF16, hidden=P, ldh=64, head=P, ldw=64, rows=3, vocab=100, dim=64, softcap=0.0, targets=P, n_targets=1, logprobs=P,
             entropy=P, top=4, ids=P, top_logprobs=P)
    assert set(kw) <= set(a)
    a.update(kw)
    return lib.clef_op_token_logprobs(*a.values(), None)


LOGPROBS_REFUSED = [
    dict(dtype=7), dict(rows=-1), dict(rows=(1 << 24) + 1), dict(vocab=0), dict(vocab=(1 << 30) + 1), dict(dim=0), dict(dim=(1 << 20) + 1, ldh=1 << 21, ldw=1 << 21),
    dict(ldh=63), dict(ldw=63), dict(softcap=-2.0), dict(softcap=float("inf")), dict(n_targets=-1), dict(top=-1), dict(top=33),
    dict(top=9, vocab=8), dict(hidden=None), dict(head=None), dict(targets=None), dict(logprobs=None), dict(ids=None),
    dict(top_logprobs=None), dict(n_targets=0, top=0, entropy=None),
]


@pytest.mark.parametrize("kw", LOGPROBS_REFUSED, ids=lambda kw: "-".join(f"{k}" for k in kw))
def test_token_logprobs_refusals(lib, kw):
    assert logprobs(lib, **kw) == _lib.CLEF_EINVAL


def test_token_logprobs_without_rows_is_a_no_op(lib):
    assert logprobs(lib, rows=0, hidden=None, head=None) == _lib.CLEF_OK


# A kernel that reads a value across its type's alignment faults: such an operand is refused without a look at the device.
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("name", ["q", "k", "qo", "ko", "pos", "qw", "kw"])
def test_rope_axes_refuses_pointers_inside_a_value(lib, name, dtype):
    off = 2 if name == "pos" or dtype == F32 else 1
    assert rope(lib, dtype=dtype, **{name: P + off}) == _lib.CLEF_EINVAL


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("name", ["q", "k", "v", "gate", "out", "cu"])
def test_attention_packed_refuses_pointers_inside_a_value(lib, name, dtype):
    off = 2 if name == "cu" or dtype == F32 else 1
    assert attention(lib, dtype=dtype, **{name: P + off}) == _lib.CLEF_EINVAL


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("name", ["hidden", "head", "targets", "logprobs", "entropy", "ids", "top_logprobs"])
def test_token_logprobs_refuses_pointers_inside_a_value(lib, name, dtype):
    off = 1 if name in ("hidden", "head") and dtype == BF16 else 2
    assert logprobs(lib, dtype=dtype, **{name: P + off}) == _lib.CLEF_EINVAL
