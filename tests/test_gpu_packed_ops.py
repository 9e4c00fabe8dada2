"""Packed-prompt operators against plain 64-bit implementations.

Tolerances are derived, not fitted.  u is half a step of the output type
(bf16 2^-8 of the value's power of two, so at most 2^-8 relative; fp32 2^-24).

* Rotary: y = x r (1 + w) carries a handful of FP32 roundings (sum of d squares
  in 32 lanes: (d/32 + 5) 2^-24 relative on the mean, halved by the root; rsqrt
  and three products: 4 * 2^-24), the angle at most 2^-24 of half a turn (so
  pi 2^-24 on cos and sin) plus sincospi's 2 ulp, and the rotation two products
  and a sum of |y_lo| + |y_hi|.  All together below 32 * 2^-24 (|y_lo| + |y_hi|);
  a bf16 result adds u |out|.
* Attention, with A = sum_j p_j |v_j| / l over a row's own keys: a score of d
  products in FP32 is off by at most e = (d + 8) 2^-24 sum_c |q_c k_c| / sqrt d (and
  as much again for sums that truncate, and for tanh under a cap), which moves
  each p, and l, by that factor: 4 e A.  P rounded to bf16 (tensor cores) adds
  2^-8 A; FP32 sums of n terms add n 2^-24 A; exponentials and the sigmoid are
  good to 2^-21.  The store adds u |out|.
* Log probabilities, with e = 2 (dim + 8) 2^-24 max_v sum_c |h_c w_c| for a score's
  products: z and lse are each off by e, by 2^-23 of their size and lse by the
  relative error r = (vocab / 32 + 64) 2^-24 + 2^-20 of the sum of exponentials
  (vocab / 32 additions to a running sum; exponents to 2^-20).  The entropy's
  two sums carry e and r against sum p |z - max| + 1.  Ids have to be equal:
  operands lie on a grid on which every score is exact in FP32.
"""

from __future__ import annotations

import ctypes

import numpy as np
import pytest

from deciax_b200 import _lib

pytestmark = pytest.mark.gpu
U32 = 2.0**-24
U = {"bf16": 2.0**-8, "fp32": U32}


def lib():
    return _lib.load()


def code(dtype: str) -> int:
    return _lib.DTYPE_BF16 if dtype == "bf16" else _lib.DTYPE_F32


def torch_type(dtype: str):
    import torch

    return torch.bfloat16 if dtype == "bf16" else torch.float32


def normal(g, *shape, dtype="bf16", std=1.0):
    import torch

    return (torch.randn(*shape, generator=g, device="cuda") * std).to(torch_type(dtype))


def generator(seed):
    import torch

    return torch.Generator(device="cuda").manual_seed(seed)


def stream():
    import torch

    return torch.cuda.current_stream().cuda_stream


# --------------------------------------------------------------------------- rotary positions


def run_rope(q, k, q_out, k_out, positions, sections, interleaved, rot, theta, q_norm, k_norm, eps=1e-6):
    """q, k and outputs [tokens, heads, d] with any strides whose last is 1; positions [axes, tokens]."""
    t, _, d = (q if q is not None else k).shape
    args = []
    for x in (q, k, q_out, k_out):
        args += [None, 0, 0] if x is None else [x.data_ptr(), x.stride(0), x.stride(1)]
    sec = (ctypes.c_int32 * len(sections))(*sections) if sections else None
    status = lib().clef_op_qk_norm_rope_axes(
        code("bf16" if (q if q is not None else k).element_size() == 2 else "fp32"), *args, positions.data_ptr(), positions.stride(0),
        positions.shape[0], sec, int(interleaved), t, q.shape[1] if q is not None else 0, k.shape[1] if k is not None else 0, d, rot, theta,
        q_norm.data_ptr() if q_norm is not None else None, k_norm.data_ptr() if k_norm is not None else None, eps, stream())
    _lib.check(status)


def axis_of_pairs(sections, interleaved, half):
    if not sections:
        return [0] * half
    if not interleaved:
        return [a for a, n in enumerate(sections) for _ in range(n)]
    n = len(sections)
    return [i % n if i // n < sections[i % n] else 0 for i in range(half)]


def rope_64(x, w, positions, sections, interleaved, rot, theta, eps=1e-6):
    """(expected, scale of its rounding error), in 64 bits on the host."""
    x = x.double().cpu().numpy()
    half = rot // 2
    y = x
    if w is not None:
        y = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * (1 + w.double().cpu().numpy())
    axis = axis_of_pairs(sections, interleaved, half)
    pos = positions.cpu().numpy().astype(np.longdouble)
    theta = np.longdouble(np.float32(theta))
    angle = pos[axis].T * theta ** (np.longdouble(-2) * np.arange(half) / rot)
    cos, sin = np.cos(angle).astype(np.float64)[:, None], np.sin(angle).astype(np.float64)[:, None]
    lo, hi = y[..., :half], y[..., half:rot]
    out = np.concatenate((lo * cos - hi * sin, hi * cos + lo * sin, y[..., rot:]), -1)
    size = np.abs(lo) + np.abs(hi)
    return out, np.concatenate((size, size, np.abs(y[..., rot:])), -1)


def assert_rope(got, expected, scale, dtype):
    got = got.double().cpu().numpy()
    tol = 32 * U32 * scale + (U["bf16"] * np.abs(expected) if dtype == "bf16" else 0) + 1e-30
    worst = np.abs(got - expected) / tol
    assert worst.max() <= 1, (worst.max(), np.unravel_index(worst.argmax(), worst.shape))


ROPE_CASES = [
    # tokens, hq, hkv, d, rot, sections, interleaved, first position
    (1, 16, 8, 256, 64, None, False, 0),
    (129, 16, 8, 256, 64, None, False, 0),
    (37, 4, 2, 128, 128, (24, 20, 20), False, 70000),
    (37, 4, 2, 128, 128, (24, 20, 20), True, 70000),
    (50, 3, 1, 64, 32, (6, 5, 5), True, -1000),
    (50, 3, 1, 96, 96, (16, 0, 16, 16), False, 5),
    (9, 2, 2, 80, 20, (4, 6), False, 1 << 30),
    (9, 2, 2, 30, 14, (5, 2), True, 123),
    (3, 1, 1, 2, 2, None, False, 9),
    (65, 32, 16, 128, 64, (16, 16), True, (1 << 31) - 70),
    (300, 14, 2, 256, 256, None, False, 2000000),
    (5, 0, 3, 64, 64, None, False, 11),
    (5, 3, 0, 48, 16, None, False, 11),
]


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("case", ROPE_CASES, ids=str)
def test_rope_axes(case, dtype):
    import torch

    t, hq, hkv, d, rot, sections, interleaved, first = case
    g = generator(t + d + rot)
    q, k = normal(g, t, hq, d, dtype=dtype, std=3.0), normal(g, t, hkv, d, dtype=dtype)
    qw, kw = normal(g, d, dtype=dtype, std=0.2), normal(g, d, dtype=dtype, std=0.2)
    axes = len(sections) if sections else 1
    pos = torch.stack([(torch.arange(t, device="cuda", dtype=torch.int64) // (1 + 3 * a) + first).clamp_(max=2**31 - 1)
                       for a in range(axes)]).int()
    qo, ko = torch.full_like(q, 7.0), torch.full_like(k, 7.0)
    run_rope(q if hq else None, k if hkv else None, qo if hq else None, ko if hkv else None, pos, sections, interleaved, rot, 1e4, qw, kw)
    for x, w, o in ((q, qw, qo), (k, kw, ko)):
        if x.shape[1]:
            assert_rope(o, *rope_64(x, w, pos, sections, interleaved, rot, 1e4), dtype)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("d,rot,shift", [(256, 64, 0), (128, 128, 0), (64, 32, 1), (40, 24, 4)])
def test_rope_axes_in_place_on_a_packed_projection(d, rot, shift, dtype):
    """The packed projection [q | gate per head, k, v] rotated in place, at a row
    stride with slack and (shift) away from 16-byte boundaries: gate, v and the
    slack keep their bits."""
    import torch

    hq, hkv, t = 4, 2, 33
    width = 2 * hq * d + 2 * hkv * d
    g = generator(d + shift)
    buf = normal(g, t, width + 24, dtype=dtype)
    before = buf.clone()
    view = buf[:, shift : shift + width]
    q, k = view[:, : 2 * hq * d].view(t, hq, 2 * d)[..., :d], view[:, 2 * hq * d : 2 * hq * d + hkv * d].view(t, hkv, d)
    pos = torch.arange(t, device="cuda", dtype=torch.int32)[None] + 100
    qw, kw = normal(g, d, dtype=dtype, std=0.2), normal(g, d, dtype=dtype, std=0.2)
    qe, ke = rope_64(q, qw, pos, None, False, rot, 5e5), rope_64(k, kw, pos, None, False, rot, 5e5)
    run_rope(q, k, q, k, pos, None, False, rot, 5e5, qw, kw)
    assert_rope(q, *qe, dtype)
    assert_rope(k, *ke, dtype)
    touched = torch.zeros_like(buf, dtype=torch.bool)
    tv = touched[:, shift : shift + width]
    tv[:, : 2 * hq * d].view(t, hq, 2 * d)[..., :d] = True
    tv[:, 2 * hq * d : 2 * hq * d + hkv * d] = True
    assert torch.equal(buf[~touched], before[~touched])


@pytest.mark.parametrize("d,rot", [(128, 64), (36, 12)])
def test_rope_axes_without_norm_keeps_the_tail(d, rot):
    import torch

    g = generator(1)
    q = normal(g, 17, 3, d)
    pos = torch.randint(-(2**31), 2**31 - 1, (1, 17), generator=g, device="cuda").int()
    out = torch.empty_like(q)
    run_rope(q, None, out, None, pos, None, False, rot, 1e6, None, None)
    assert_rope(out, *rope_64(q, None, pos, None, False, rot, 1e6), "bf16")
    assert torch.equal(out[..., rot:], q[..., rot:])


def test_rope_axes_zero_rows_and_infinities_stay_in_their_head():
    """A zero head stays zero (eps), an infinite one spoils only itself."""
    import torch

    q = normal(generator(2), 4, 3, 128)
    q[1, 1] = 0
    q[2, 0, 5] = float("inf")
    out, w = torch.empty_like(q), torch.zeros(128, dtype=torch.bfloat16, device="cuda")
    pos = torch.arange(4, device="cuda", dtype=torch.int32)[None]
    run_rope(q, None, out, None, pos, None, False, 64, 1e4, w, None)
    assert (out[1, 1] == 0).all()
    ok = torch.ones(4, 3, dtype=torch.bool, device="cuda")
    ok[2, 0] = False
    assert torch.isfinite(out[ok]).all() and out[2, 0].isnan().any()


def test_rope_axes_refuses_host_memory():
    import torch

    x = torch.zeros(2, 1, 64, dtype=torch.bfloat16)
    pos = torch.zeros(1, 2, dtype=torch.int32)
    with pytest.raises(ValueError, match="current device"):
        run_rope(x, None, x, None, pos, None, False, 64, 1e4, None, None)


def test_rope_axes_captured_and_replayed_on_another_stream():
    import torch

    g = generator(3)
    q = normal(g, 40, 4, 128)
    out, pos = torch.empty_like(q), torch.arange(40, device="cuda", dtype=torch.int32)[None].contiguous()
    w = normal(g, 128, std=0.1)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run_rope(q, None, out, None, pos, None, False, 64, 1e4, w, None)
    for shift in (0, 1000):
        pos.copy_(torch.arange(40, device="cuda")[None] + shift)
        graph.replay()
        assert_rope(out, *rope_64(q, w, pos, None, False, 64, 1e4), "bf16")


def test_rope_axes_replayed_on_a_stream_of_its_own():
    """The graph runs behind what its stream holds, not on the stream that captured it."""
    import torch

    g = generator(28)
    q, other = normal(g, 4000, 4, 128), normal(g, 4000, 4, 128)
    out, pos = torch.empty_like(q), torch.arange(4000, device="cuda", dtype=torch.int32)[None].contiguous()
    w = normal(g, 128, std=0.1)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run_rope(q, None, out, None, pos, None, False, 64, 1e4, w, None)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        q.copy_(other)
        graph.replay()
    side.synchronize()
    assert_rope(out, *rope_64(other, w, pos, None, False, 64, 1e4), "bf16")


# --------------------------------------------------------------------------- packed attention


def run_attention(q, k, v, gate, out, cu, softcap=0.0, window=0):
    args = []
    for x in (q, k, v, gate, out):
        args += [None, 0, 0] if x is None else [x.data_ptr(), x.stride(0), x.stride(1)]
    t, hq, d = q.shape
    _lib.check(lib().clef_op_attention_packed(code("bf16" if q.element_size() == 2 else "fp32"), *args, cu.data_ptr(), cu.numel() - 1, t, hq,
                                              k.shape[1], d, softcap, window, stream()))


def attention_64(q, k, v, gate, bounds, softcap, window, rounded_p):
    """{(first, end): (expected [rows, heads, d], tolerance before the store)} of each sequence, in 64 bits."""
    import torch

    hq, hkv, d = q.shape[1], k.shape[1], q.shape[2]
    found = {}
    for a, b in zip(bounds[:-1], bounds[1:]):
        if a == b:
            continue
        qs = q[a:b].double().transpose(0, 1)
        ks, vs = (x[a:b].double().transpose(0, 1).repeat_interleave(hq // hkv, 0) for x in (k, v))
        s = qs @ ks.transpose(1, 2) / d**0.5
        e = (d + 8) * U32 * (qs.abs() @ ks.abs().transpose(1, 2)) / d**0.5
        if softcap:
            s = softcap * torch.tanh(s / softcap)
        i = torch.arange(b - a, device="cuda")
        ago = i[:, None] - i
        seen = (ago >= 0) & ((ago < window) if window else True)
        s = s.masked_fill(~seen, float("-inf"))
        p = torch.softmax(s, -1)
        e = torch.where(seen, e, 0).amax(-1, keepdim=True)
        y, size = p @ vs, p @ vs.abs()
        g = torch.sigmoid(gate[a:b].double().transpose(0, 1)) if gate is not None else 1.0
        tol = (4 * e + (2.0**-8 if rounded_p else 0) + (b - a + 16) * U32 + 2.0**-21) * size * g
        found[a, b] = (y * g).transpose(0, 1), tol.transpose(0, 1)
    return found


def check_attention(lens, hq, hkv, d, dtype="bf16", *, gate=True, softcap=0.0, window=0, layout="packed", lead=0, pad=0, qscale=1.0, seed=0,
                    tensor_cores=True, spoil=None):
    import torch

    g = generator(seed + d + len(lens))
    n = lead + sum(lens)
    t = n + pad
    bounds = [lead]
    for x in lens:
        bounds.append(bounds[-1] + x)
    if layout in ("packed", "odd"):  # one projection [q | gate per head, k, v]; odd: off 16-byte boundaries
        width, off = 2 * hq * d + 2 * hkv * d, 1 if layout == "odd" else 0
        proj = normal(g, t, width + 8 + off, dtype=dtype)[:, off : off + width]
        heads = proj[:, : 2 * hq * d].unflatten(1, (hq, 2 * d))
        q, gt = heads[..., :d], heads[..., d:]
        k = proj[:, 2 * hq * d : 2 * hq * d + hkv * d].unflatten(1, (hkv, d))
        v = proj[:, 2 * hq * d + hkv * d :].unflatten(1, (hkv, d))
        out = normal(g, t, hq, d, dtype=dtype)
    elif layout == "heads":  # [heads, rows, d]
        q, gt, k, v, out = (normal(g, h, t, d, dtype=dtype).transpose(0, 1) for h in (hq, hq, hkv, hkv, hq))
    else:
        q, gt, k, v, out = (normal(g, t, h, d, dtype=dtype) for h in (hq, hq, hkv, hkv, hq))
    q.mul_(qscale)
    for x in (q, gt, k, v):  # rows of no sequence hold anything
        x[:lead] = float("nan")
        x[n:] = float("inf")
        x[n + 1 :] = float("nan")
    spoiled = spoil(bounds, q, k, v) if spoil else ()
    before = out.clone()
    cu = torch.tensor(bounds, dtype=torch.int32, device="cuda")
    run_attention(q, k, v, gt if gate else None, out, cu, softcap, window)
    assert torch.equal(out[:lead], before[:lead]) and torch.equal(out[n:], before[n:])
    u = U[dtype]
    for (a, b), (y, tol) in attention_64(q, k, v, gt if gate else None, bounds, softcap, window, tensor_cores and dtype == "bf16").items():
        if (a, b) in spoiled:
            continue
        off = (out[a:b].double() - y).abs() / (tol + u * y.abs() + 1e-30)
        assert off.max() <= 1, ((a, b), off.max().item(), (off.isnan().sum()).item(), np.unravel_index(off.argmax().item(), off.shape))
    return out, bounds


LENGTHS = {
    "one": [1], "tile": [128], "small": [1, 31, 64], "empty": [0, 0, 5, 0, 130, 0], "ragged": [257, 1, 1, 300], "long": [700],
    "many": [(7 * i * i + 3 * i) % 21 for i in range(120)],
}


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("lens", LENGTHS)
def test_attention_packed_lengths(lens, d, dtype):
    check_attention(LENGTHS[lens], 4, 2, d, dtype, pad=37 if lens != "tile" else 0)


@pytest.mark.parametrize("hq,hkv", [(1, 1), (8, 1), (6, 3), (14, 2)])
@pytest.mark.parametrize("layout", ["packed", "heads", "split"])
@pytest.mark.parametrize("gate", [True, False])
def test_attention_packed_heads_and_strides(hq, hkv, layout, gate):
    check_attention([100, 60, 33], hq, hkv, 128, gate=gate, layout=layout, pad=3, lead=5)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("d", [8, 40, 72, 96, 200])
def test_attention_packed_other_head_sizes(d, dtype):
    check_attention([140, 3, 77], 4, 2, d, dtype, layout="split", pad=60)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("d,layout", [(30, "packed"), (64, "odd"), (1, "split"), (255, "heads")])
def test_attention_packed_unaligned_rows(d, layout, dtype):
    check_attention([90, 0, 41], 4, 2, d, dtype, layout=layout, pad=2, tensor_cores=False)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("window,softcap", [(1, 0.0), (50, 0.0), (200, 5.0), (0, 30.0), (1 << 30, 0.0)])
def test_attention_packed_window_and_softcap(window, softcap, d, dtype):
    check_attention([300, 17, 260], 2, 1, d, dtype, window=window, softcap=softcap, qscale=3.0, pad=1)


@pytest.mark.parametrize("d", [64, 128, 256])
def test_attention_packed_long_rows_with_large_scores(d):
    """The running maximum moves often: O is rescaled in tensor memory."""
    check_attention([1500, 20, 600], 2, 1, d, qscale=6.0)


@pytest.mark.parametrize("d", [64, 128, 256])
def test_attention_packed_scores_that_jump(d):
    """Scores of some +-2000: they grow by more than FP32's range from one key tile to the next."""
    check_attention([400, 7, 300], 2, 1, d, qscale=500.0, pad=9)


@pytest.mark.parametrize("dtype,tokens", [("bf16", 4500), ("fp32", 1100)])
def test_attention_packed_benchmark_heads(dtype, tokens):
    check_attention([tokens], 16, 8, 256, dtype)


@pytest.mark.parametrize("dtype,d", [("bf16", 64), ("bf16", 128), ("bf16", 256), ("fp32", 64), ("fp32", 256)])
def test_attention_packed_infinities_stay_in_their_sequence(dtype, d):
    """Values and keys of the middle sequence are infinite or NaN: its rows from
    there on are, and its earlier rows and every other sequence keep their values."""

    def spoil(bounds, q, k, v):
        a = bounds[1]
        v[a + 20, 0, 3] = float("inf")
        v[a + 25, :, :] = float("nan")
        k[a + 30, 0, 0] = float("nan")
        return [(bounds[1], bounds[2])]

    out, bounds = check_attention([40, 35, 30, 100], 4, 2, d, dtype, spoil=spoil, pad=30)
    a = bounds[1]
    assert out[a : a + 20].isfinite().all()
    assert (~out[a + 20 : bounds[2], :2, 3].isfinite()).all()
    assert out[a + 20 : a + 25, 2:].isfinite().all() and out[a + 25 : bounds[2]].isnan().any(-1).all()


@pytest.mark.parametrize("dtype,d", [("bf16", 64), ("bf16", 128), ("bf16", 256), ("fp32", 64), ("fp32", 256)])
def test_attention_packed_scores_of_minus_infinity(dtype, d):
    """A key whose score is -inf has weight 0; a row that sees no other key is NaN."""
    import torch

    g = generator(21)
    q, k, v, out = (normal(g, 560, h, d, dtype=dtype) for h in (2, 1, 1, 2))
    q[40:500, :, 0] = q[40:500, :, 0].abs() + 0.5
    k[40:240, 0, 0] = float("-inf")
    v[500:] = float("nan")  # the next sequence, in the same tiles
    run_attention(q, k, v, None, out, torch.tensor([0, 40, 500, 560], dtype=torch.int32, device="cuda"))
    assert out[40:240].isnan().all() and out[500:].isnan().all()
    # a row after those keys is that of a sequence without them
    for a, b in ((0, 40), (240, 500)):
        y, tol = attention_64(q, k, v, None, [a, b], 0.0, 0, dtype == "bf16")[a, b]
        assert ((out[a:b].double() - y).abs() <= tol + U[dtype] * y.abs()).all()


def attention_of_seen_keys(q, k, v, seen, rounded_p):
    """(expected [rows, heads, d], tolerance before the store) of one sequence whose row i sees the keys seen[i], in 64 bits."""
    import torch

    hq, hkv, d = q.shape[1], k.shape[1], q.shape[2]
    qs, ks, vs = q.double().transpose(0, 1), *(x.double().transpose(0, 1).repeat_interleave(hq // hkv, 0) for x in (k, v))
    p = torch.softmax((qs @ ks.transpose(1, 2) / d**0.5).masked_fill(~seen, float("-inf")), -1)
    e = (d + 8) * U32 * (qs.abs() @ ks.abs().transpose(1, 2)) / d**0.5
    e = torch.where(seen, e, 0).amax(-1, keepdim=True)
    tol = (4 * e + (2.0**-8 if rounded_p else 0) + (q.shape[0] + 16) * U32 + 2.0**-21) * (p @ vs.abs())
    return (p @ vs).transpose(0, 1), tol.transpose(0, 1)


@pytest.mark.parametrize("low", [False, True])
@pytest.mark.parametrize("n,blocked", [(560, slice(300, None)), (560, slice(128, None, 128)), (560, slice(64, None, 64)), (128, slice(64, None)),
                                       (256, slice(128, None))])
@pytest.mark.parametrize("dtype,d", [("bf16", 64), ("bf16", 128), ("bf16", 256), ("fp32", 64), ("fp32", 128), ("fp32", 256)])
def test_attention_packed_own_keys_of_minus_infinity(dtype, d, n, blocked, low):
    """Rows whose nearest keys (their own among them) score -inf answer from the keys before those.
    low: those score -87, near the end of FP32's exponents below 0."""
    import torch

    g = generator(25)
    q, k, v, out = (normal(g, n, h, d, dtype=dtype) for h in (2, 1, 1, 2))
    q[:, :, 0] = q[:, :, 0].abs() + 0.5
    if low:
        q[:, :, 2:].mul_(4)  # scores a few nats apart
        q[:, :, 1], k[:, :, 1] = 16, -87 * d**0.5 / 16
    i = torch.arange(n, device="cuda")
    seen = i[:, None] >= i
    seen[:, blocked] = False
    y, tol = attention_of_seen_keys(q, k, v, seen, dtype == "bf16")
    k[blocked, :, 0] = float("-inf")
    run_attention(q, k, v, None, out, torch.tensor([0, n], dtype=torch.int32, device="cuda"))
    off = (out.double() - y).abs() / (tol + U[dtype] * y.abs() + 1e-30)
    assert off.max() <= 1, (off.max().item(), off.isnan().sum().item(), (off.amax((1, 2)) > 1).nonzero()[:, 0].tolist())


@pytest.mark.parametrize("dtype,d", [("bf16", 64), ("bf16", 128), ("bf16", 256), ("fp32", 128), ("fp32", 256)])
def test_attention_packed_scores_that_jump_by_the_range_of_the_exponent(dtype, d):
    """One key's score is 84 to 92 above those of the keys between it and the row, 2^121 to 2^133 in weight,
    and keys before it score a little more than those: a finite weight whose inverse FP32 does not hold."""

    def spoil(bounds, q, k, v):
        import torch

        q.mul_(0.3), k.mul_(0.3)
        q[:, :, 0], k[:, :, 0] = 16, 0
        k[:64, :, 0] = 6 * d**0.5 / 16
        k[200, :, 0] = (84 + 0.5 * torch.arange(16, device="cuda")) * d**0.5 / 16
        return ()

    check_attention([512], 16, 16, d, dtype, layout="split", gate=False, spoil=spoil)


@pytest.mark.parametrize("dtype,d", [("bf16", 64), ("bf16", 128), ("bf16", 256), ("fp32", 64), ("fp32", 256)])
def test_attention_packed_a_prompt_gone_nan(dtype, d):
    """All of the middle sequence is NaN; its neighbours keep their values."""
    import torch

    g = generator(22)
    cu = torch.tensor([0, 70, 400, 470], dtype=torch.int32, device="cuda")
    q, k, v, gt = (normal(g, 470, h, d, dtype=dtype) for h in (4, 2, 2, 4))
    out = torch.empty_like(q)
    for x in (q, k, v, gt):
        x[70:400] = float("nan")
    run_attention(q, k, v, gt, out, cu)
    assert out[70:400].isnan().all()
    for a, b in ((0, 70), (400, 470)):
        y, tol = attention_64(q, k, v, gt, [a, b], 0.0, 0, dtype == "bf16")[a, b]
        assert ((out[a:b].double() - y).abs() <= tol + U[dtype] * y.abs()).all()


@pytest.mark.parametrize("dtype,d", [("bf16", 128), ("bf16", 256), ("fp32", 128)])
def test_attention_packed_one_infinite_value_is_no_thousand_passes(dtype, d):
    """Every later row of the prompt is computed once more, as the rows' own keys ask: by warps side by side
    (one row after the other they took 700 times the plain call at 128 and 1000 at 256; by warps, 50 to 160)."""
    import torch

    g = generator(26)
    q, k, v, out = (normal(g, 2048, h, d, dtype=dtype) for h in (16, 8, 8, 16))
    cu = torch.tensor([0, 2048], dtype=torch.int32, device="cuda")

    def took():
        best = 1e9
        for _ in range(3):
            start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            start.record()
            run_attention(q, k, v, None, out, cu)
            end.record()
            torch.cuda.synchronize()
            best = min(best, start.elapsed_time(end))
        return best

    plain = took()
    v[0, 0, 0] = float("inf")
    assert took() < 450 * plain
    assert (out[:, :2, 0] == float("inf")).all() and out[:, :, 1:].isfinite().all()


@pytest.mark.parametrize("dtype,d", [("bf16", 128), ("bf16", 30), ("fp32", 64)])
def test_attention_packed_offsets_past_32_bits(dtype, d):
    """The last rows of buffers of more than 2^31 elements."""
    import torch

    hq, ld = 2, 1 << 16
    t = (1 << 31) // ld + 200
    buf = torch.empty(t, ld, dtype=torch_type(dtype), device="cuda")
    n, at = 150, t - 170
    buf[at:] = normal(generator(4), t - at, ld, dtype=dtype)
    q, k, v, out = (buf[:, i * hq * d : (i + 1) * hq * d].unflatten(1, (hq, d)) for i in range(4))
    cu = torch.tensor([at, at + 100, at + n], dtype=torch.int32, device="cuda")
    run_attention(q, k, v, None, out, cu)
    for (a, b), (y, tol) in attention_64(q, k, v, None, [at, at + 100, at + n], 0.0, 0, d == 128).items():
        assert ((out[a:b].double() - y).abs() <= tol + U[dtype] * y.abs()).all()


def test_attention_packed_captured_and_replayed_with_other_lengths():
    """The lengths are device data: a captured call follows them."""
    import torch

    g = generator(5)
    q, k, v, out = (normal(g, 400, h, 128) for h in (4, 2, 2, 4))
    cu = torch.tensor([0, 100, 400, 400], dtype=torch.int32, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run_attention(q, k, v, None, out, cu)
    for bounds in ([0, 100, 400, 400], [0, 1, 1, 333], [10, 200, 201, 390]):
        cu.copy_(torch.tensor(bounds))
        out.fill_(7)
        graph.replay()
        for (a, b), (y, tol) in attention_64(q, k, v, None, bounds, 0.0, 0, True).items():
            assert ((out[a:b].double() - y).abs() <= tol + U["bf16"] * y.abs()).all()
        assert (out[: bounds[0]] == 7).all() and (out[bounds[-1] :] == 7).all()


@pytest.mark.parametrize("d", [64, 128])
def test_attention_packed_fp32_graphs_and_streams_have_their_own_scratch(d):
    """Two captured calls replayed side by side, and eager calls on two streams."""
    import torch

    g = generator(23)
    cu = torch.tensor([0, 150, 400], dtype=torch.int32, device="cuda")
    inputs = [[normal(g, 400, h, d, dtype="fp32") for h in (4, 2, 2)] for _ in range(2)]
    want = [torch.empty_like(x[0]) for x in inputs]
    for x, o in zip(inputs, want):
        run_attention(*x, None, o, cu)
    torch.cuda.synchronize()
    graphs, outs = [], [torch.empty_like(x[0]) for x in inputs]
    for x, o in zip(inputs, outs):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            run_attention(*x, None, o, cu)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for run in range(4):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for s, graph, x, o in zip(streams, graphs, inputs, outs):
            with torch.cuda.stream(s):
                graph.replay() if run % 2 else run_attention(*x, None, o, cu)
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o, w in zip(outs, want))


@pytest.mark.parametrize("window,softcap", [(0, 0.0), (70, 20.0)])
@pytest.mark.parametrize("d", [64, 72, 128])
@pytest.mark.parametrize("layout", ["packed", "odd", "heads"])
def test_attention_packed_fp32_layouts(layout, d, window, softcap):
    """Scores on both sides of the cap's bend, rows before the first sequence and behind the last."""
    check_attention([129, 0, 200, 1, 66], 6, 3, d, "fp32", window=window, softcap=softcap, qscale=6.0, layout=layout, lead=3, pad=70)


def test_attention_packed_rows_do_not_depend_on_their_neighbours():
    """Twice the same call gives the same bits, and so do two streams at once."""
    import torch

    g = generator(6)
    q, k, v = (normal(g, 600, h, 256) for h in (4, 2, 2))
    cu = torch.tensor([0, 250, 600], dtype=torch.int32, device="cuda")
    outs = [torch.empty_like(q) for _ in range(3)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s, o in zip(streams, outs):
        with torch.cuda.stream(s):
            run_attention(q, k, v, None, o, cu)
    torch.cuda.synchronize()
    run_attention(q, k, v, None, outs[2], cu)
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


@pytest.mark.parametrize("d", [64, 128])
def test_attention_packed_fp32_of_empty_sequences_then_full_ones(d):
    """A call without a row leaves its scratch whole for the next one, which takes the same memory."""
    import torch

    g = generator(29)
    q, k, v = (normal(g, 4000, h, d, dtype="fp32") for h in (4, 2, 2))
    lengths = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([0, 0, 0], [0, 1500, 4000])]
    want, out = torch.empty_like(q), torch.empty_like(q)
    run_attention(q, k, v, None, want, lengths[1])
    untouched = torch.full_like(q, 7.0)
    for _ in range(5):
        run_attention(q.neg(), v, k, None, untouched, lengths[0])
        run_attention(q, k, v, None, out, lengths[1])
        assert torch.equal(out, want)
    assert (untouched == 7).all()


@pytest.mark.parametrize("check", [test_attention_packed_infinities_stay_in_their_sequence, test_attention_packed_scores_of_minus_infinity,
                                   test_attention_packed_a_prompt_gone_nan], ids=lambda f: f.__name__.removeprefix("test_attention_packed_"))
def test_attention_packed_fp32_heads_of_128_that_are_not_finite(check):
    check("fp32", 128)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_attention_packed_neighbours_of_any_size(d, dtype):
    """A sequence keeps its values whatever the rows before and behind it in the same tiles hold."""
    import torch

    g = generator(27)
    bounds = [0, 70, 300, 600]
    q, k, v, gt = (normal(g, 600, h, d, dtype=dtype) for h in (4, 2, 2, 4))
    cu = torch.tensor(bounds, dtype=torch.int32, device="cuda")
    y, tol = attention_64(q[70:300], k[70:300], v[70:300], gt[70:300], [0, 230], 0.0, 0, dtype == "bf16")[0, 230]
    for fill in (0.0, 50.0, -3e38, float("inf"), float("nan")):
        for x in (q, k, v, gt):
            x[:70] = x[300:] = fill
        out = torch.empty_like(q)
        run_attention(q, k, v, gt, out, cu)
        assert ((out[70:300].double() - y).abs() <= tol + U[dtype] * y.abs()).all(), fill


@pytest.mark.parametrize("dtype,d,layout", [("bf16", 64, "split"), ("bf16", 128, "split"), ("bf16", 256, "split"), ("bf16", 72, "odd"),
                                            ("fp32", 64, "split"), ("fp32", 128, "odd"), ("fp32", 256, "split")])
@pytest.mark.parametrize("rows", [1, 3, 40])
def test_attention_packed_some_rows_of_a_tile_are_computed_again(rows, dtype, d, layout):
    """The first rows of a tile come before a value of their own tile that is infinite and masked for them, and
    their scores jump by 100: the block's warps share a few such rows' keys, or take a row each."""
    import torch

    g = generator(30 + rows)
    bounds, width = [0, 50, 1150, 1220], d + (layout == "odd")
    q, k, v, gt, out = (normal(g, 1220, h, width, dtype=dtype)[..., width - d :] for h in (4, 2, 2, 4, 4))
    bad = 7 * 128 + rows
    v[bad] = float("inf")
    q.mul_(0.3), k.mul_(0.3)
    q[:, :, 0], k[:, :, 0] = 16, 0
    k[70, :, 0] = 100 * d**0.5 / 16
    run_attention(q, k, v, gt, out, torch.tensor(bounds, dtype=torch.int32, device="cuda"))
    # weights of 2^-144 beside that key's: 0 times the infinite value is NaN
    assert not out[bad : bounds[2]].isfinite().any()
    v[bad] = 0  # nothing before it sees it
    for a, b in ((0, 50), (50, bad), (1150, 1220)):
        y, tol = attention_64(q[a:b], k[a:b], v[a:b], gt[a:b], [0, b - a], 0.0, 0, dtype == "bf16")[0, b - a]
        assert ((out[a:b].double() - y).abs() <= tol + U[dtype] * y.abs()).all(), (a, b)


# --------------------------------------------------------------------------- token log probabilities


def run_logprobs(hidden, head, targets=None, top=0, softcap=0.0, entropy=True):
    import torch

    n, dim = hidden.shape
    c = targets.shape[1] if targets is not None else 0
    logp = torch.full((n, c), 5.0, device="cuda")
    ent = torch.full((n,), 5.0, device="cuda")
    ids = torch.full((n, top), -7, dtype=torch.int32, device="cuda")
    best = torch.full((n, top), 5.0, device="cuda")
    _lib.check(lib().clef_op_token_logprobs(
        code("bf16" if hidden.element_size() == 2 else "fp32"), hidden.data_ptr(), hidden.stride(0), head.data_ptr(), head.stride(0), n,
        head.shape[0], dim, softcap, targets.data_ptr() if c else None, c, logp.data_ptr() if c else None,
        ent.data_ptr() if entropy else None, top, ids.data_ptr() if top else None, best.data_ptr() if top else None, stream()))
    return logp, ent, ids, best


def grid_operands(g, n, vocab, dim, dtype, std=0.02, slack=0, twins=False):
    """hidden on 1/16, head on 2^-11: every product and sum is exact in FP32."""
    import torch

    ty = torch_type(dtype)
    hidden = (torch.randn(n, dim + slack, generator=g, device="cuda") * 16).round().clamp(-127, 127).div(16).to(ty)[:, :dim]
    head = (torch.randn(vocab, dim + slack, generator=g, device="cuda") * (std * 2048)).round().clamp(-255, 255).div(2048)
    if twins:  # every token has an equal one elsewhere
        head = head[torch.arange(vocab, device="cuda") * 7 % (vocab // 2 + 1)]
    return hidden, head.to(ty)[:, :dim]


def check_logprobs(n, vocab, dim, dtype, top=8, n_targets=2, softcap=0.0, seed=0, **kw):
    import torch

    g = generator(seed + n + vocab + dim)
    hidden, head = grid_operands(g, n, vocab, dim, dtype, **kw)
    targets = torch.randint(0, vocab, (n, n_targets), generator=g, device="cuda", dtype=torch.int32)
    if n_targets > 1:
        targets[:, 1] = targets[:, 0]  # the same token twice
    logp, ent, ids, best = run_logprobs(hidden, head, targets, top, softcap)
    raw = hidden.double() @ head.double().T
    z = softcap * torch.tanh(raw / softcap) if softcap else raw
    lse = torch.logsumexp(z, 1, keepdim=True)
    want = z - lse
    e = 2 * (dim + 8) * U32 * (hidden.double().abs() @ head.double().abs().T).amax(1, keepdim=True)
    r = (vocab / 32 + 64) * U32 + 2.0**-20
    tol = 2 * e + r + 2 * U32 * (z.abs() + lse.abs())
    if n_targets:
        t = targets.long()
        assert ((logp.double() - want.gather(1, t)).abs() <= tol.gather(1, t)).all()
    p = want.exp()
    away = (p * (z - z.amax(1, keepdim=True)).abs()).sum(1)
    assert ((ent.double() + (p * want).sum(1)).abs() <= (4 * e[:, 0] + 2 * r) * (away + 1)).all()
    if top:
        order = torch.sort(raw, dim=1, descending=True, stable=True).indices[:, :top]
        assert torch.equal(ids.long(), order)
        assert ((best.double() - want.gather(1, order)).abs() <= tol.gather(1, order)).all()


LOGPROB_SHAPES = [(1, 50, 8), (1, 5003, 1024), (5, 255, 72), (100, 256, 64), (128, 257, 128), (129, 3001, 256), (300, 70000, 512),
                  (513, 1000, 320), (2, 40000, 3584)]


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("n,vocab,dim", LOGPROB_SHAPES)
def test_token_logprobs_shapes(n, vocab, dim, dtype):
    check_logprobs(n, vocab, dim, dtype)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("n", [3, 200])
@pytest.mark.parametrize("top,n_targets", [(0, 1), (1, 0), (32, 9), (20, 1)])
def test_token_logprobs_outputs(top, n_targets, n, dtype):
    check_logprobs(n, 4000, 64, dtype, top=top, n_targets=n_targets)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("n", [3, 200])
@pytest.mark.parametrize("softcap", [0.0, 30.0, 1.0])
def test_token_logprobs_ties_go_to_the_lowest_id(softcap, n, dtype):
    """Every token has a twin; under a low cap most capped scores are equal as well, and the order is still that of x."""
    check_logprobs(n, 3000, 128, dtype, top=32, softcap=softcap, std=0.1, twins=True)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("n,dim,slack", [(7, 30, 0), (200, 64, 3), (9, 64, 8), (150, 128, 64), (1, 1, 0)])
def test_token_logprobs_row_strides(n, dim, slack, dtype):
    check_logprobs(n, 700, dim, dtype, slack=slack)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_token_logprobs_of_a_sharp_distribution(dtype):
    """Scores of +-100: one token holds nearly all the probability."""
    check_logprobs(140, 3000, 1024, dtype, std=0.1)


@pytest.mark.parametrize("n,dim,dtype", [(5, 1024, "fp32"), (150, 516, "fp32"), (60, 1022, "fp32"), (5, 1024, "bf16"), (300, 2048, "bf16")])
def test_token_logprobs_of_full_mantissas(n, dim, dtype):
    """Values off the grid: every product and sum rounds.  The alternatives' scores have to be the largest up to the tolerance."""
    import torch

    g = generator(n)
    hidden, head = normal(g, n, dim, dtype=dtype), normal(g, 5000, dim, dtype=dtype, std=0.05)
    targets = torch.randint(0, 5000, (n, 3), generator=g, device="cuda", dtype=torch.int32)
    logp, ent, ids, best = run_logprobs(hidden, head, targets, 6)
    z = hidden.double() @ head.double().T
    lse = torch.logsumexp(z, 1, keepdim=True)
    want = z - lse
    e = 2 * (dim + 8) * U32 * (hidden.double().abs() @ head.double().abs().T).amax(1, keepdim=True)
    tol = 2 * e + (5000 / 32 + 64) * U32 + 2.0**-20 + 2 * U32 * (z.abs() + lse.abs())
    assert ((logp.double() - want.gather(1, targets.long())).abs() <= tol.gather(1, targets.long())).all()
    assert ((best.double() - want.gather(1, ids.long())).abs() <= tol.gather(1, ids.long())).all()
    assert ((best.double() - torch.topk(want, 6, 1).values).abs() <= 2 * tol.amax(1, keepdim=True)).all()
    assert (ids.sort(1).values.diff(dim=1) > 0).all()
    p = want.exp()
    assert ((ent.double() + (p * want).sum(1)).abs() <= (4 * e[:, 0] + 2 * (5000 / 32 + 64) * U32 + 2.0**-19) * ((p * (z - z.amax(1, keepdim=True)).abs()).sum(1) + 1)).all()
    print("mean error in units of 2^-24", ((logp.double() - want.gather(1, targets.long())).abs().mean() / U32).item())


def test_token_logprobs_every_token_is_an_alternative():
    check_logprobs(130, 32, 64, "bf16", top=32)
    check_logprobs(3, 5, 64, "fp32", top=5)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("n", [4, 150])
def test_token_logprobs_padded_and_unknown_targets(n, dtype):
    import torch

    hidden, head = grid_operands(generator(9), n, 300, 64, dtype)
    targets = torch.full((n, 3), -1, dtype=torch.int32, device="cuda")
    targets[:, 1], targets[:, 2] = 300, 2**31 - 1
    logp, _, _, _ = run_logprobs(hidden, head, targets)
    assert (logp[:, 0] == 0).all() and logp[:, 1:].isnan().all()


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("n", [4, 150])
def test_token_logprobs_nan_rows_stay_alone(n, dtype):
    import torch

    hidden, head = grid_operands(generator(10), n, 500, 64, dtype)
    targets = torch.zeros(n, 1, dtype=torch.int32, device="cuda")
    clean = run_logprobs(hidden, head, targets, 4)
    hidden[2, 5] = float("nan")
    logp, ent, ids, best = run_logprobs(hidden, head, targets, 4)
    assert logp[2].isnan().all() and ent[2].isnan()
    keep = torch.arange(n, device="cuda") != 2
    for got, want in zip((logp, ent, ids, best), clean):
        assert torch.equal(got[keep], want[keep])


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("n", [3, 60, 200])
@pytest.mark.parametrize("top", [4, 20, 32])
@pytest.mark.parametrize("finite", [(), (5,), (33, 34, 700, 899), tuple(range(0, 900, 37))])
def test_token_logprobs_tokens_of_minus_infinity_are_alternatives_too(finite, top, n, dtype):
    """All tokens but a few score -inf: products of 3e38 and -3e38 that FP32 does not hold.  They follow the finite
    ones as alternatives, the lowest ids first, with log probabilities of -inf; a row without any finite score has no sum."""
    import torch

    hidden, head = grid_operands(generator(13), n, 900, 64, dtype)
    hidden[:, 0] = 2.0**127
    low = torch.ones(900, dtype=torch.bool, device="cuda")
    low[list(finite)] = False
    head[:, 0] = torch.where(low, -(2.0**127), 0.0)
    targets = torch.tensor([[5, 6]], dtype=torch.int32, device="cuda").repeat(n, 1)
    logp, ent, ids, best = run_logprobs(hidden, head, targets, top)
    assert (ent.isfinite() if finite else ent.isnan()).all()
    h, w = hidden.double(), head.double()
    h[:, 0] = 0
    raw = (h @ w.T).masked_fill(low, float("-inf"))
    order = torch.sort(raw, dim=1, descending=True, stable=True).indices[:, :top]
    assert torch.equal(ids.long(), order)
    if finite:
        want = raw - torch.logsumexp(raw, 1, keepdim=True)
        # the finite scores are exact: the relative error of the sum, and a few roundings of the results
        tol = (900 / 32 + 64) * U32 + 2.0**-20 + 8 * U32 * (raw[:, ~low].abs().amax() + 10)
        for got, at in ((logp, targets.long()), (best, order)):
            expected = want.gather(1, at)
            assert torch.equal(got == float("-inf"), expected == float("-inf"))
            assert ((got.double() - expected).abs().nan_to_num(0) <= tol).all()
        p = want.exp()
        z = (raw - raw.amax(1, keepdim=True)).masked_fill(low, 0.0)
        assert ((ent.double() + (p * want.masked_fill(low, 0.0)).sum(1)).abs() <= 4 * tol * ((p * z.abs()).sum(1) + 1)).all()
    else:
        assert logp.isnan().all() and best.isnan().all()


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("softcap", [0.0, 30.0])
@pytest.mark.parametrize("n", [3, 200])
def test_token_logprobs_a_token_of_infinity_comes_first(n, softcap, dtype):
    """Without a cap it leaves no sum; under one it scores the cap, and one of -inf its negative."""
    import torch

    hidden, head = grid_operands(generator(14), n, 900, 64, dtype)
    hidden[:, 0], head[:, 0] = 2.0**127, 0
    head[700, 0], head[3, 0] = 2.0**127, -(2.0**127)
    targets = torch.tensor([[700, 3]], dtype=torch.int32, device="cuda").repeat(n, 1)
    logp, ent, ids, best = run_logprobs(hidden, head, targets, 3, softcap)
    assert (ids[:, 0] == 700).all() and (ids != 3).all()
    if not softcap:
        assert logp.isnan().all() and ent.isnan().all() and best.isnan().all()
        return
    h = hidden.double()
    h[:, 0] = 0
    z = softcap * torch.tanh(h @ head.double().T / softcap)
    z[:, 700], z[:, 3] = softcap, -softcap
    want = torch.log_softmax(z, 1)
    tol = (900 / 32 + 64) * U32 + 2.0**-20 + 8 * U32 * (softcap + 10)
    assert ((logp.double() - want[:, [700, 3]]).abs() <= tol).all() and ((best.double() - torch.topk(want, 3, 1).values).abs() <= tol).all()
    away = (want.exp() * (z - z.amax(1, keepdim=True)).abs()).sum(1)
    assert ((ent.double() + (want.exp() * want).sum(1)).abs() <= 4 * tol * (away + 1)).all()


def test_token_logprobs_captured_and_replayed():
    import torch

    g = generator(11)
    hidden, head = grid_operands(g, 20, 900, 64, "bf16")
    other, _ = grid_operands(g, 20, 900, 64, "bf16")
    targets = torch.randint(0, 900, (20, 2), generator=g, device="cuda", dtype=torch.int32)
    want = [run_logprobs(h, head, targets, 5) for h in (hidden, other)]
    torch.cuda.synchronize()
    graphs, outs, inputs = [], [], []
    for h in (hidden, other):  # two captured calls, each with scratch of its own
        inputs.append(h.clone())
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(run_logprobs(inputs[-1], head, targets, 5))
    for _ in range(2):
        for s, graph in zip([torch.cuda.Stream(), torch.cuda.Stream()], graphs):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for got, w in zip(outs, want):
        assert all(torch.equal(a, b) for a, b in zip(got, w))


def test_token_logprobs_of_two_streams_at_once():
    import torch

    hidden, head = grid_operands(generator(12), 200, 5000, 256, "bf16")
    targets = torch.zeros(200, 1, dtype=torch.int32, device="cuda")
    want = run_logprobs(hidden, head, targets, 3)
    torch.cuda.synchronize()
    got = []
    streams = [torch.cuda.Stream() for _ in range(2)]
    for i in range(6):
        with torch.cuda.stream(streams[i % 2]):
            got.append(run_logprobs(hidden, head, targets, 3))
    torch.cuda.synchronize()
    for x in got:
        assert all(torch.equal(a, b) for a, b in zip(x, want))


# --------------------------------------------------------------------------- together, as a prompt runs through them


def test_a_packed_prompt_from_projection_to_token_scores():
    """Three prompts end to end, one with image tokens: rotary positions in place on
    the packed projection, attention, output projection with the residual, norm and
    token scores, on one stream.  Each stage is held against 64 bits from what the
    stage before left; each prompt alone gives the same scores within its roundings,
    and so do the padded operators for the text prompts."""
    import torch

    hq, hkv, d, dim, vocab, rot = 4, 2, 128, 512, 3000, 64
    lens = [150, 0, 37, 200]
    n, bounds = sum(lens), [0, 150, 150, 187, 387]
    g = generator(21)
    width = 2 * hq * d + 2 * hkv * d
    proj, res = normal(g, n, width), normal(g, n, dim)
    qw, kw, nw = normal(g, d, std=0.1), normal(g, d, std=0.1), normal(g, dim, std=0.1)
    w_o, head = normal(g, dim, hq * d, std=0.05), normal(g, vocab, dim, std=0.05)
    targets = torch.randint(0, vocab, (n, 1), generator=g, device="cuda", dtype=torch.int32)
    sections = (12, 10, 10)
    pos = torch.cat([torch.arange(m, device="cuda") for m in lens]).int().repeat(3, 1)
    patch = torch.arange(64, device="cuda").int()  # rows 200..263 of the last prompt: a frame of 8 x 8 patches
    pos[0, 200:264], pos[1, 200:264], pos[2, 200:264] = 13, 13 + patch // 8, 13 + patch % 8
    cu = torch.tensor(bounds, dtype=torch.int32, device="cuda")

    def views(p):
        t = p.shape[0]
        heads = p[:, : 2 * hq * d].unflatten(1, (hq, 2 * d))
        k0 = 2 * hq * d
        return heads[..., :d], heads[..., d:], p[:, k0 : k0 + hkv * d].view(t, hkv, d), p[:, k0 + hkv * d :].view(t, hkv, d)

    def through(p, r, positions, lengths, tgt):
        t = p.shape[0]
        q, gate, k, v = views(p)
        run_rope(q, k, q, k, positions, sections, True, rot, 1e4, qw, kw)
        att = torch.empty(t, hq, d, dtype=torch.bfloat16, device="cuda")
        run_attention(q, k, v, gate, att, lengths)
        x, y = torch.empty(t, dim, dtype=torch.bfloat16, device="cuda"), torch.empty(t, dim, dtype=torch.bfloat16, device="cuda")
        _lib.check(lib().clef_op_gemm(_lib.DTYPE_BF16, 2, t, dim, hq * d, att.data_ptr(), w_o.data_ptr(), x.data_ptr(), dim, None,
                                      r.data_ptr(), dim, stream()))
        _lib.check(lib().clef_op_rmsnorm(_lib.DTYPE_BF16, x.data_ptr(), nw.data_ptr(), y.data_ptr(), t, dim, 1e-6, stream()))
        return att, x, y, run_logprobs(y, head, tgt, 3)

    before = proj.clone()
    att, x, y, (logp, ent, ids, best) = through(proj, res, pos, cu, targets)
    for view, old, w in zip(views(proj)[::2], views(before)[::2], (qw, kw)):
        assert_rope(view, *rope_64(old, w, pos, sections, True, rot, 1e4), "bf16")
    q, gate, k, v = views(proj)
    for (a, b), (o, tol) in attention_64(q, k, v, gate, bounds, 0.0, 0, True).items():
        assert ((att[a:b].double() - o).abs() <= tol + U["bf16"] * o.abs()).all()
    z = y.double() @ head.double().T
    want = torch.log_softmax(z, 1)
    e = 2 * (dim + 8) * U32 * (y.double().abs() @ head.double().abs().T).amax()
    assert ((logp.double() - want.gather(1, targets.long())).abs() <= 2 * e + 2.0**-16).all()
    assert ((best.double() - torch.topk(want, 3, 1).values).abs() <= 4 * e + 2.0**-16).all()

    # Each prompt alone: the same rotations, then attention sums in another order.  Its
    # rounding moves att by 2^-7 of sum p |v| at most, that moves x by 2^-7 sum |att||w| and a step.
    for a, b in zip(bounds[:-1], bounds[1:]):
        if a == b:
            continue
        one = torch.tensor([0, b - a], dtype=torch.int32, device="cuda")
        part = before[a:b].clone()
        att1, _, _, (logp1, ent1, _, _) = through(part, res[a:b].contiguous(), pos[:, a:b].contiguous(), one, targets[a:b].contiguous())
        assert torch.equal(part, proj[a:b])
        tol = attention_64(q[a:b], k[a:b], v[a:b], gate[a:b], [0, b - a], 0.0, 0, True)[0, b - a][1]
        assert ((att1.double() - att[a:b].double()).abs() <= 2 * tol + 2 * U["bf16"] * att1.double().abs()).all()
        # scores: the norm and the head see vectors that differ by bf16 steps
        assert (logp1 - logp[a:b]).abs().max() <= 0.1 and (ent1 - ent[a:b]).abs().max() <= 0.1


def test_packed_operators_agree_with_the_padded_ones():
    """One text prompt through clef_op_qk_norm_rope + clef_op_attention and through the
    packed operators: the former round the norm, cos, sin and both products (four more
    bf16 half-steps of |y_lo| + |y_hi|), and the attention output before its gate."""
    import torch

    hq, hkv, d, n, rot = 4, 2, 128, 300, 64
    g = generator(22)
    a = normal(g, n, 2 * hq * d + 2 * hkv * d)
    qw, kw = normal(g, d, std=0.1), normal(g, d, std=0.1)
    b = a.clone()
    _lib.check(lib().clef_op_qk_norm_rope(_lib.DTYPE_BF16, a.data_ptr(), 1, n, hq, hkv, d, rot / d, 1e4, qw.data_ptr(), kw.data_ptr(), 1e-6,
                                          stream()))
    q, k = b[:, : 2 * hq * d].view(n, hq, 2 * d)[..., :d], b[:, 2 * hq * d : 2 * hq * d + hkv * d].view(n, hkv, d)
    _, scale = rope_64(q, qw, torch.arange(n, device="cuda")[None], None, False, rot, 1e4)
    run_rope(q, k, q, k, torch.arange(n, device="cuda", dtype=torch.int32)[None], None, False, rot, 1e4, qw, kw)
    off = (a[:, : 2 * hq * d].view(n, hq, 2 * d)[..., :d].double() - q.double()).abs().cpu().numpy()
    assert (off <= 6 * U["bf16"] * scale + 1e-30).all()
    out1, out2 = torch.empty(n, hq * d, dtype=torch.bfloat16, device="cuda"), torch.empty(n, hq, d, dtype=torch.bfloat16, device="cuda")
    _lib.check(lib().clef_op_attention(_lib.DTYPE_BF16, b.data_ptr(), None, out1.data_ptr(), 1, n, hq, hkv, d, 0.0, 0, stream()))
    v, gate = b[:, 2 * hq * d + hkv * d :].view(n, hkv, d), b[:, : 2 * hq * d].view(n, hq, 2 * d)[..., d:]
    cu = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    run_attention(q, k, v, gate, out2, cu)
    tol = attention_64(q, k, v, gate, [0, n], 0.0, 0, True)[0, n][1]
    y = out2.double()
    assert ((out1.view(n, hq, d).double() - y).abs() <= 2 * tol + 4 * U["bf16"] * y.abs() + 1e-30).all()
