"""Kernels of the packed-prompt operators whose waits run out.

tests/abandoned_waits.cu launches them with tensor maps that deliver fewer bytes
than a wait counts on.  Each wait then ends after its own limit (about two
seconds), and the kernel returns: the context stays usable, and the rows that it
could not compute are NaN."""

from __future__ import annotations

import ctypes
import subprocess
from pathlib import Path

import pytest

from deciax_b200 import build

pytestmark = pytest.mark.gpu
HERE = Path(__file__).resolve().parent
ROWS, VOCAB, DIM, TOP, TOKENS = 20, 512, 64, 5, 100


@pytest.fixture(scope="module")
def abandoned(tmp_path_factory):
    """Every launch of abandoned_waits.cu once, side by side: {name: outputs}."""
    import torch

    so = tmp_path_factory.mktemp("abandoned") / "libabandoned.so"
    subprocess.run([build.nvcc(), *build.ARCH, "-O3", "-std=c++17", "-Xcompiler", "-fPIC", "-shared", str(HERE / "abandoned_waits.cu"), "-o",
                    str(so)], check=True, capture_output=True)
    lib = ctypes.CDLL(str(so))
    vp, i32 = ctypes.c_void_p, ctypes.c_int
    lib.abandoned_logprobs.argtypes = [i32, vp, vp, i32, i32, vp, vp, vp, vp, vp, vp, vp, vp, vp]
    lib.abandoned_attention.argtypes = [i32, i32, vp, vp, vp, vp, vp, i32, vp]
    found, keep = {}, []
    cu = torch.tensor([0, TOKENS], dtype=torch.int32, device="cuda")
    for fp32 in (0, 1):
        ty = torch.float32 if fp32 else torch.bfloat16
        hidden = torch.zeros(60 if fp32 else ROWS, DIM, dtype=torch.bfloat16, device="cuda")
        head, targets = torch.zeros(VOCAB, DIM, dtype=ty, device="cuda"), torch.full((ROWS, 1), 7, dtype=torch.int32, device="cuda")
        # scratch as an earlier call might have left it
        part = torch.tensor([3.0, 2.0, -1.0, 0.0], device="cuda").repeat(ROWS * 2, 1)
        list_x, list_id = torch.zeros(ROWS * 2, TOP, device="cuda"), torch.arange(TOP, dtype=torch.int32, device="cuda").repeat(ROWS * 2, 1)
        outs = [torch.zeros(ROWS, 1, device="cuda"), torch.zeros(ROWS, device="cuda"),
                torch.zeros(ROWS, TOP, dtype=torch.int32, device="cuda"), torch.zeros(ROWS, TOP, device="cuda")]
        keep.append((hidden, head, targets, part, list_x, list_id))
        found["logprobs", fp32] = outs
        qkv = [torch.zeros(3 * TOKENS if fp32 else TOKENS, 64, dtype=torch.bfloat16, device="cuda") for _ in range(3)]
        keep.append(qkv)
        for which in (1, 2):
            found["attention", fp32, which] = torch.full((TOKENS + 28, 64), 3.0, dtype=ty, device="cuda")
    torch.cuda.synchronize()
    for fp32 in (0, 1):
        hidden, head, targets, part, list_x, list_id = keep[2 * fp32]
        s = torch.cuda.Stream()
        keep.append(s)
        assert lib.abandoned_logprobs(fp32, hidden.data_ptr(), head.data_ptr(), DIM, TOP, part.data_ptr(), list_x.data_ptr(),
                                      list_id.data_ptr(), targets.data_ptr(), *(o.data_ptr() for o in found["logprobs", fp32]),
                                      s.cuda_stream) == 0
        for which in (1, 2):
            s = torch.cuda.Stream()
            keep.append(s)
            assert lib.abandoned_attention(fp32, which, *(x.data_ptr() for x in keep[2 * fp32 + 1]),
                                           found["attention", fp32, which].data_ptr(), cu.data_ptr(), TOKENS, s.cuda_stream) == 0
    torch.cuda.synchronize()  # each of them returns
    return found


def test_abandoned_kernels_return_and_the_context_stays_usable(abandoned):
    import torch

    from test_gpu_packed_ops import check_attention, check_logprobs

    check_logprobs(ROWS, VOCAB, DIM, "fp32", top=TOP)
    check_attention([TOKENS], 1, 1, 64, "bf16")
    torch.cuda.synchronize()


@pytest.mark.parametrize("fp32", [0, 1])
def test_abandoned_scores_are_nan(abandoned, fp32):
    """Not what the scratch held, in either of the two runs of columns."""
    logp, entropy, ids, best = abandoned["logprobs", fp32]
    assert logp.isnan().all() and entropy.isnan().all()
    assert (ids == -1).all()


@pytest.mark.parametrize("which", [1, 2])
@pytest.mark.parametrize("fp32", [0, 1])
def test_abandoned_attention_rows_are_nan(abandoned, fp32, which):
    """Whether the keys or the values are missing; rows of no sequence are left as they were."""
    out = abandoned["attention", fp32, which]
    assert out[:TOKENS].isnan().all() and (out[TOKENS:] == 3).all()
