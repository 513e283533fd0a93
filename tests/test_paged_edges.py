"""The operators over a paged cache at the edges of what their documentation allows: what follows a call in its stream, calls beside other work, memory and numbers that are
just not allowed. The plain forms and helpers are test_paged.py's."""
import ctypes as C
import subprocess
from pathlib import Path

import numpy as np
import pytest
import torch

from dooms_b200 import build as B
from dooms_b200 import paged
from test_paged import cuda

gpu = pytest.mark.gpu
HERE = Path(__file__).resolve().parent


@pytest.fixture(scope="module")
def probes():
    source, out = HERE / "paged_probes.cu", HERE / "_build" / "libpaged_probes.so"
    if not out.exists() or out.stat().st_mtime < source.stat().st_mtime:
        out.parent.mkdir(exist_ok=True)
        subprocess.run([B.nvcc(), *B.NVCC_FLAGS, "-shared", str(source), "-o", str(out)], check=True, capture_output=True)
    lib = C.CDLL(str(out))
    lib.probe_copy_at_once.argtypes = [C.c_void_p, C.c_void_p, C.c_int, C.c_void_p]
    lib.probe_hold.argtypes = [C.c_int, C.c_longlong, C.c_void_p]
    return lib


# ---------------------------------------------------------------- what follows a call

@gpu
@pytest.mark.parametrize("rows, n", [(1, 151936), (60, 30000), (200, 30000)])
def test_what_follows_the_sampling_sees_its_tokens(probes, rows, n):
    """A dependent that reads without a wait of its own, as the next kernel in the stream: no launch of a call lets it go before the tokens are there (one launch, and two)."""
    g = np.random.default_rng(rows)
    x, u = cuda(g.standard_normal((rows, n)) * 2, torch.float32), cuda(g.random(rows), torch.float32)
    top_k = cuda(np.where(np.arange(rows) % 3 == 0, 40, 0), torch.int32)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(20):
        tokens, seen = (torch.full((rows,), -9, dtype=torch.int32, device="cuda") for _ in range(2))
        torch.cuda.synchronize()
        paged.sample_rows(x, u, tokens, top_k=top_k, stream=stream.cuda_stream)
        assert probes.probe_copy_at_once(tokens.data_ptr(), seen.data_ptr(), rows, stream.cuda_stream) == 0
        torch.cuda.synchronize()
        assert (tokens >= 0).all() and torch.equal(tokens, seen)
