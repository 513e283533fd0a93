"""The operators over a paged cache at the edges of what their documentation allows: what follows a call in its stream, calls beside other work, memory and numbers that are
just not allowed. The plain forms and helpers are test_paged.py's."""
import ctypes as C
import subprocess
import sys
import time
from pathlib import Path

import numpy as np
import pytest
import torch

from dooms_b200 import _lib as L
from dooms_b200 import build as B
from dooms_b200 import paged
from test_paged import HALF, Cache, attend, attention_code, bound, chain, check_sample, cuda, fake_cache, fake_rope, prompt_code, sample_code, status, store_code

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


# ---------------------------------------------------------------- one token in f16

@gpu
@pytest.mark.parametrize("heads, head_dim", [((14, 2), 64), ((32, 8), 128), ((16, 1), 64), ((40, 2), 128)])
def test_f16_rows_of_one_token_are_rounded_once(heads, head_dim):
    """Queries, keys and values are f16 numbers, and what happens between them and the result is f32 arithmetic: the bound of f32 rows and half a step of the result (2^-11 of it,
    2^-25 where it is subnormal). A probability of f16 would be half a step of every product, 2^-11 of their sum."""
    (H, K), D = heads, head_dim
    lengths = [1, 2, 17, 63, 64, 65, 300, 2000, 9000]
    cache = Cache(lengths, K, D, 16, seed=5)
    q = np.random.default_rng(6).standard_normal((len(lengths), H, D)).astype(np.float16)
    out = torch.zeros(len(lengths), H, D, dtype=torch.float16, device="cuda")
    cache.cache.attention(cuda(q), torch.arange(len(lengths), dtype=torch.int32, device="cuda"), cuda(np.array(lengths, np.int32)), max(lengths), out, cache.scratch(H))
    assert status() == (L.OK, 0)
    s = 1 / np.sqrt(D)
    for r, n in enumerate(lengths):
        want, mass, reach = attend(q[r].astype(np.float64), *cache.sequence(r, n), s)
        tol = bound(want, mass, reach, D, s, False) + np.abs(want) * HALF + 2.0 ** -25
        assert (np.abs(out[r].cpu().numpy().astype(np.float64) - want) <= tol).all(), n


# ---------------------------------------------------------------- sampling

@gpu
@pytest.mark.parametrize("n", [5, 3000, 151936])
def test_a_min_p_above_one_keeps_the_first_alone(n):
    """None of the tokens reaches more than the largest probability, so the first of them, and it alone, is kept: of equal largest logits the one in front, whatever the other
    filters and the random number. A min-p of 1 keeps all of the largest."""
    g = np.random.default_rng(n)
    x = g.standard_normal((16, n)).astype(np.float32)
    x[:, g.integers(0, n, 4)] = 9.0
    x[3], x[5, n // 2] = 0.25, np.inf
    m = np.array([1.0, np.nextafter(np.float32(1), np.float32(2)), 1.5, 7.0, np.inf, 1.25, 1.0, 2.0] * 2, np.float32)
    check_sample(x, np.array([1.0, 0.7] * 8), np.array([0, 0, 40, 2] * 4), np.array([1.0] * 8 + [0.9] * 8), m, g.random(16))


# ---------------------------------------------------------------- the counters in the scratch

@pytest.fixture(scope="module")
def arrivals():
    source, header, out = HERE / "paged_arrivals.cpp", B.CSRC / "kernels" / "arrivals.h", HERE / "_build" / "libpaged_arrivals.so"
    if not out.exists() or out.stat().st_mtime < max(source.stat().st_mtime, header.stat().st_mtime):
        out.parent.mkdir(exist_ok=True)
        subprocess.run(["g++", "-std=c++20", "-O2", "-Wall", "-shared", "-fPIC", f"-I{header.parent}", str(source), "-o", str(out)], check=True, capture_output=True)
    lib = C.CDLL(str(out))
    lib.arrivals_orders.argtypes = [C.c_int, C.c_ulonglong, C.c_uint, C.c_ulonglong, C.POINTER(C.c_longlong)]
    lib.arrivals_orders.restype = C.c_longlong
    return lib


@pytest.mark.parametrize("start", [0, 1, (1 << 64) - 1, 76 << 20 | 3, 78 << 20 | 1 << 10 | 2, 77 << 16 | 1])
def test_of_those_that_arrive_one_is_the_last_and_leaves_zero(arrivals, start):
    """In every order of their memory operations, whatever the counter held (but the call's own number), and those that failed before: a launch in which a wait ran out leaves
    nothing behind that its replay, whose number is the same, would count on from."""
    for n, orders in ((1, 1), (2, 1), (3, 100)):
        for failed in range(1 << n):
            wrong = C.c_longlong(-1)
            assert arrivals.arrivals_orders(n, 77, failed, start, C.byref(wrong)) >= orders
            assert wrong.value == 0, (n, failed)


@gpu
def test_counters_are_zero_behind_a_call_and_behind_its_replays():
    """Of what the scratch held before, every counter that was used is zero and every other is left as it was: items and units that two blocks share and that many do."""
    H, D = 8, 128
    cache = Cache([9000, 1, 0, 30000, 64], 1, D, 64)
    g = np.random.default_rng(4)
    lengths, seq = cuda(np.array(cache.lengths, np.int32)), torch.arange(5, dtype=torch.int32, device="cuda")
    q, out = cuda(g.standard_normal((5, H, D)), torch.float32), torch.zeros(5, H, D, device="cuda")
    start = cuda(np.array([0, 700, 701, 701, 731, 750], np.int32))
    pq, pout = cuda(g.standard_normal((750, H, D)), torch.float16), torch.zeros(750, H, D, dtype=torch.float16, device="cuda")
    for call in (lambda s, stream: cache.cache.attention(q, seq, lengths, 30000, out, s, stream=stream),
                 lambda s, stream: cache.cache.attention_prompt(pq, seq, start, lengths, pout, s, stream=stream)):
        scratch = cache.scratch(H)
        counters = scratch[:160 * 8].view(torch.int64)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call(scratch, torch.cuda.current_stream().cuda_stream)
        results = []
        for _ in range(3):
            graph.replay()
            results.append((out.clone(), pout.clone()))
            assert ((counters == 0) | (counters == -1)).all() and (counters == 0).any()
        assert all(torch.equal(a, b) for r in results[1:] for a, b in zip(r, results[0]))
    assert status() == (L.OK, 0)


# ---------------------------------------------------------------- numbers beyond 32 bits

def test_the_python_face_refuses_sizes_beyond_32_bits():
    """The C arguments would be their low 32 bits: a row of the first 100 logits, say."""
    keys, ids, q = torch.zeros(4, 16, 2, 64, dtype=torch.float16), torch.zeros(3, dtype=torch.int32), torch.zeros(3, 4, 64)
    cache = paged.PagedCache(keys, keys.clone(), torch.zeros(2, 2, dtype=torch.int32))
    with pytest.raises(L.DoomsError, match="32 bits"):
        paged.sample_rows(torch.empty(1, (1 << 32) + 100, device="meta"), torch.zeros(1), ids[:1])
    with pytest.raises(L.DoomsError, match="32 bits"):
        paged.PagedCache(keys, keys.clone(), torch.empty(1, (1 << 32) + 1, dtype=torch.int32, device="meta"))
    with pytest.raises(L.DoomsError, match="32 bits"):
        cache.rope_store(torch.zeros(3, 512), ids, ids, ids[None], q, 1e4, True, sections=[(1 << 32) + 32])
    with pytest.raises(L.DoomsError, match="32 bits"):
        cache.attention_prompt(q.half(), torch.empty(1 << 32, dtype=torch.int32, device="meta"), ids, ids, q.half(), torch.zeros(1))
    with pytest.raises(L.DoomsError, match="32 bits"):
        cache.scratch_bytes((1 << 32) + 4)


def test_a_longest_length_beyond_32_bits_is_the_longest_there_is(monkeypatch):
    seen = []

    class Library:
        def dooms_cuda_attention_paged(self, *args):
            seen.append(args[5])
            return L.OK
    keys, ids, q = torch.zeros(4, 16, 2, 64, dtype=torch.float16), torch.zeros(3, dtype=torch.int32), torch.zeros(3, 4, 64)
    cache = paged.PagedCache(keys, keys.clone(), torch.zeros(2, 2, dtype=torch.int32))
    monkeypatch.setattr(L, "lib", Library)
    for most in (0, 5, (1 << 31) - 1, 1 << 31, 1 << 32, 1 << 60, -1, -(1 << 33)):
        cache.attention(q, ids, ids, most, q.clone(), torch.zeros(1))
    assert seen == [0, 5] + [(1 << 31) - 1] * 4 + [-1, -1]


# ---------------------------------------------------------------- streams

def test_where_torch_has_no_gpu_the_default_stream_is_meant():
    if not torch.cuda.is_available():
        assert paged._stream(None) == 0
    assert paged._stream(0) == 0 and paged._stream(77) == 77


@gpu
def test_calls_without_a_stream_go_to_torchs_current_one(probes):
    """Under torch.cuda.stream, with tensors that the stream's own work makes (behind half a second of something else) and reads; and captured, as part of the graph."""
    H, K, D, V = 8, 2, 64, 5000
    cache = Cache([100, 40], K, D, 16, fill=0.0)
    scratch, seq = cache.scratch(H), torch.arange(2, dtype=torch.int32, device="cuda")
    lengths, start = cuda(np.array([100, 40], np.int32)), cuda(np.array([0, 5, 12], np.int32))
    made = [torch.randn(2, (H + 2 * K) * D, device="cuda"), torch.randn(12, H, D, device="cuda").half(), torch.randn(2, V, device="cuda")]
    u = torch.rand(2, device="cuda")

    def run(inputs):
        qkv, pq, logits = inputs
        q, out, pout, tokens = torch.zeros(2, H, D, device="cuda"), torch.zeros(2, H, D, device="cuda"), torch.zeros_like(pq), torch.zeros(2, dtype=torch.int32, device="cuda")
        cache.cache.rope_store(qkv, seq, lengths - 1, (lengths - 1)[None], q, base=1e4, neox=True)
        cache.cache.attention(q, seq, lengths, 100, out, scratch)
        cache.cache.attention_prompt(pq, seq, start, lengths, pout, scratch)
        paged.sample_rows(logits, u, tokens)
        return [t.clone() for t in (q, out, pout, tokens)]
    want = run(made)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        inputs = [torch.zeros_like(t) for t in made]
        torch.cuda.synchronize()
        assert probes.probe_hold(1, 500_000_000, stream.cuda_stream) == 0
        for t, m in zip(inputs, made):
            t.copy_(m)
        got = run(inputs)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = run(inputs)
    for t in captured:
        t.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, captured)) and status() == (L.OK, 0)


# ---------------------------------------------------------------- beside other work

@gpu
@pytest.mark.parametrize("heads, head_dim", [((8, 1), 128), ((14, 2), 64)])
def test_calls_that_get_one_sm_beside_a_long_kernel(probes, heads, head_dim):
    """Blocks that share an item or a unit may run one after another: no call needs two of its blocks at once, and what it gives does not depend on it. Cut in two and in many, with
    a value that is not finite and that only later queries see."""
    (H, K), D = heads, head_dim
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    cache = Cache([30000, 1, 2100, 1300], K, D, 64)
    for i, at in ((0, 29950), (2, 2050)):
        cache.host[1].reshape(-1, K, D)[cache.line(i, cache.lengths[i])[at], :, 3] = np.inf
    cache.upload()
    g = np.random.default_rng(11)
    lengths, seq = cuda(np.array(cache.lengths, np.int32)), torch.arange(4, dtype=torch.int32, device="cuda")
    rows = [300, 1, 500, 1300]
    start = cuda(np.concatenate([[0], np.cumsum(rows)]).astype(np.int32))
    q, pq = cuda(g.standard_normal((4, H, D)), torch.float32), cuda(g.standard_normal((sum(rows), H, D)), torch.float16)
    scratch, side, other = cache.scratch(H), torch.cuda.Stream(), torch.cuda.Stream()

    def run():
        out, pout = torch.zeros(4, H, D, device="cuda"), torch.zeros_like(pq)
        torch.cuda.synchronize()
        return out, pout, lambda: (cache.cache.attention(q, seq, lengths, 30000, out, scratch, stream=side.cuda_stream),
                                   cache.cache.attention_prompt(pq, seq, start, lengths, pout, scratch, stream=side.cuda_stream))
    alone, palone, call = run()
    call()
    torch.cuda.synchronize()
    assert palone.isfinite().float().mean() > 0.9 and not palone.isfinite().all()
    out, pout, call = run()
    begun, held, done = (torch.cuda.Event() for _ in range(3))
    with torch.cuda.stream(other):
        begun.record()
        assert probes.probe_hold(sms - 1, 1_500_000_000, other.cuda_stream) == 0
        held.record()
    begun.synchronize()
    time.sleep(0.02)
    call()
    done.record(side)
    done.synchronize()
    assert not held.query()      # (they did not have to wait for the other SMs)
    torch.cuda.synchronize()
    assert status() == (L.OK, 0)
    assert torch.equal(out, alone) and torch.equal(pout.nan_to_num(5.0), palone.nan_to_num(5.0))


# ---------------------------------------------------------------- memory that overlaps

POOL = 10 * 16 * 2 * 64 * 2      # bytes of fake_cache's pools; its page table has 48
BIG = 1 << 32


def apart():
    return fake_cache(keys=BIG, values=2 * BIG, page_table=3 * BIG)


WRITTEN_AND_READ = [
    # the entry, what is written (argument, bytes), and what it may not meet (argument or field of the cache, bytes)
    (lambda **kw: store(**kw), {"q": 2 * 4 * 64 * 4, "keys": POOL, "values": POOL}, {"q": 2 * 4 * 64 * 4, "keys": POOL, "values": POOL, "qkv": 2 * 512 * 4, "page_table": 48, "seq": 8, "at": 8, "pos": 8}),
    (lambda **kw: attend_one(**kw), {"out": 2 * 4 * 64 * 4, "scratch": None}, {"out": 2 * 4 * 64 * 4, "scratch": None, "q": 2 * 4 * 64 * 4, "keys": POOL, "values": POOL, "page_table": 48, "seq": 8, "lengths": 8}),
    (lambda **kw: attend_prompt(**kw), {"out": 5 * 4 * 64 * 2, "scratch": None},
     {"out": 5 * 4 * 64 * 2, "scratch": None, "q": 5 * 4 * 64 * 2, "keys": POOL, "values": POOL, "page_table": 48, "seq": 8, "start": 12, "lengths": 8}),
    (lambda **kw: sample(**kw), {"tokens": 8, "prob": 8}, {"tokens": 8, "prob": 8, "logits": 800, "t": 8, "k": 8, "p": 8, "m": 8, "u": 8}),
]


def split(kw):
    return apart_with({k: v for k, v in kw.items() if k in ("keys", "values", "page_table")}), {k: v for k, v in kw.items() if k not in ("keys", "values", "page_table")}


def apart_with(fields):
    c = apart()
    for k, v in fields.items():
        setattr(c, k, v)
    return c


def store(**kw):
    c, kw = split(kw)
    return store_code(c, fake_rope(), **({"qkv": 4 * BIG, "seq": 5 * BIG, "at": 6 * BIG, "pos": 7 * BIG, "q": 8 * BIG} | kw))


def attend_one(**kw):
    c, kw = split(kw)
    return attention_code(c, **({"q": 4 * BIG, "seq": 5 * BIG, "lengths": 6 * BIG, "out": 7 * BIG, "scratch": 8 * BIG} | kw))


def attend_prompt(**kw):
    c, kw = split(kw)
    return prompt_code(c, **({"q": 4 * BIG, "seq": 5 * BIG, "start": 9 * BIG, "lengths": 6 * BIG, "out": 7 * BIG, "scratch": 8 * BIG} | kw))


def sample(**kw):
    return sample_code(**({"logits": BIG, "t": 2 * BIG, "k": 3 * BIG, "p": 4 * BIG, "m": 5 * BIG, "u": 6 * BIG, "tokens": 7 * BIG, "prob": 8 * BIG} | kw))


def overlaps(code):
    return code == L.INVALID_ARGUMENT and b"overlap" in L.lib().dooms_cuda_last_error()


@pytest.mark.parametrize("entry", range(4))
def test_what_is_written_may_meet_nothing_else(entry):
    """Every pair of a piece that a call writes and any other, by their first and by their last bytes; side by side they are fine (the refusal is another one then)."""
    call, written, others = WRITTEN_AND_READ[entry]
    scratch = L.lib().dooms_cuda_attention_paged_scratch_bytes(4, 2, 64)
    assert not overlaps(call())
    for w, w_bytes in written.items():
        for o, o_bytes in others.items():
            if w == o:
                continue
            w_size, o_size, at = w_bytes or scratch, o_bytes or scratch, 64 * BIG
            # (on boundaries of 16 bytes, which some of them need)
            for there in (at, at + (w_size - 1) // 16 * 16, at - (o_size - 1) // 16 * 16):
                assert overlaps(call(**{w: at, o: there})), (w, o, there - at)
            for there in (at + (w_size + 15) // 16 * 16, at - (o_size + 15) // 16 * 16):
                assert not overlaps(call(**{w: at, o: there})), (w, o, there - at)


def test_what_is_written_between_rows_meets_nothing():
    """Rows that are further apart than they are long leave room between them, which belongs to no row."""
    for tokens, meets in ((BIG + 400, False), (BIG + 396, True), (BIG + 632, False), (BIG + 636, True), (BIG + 640 + 400, False), (BIG - 8, False), (BIG - 4, True)):
        assert overlaps(sample(logits=BIG, stride=160, tokens=tokens)) == meets, tokens - BIG
    for q, meets in ((4 * BIG + 2048, False), (4 * BIG + 2032, True), (4 * BIG + 6144, True), (4 * BIG + 8192, False)):
        assert overlaps(store(qkv=4 * BIG, stride=1024 + 512, q=q)) == meets, q - 4 * BIG


@gpu
def test_tokens_behind_each_row_of_logits():
    """Logits with room behind every row, and outputs in the first rows' room: allowed, and what is there is what separate outputs get."""
    g = np.random.default_rng(3)
    rows, n = 6, 1000
    buffer = torch.zeros(rows, 1024, device="cuda")
    x, u = g.standard_normal((rows, n)).astype(np.float32) * 2, g.random(rows).astype(np.float32)
    buffer[:, :n] = cuda(x)
    tokens, prob = buffer[0, n + 4:n + 4 + rows].view(torch.int32), buffer[2, n + 4:n + 4 + rows]
    paged.sample_rows(buffer[:, :n], cuda(u), tokens, prob)
    assert tokens.tolist() == [chain(x[r], 1.0, 0, 1.0, 0.0, u[r])[0] for r in range(rows)] and (prob > 0).all()
    with pytest.raises(L.DoomsError, match="overlap"):
        paged.sample_rows(buffer[:, :n], cuda(u), buffer[3, n - rows:n].view(torch.int32))


@gpu
def test_pools_scratch_and_queries_of_prompts_are_device_memory():
    """Mapped host memory serves for what the kernels read with plain loads; what tensor copies read, and what blocks count in, is refused there."""
    H, K, D = 4, 2, 64
    cache = Cache([40, 20], K, D, 16)
    scratch, seq, lengths = cache.scratch(H), torch.arange(2, dtype=torch.int32, device="cuda"), cuda(np.array([40, 20], np.int32))
    q, start = torch.randn(2, H, D, device="cuda"), torch.arange(3, dtype=torch.int32, device="cuda")
    out, want = torch.zeros_like(q), torch.zeros_like(q)
    pinned = lambda t: t.cpu().pin_memory()  # noqa: E731
    cache.cache.attention(q, seq, lengths, 40, want, scratch)
    cache.cache.attention(pinned(q), pinned(seq), pinned(lengths), 40, out, scratch)
    torch.cuda.synchronize()
    assert torch.equal(out, want) and status() == (L.OK, 0)
    pools = paged.PagedCache(pinned(cache.keys), pinned(cache.values), cache.d_table)
    pout = torch.zeros_like(q).half()
    for call in (lambda: pools.attention(q, seq, lengths, 40, out, scratch), lambda: cache.cache.attention(q, seq, lengths, 40, out, pinned(scratch)),
                 lambda: pools.attention_prompt(q.half(), seq, start, lengths, pout, scratch), lambda: cache.cache.attention_prompt(pinned(q.half()), seq, start, lengths, pout, scratch),
                 lambda: pools.rope_store(torch.zeros(2, 8 * D, device="cuda"), seq, lengths - 1, lengths[None], torch.zeros_like(q), 1e4, True)):
        with pytest.raises(L.DoomsError, match="device memory"):
            call()
    assert status() == (L.OK, 0)


# ---------------------------------------------------------------- the error word

@gpu
def test_a_bad_page_is_reported_after_a_call_that_could_not_allocate_the_error_word():
    """A process whose first call needs the word under a capture, which forbids its allocation: that call fails, and the word is there for the next one."""
    code = """
import ctypes as C
import torch
from dooms_b200 import _lib as L
from dooms_b200 import paged
w, x, y = torch.zeros(6145 * 4096 // 32 * 18, dtype=torch.uint8, device="cuda"), torch.zeros(4096, device="cuda"), torch.zeros(6145, device="cuda")
keys, values = (torch.randn(8, 16, 2, 64, device="cuda").half() for _ in range(2))
cache = paged.PagedCache(keys, values, torch.full((2, 4), 99, dtype=torch.int32, device="cuda"))
scratch = torch.empty(cache.scratch_bytes(4), dtype=torch.uint8, device="cuda")
seq, lengths = torch.arange(2, dtype=torch.int32, device="cuda"), torch.full((2,), 20, dtype=torch.int32, device="cuda")
q, out = (torch.zeros(2, 4, 64, device="cuda") for _ in range(2))
torch.cuda.synchronize()
stream, graph, first = torch.cuda.Stream(), torch.cuda.CUDAGraph(), None
with torch.cuda.stream(stream):
    graph.capture_begin()
    first = L.lib().dooms_cuda_matvec(L.Q4_0, w.data_ptr(), x.data_ptr(), y.data_ptr(), None, 6145, 4096, 0, stream.cuda_stream)
    try:
        graph.capture_end()
    except RuntimeError as e:
        print("capture:", e)
torch.cuda.synchronize()
print("first:", first)
assert first != L.OK
cache.attention(q, seq, lengths, 64, out, scratch)
flag = C.c_int32()
print("status:", L.lib().dooms_cuda_kernel_status(None, C.byref(flag)), flag.value)
"""
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300, cwd=HERE.parent)
    assert r.returncode == 0 and f"status: {L.INTERNAL} 8" in r.stdout, r.stdout[-2000:] + r.stderr[-2000:]


@gpu
def test_a_flag_takes_no_other_flags_place():
    """A page out of range is noted behind what other kernels have noted, and read and cleared with it."""
    objects = [B.OBJ / (str(src.relative_to(B.CSRC)).replace("/", "_") + ".o") for src in B.sources() if src.parent.name == "kernels"]
    if not all(o.exists() for o in objects):
        B.build()
    source, out = HERE / "paged_entries.cpp", HERE / "_build" / "libpaged_entries.so"
    if not out.exists() or out.stat().st_mtime < max(p.stat().st_mtime for p in [source, *objects]):
        out.parent.mkdir(exist_ok=True)
        subprocess.run([B.nvcc(), *B.NVCC_FLAGS, "-shared", "-x", "cu", str(source), *[f"-Xlinker={o}" for o in objects], "-o", str(out), "-ldl"], check=True, capture_output=True)
    entry = C.CDLL(str(out)).paged_entry_rope_store
    P, I = C.c_void_p, C.c_int
    entry.argtypes = [P, P, P, I, I, I, I, I, I, P, I, I, P, P, P, P, P]
    cache = Cache([40, 40], 2, 64, fill=0.0)
    cache.table[1, 2] = -1
    cache.upload()
    seq, at = cuda(np.array([0, 1], np.int32)), cuda(np.array([3, 39], np.int32))
    qkv, q = torch.randn(2, 8 * 64, device="cuda"), torch.zeros(2, 4, 64, device="cuda")
    error = torch.tensor([2, 0, 16, 0], dtype=torch.int32).pin_memory()
    assert entry(cache.keys.data_ptr(), cache.values.data_ptr(), cache.d_table.data_ptr(), cache.keys.shape[0], 16, 2, cache.table.shape[1], 2, 64, qkv.data_ptr(), 4, 2, seq.data_ptr(),
                 at.data_ptr(), at.data_ptr(), q.data_ptr(), error.data_ptr()) == 0
    torch.cuda.synchronize()
    assert error.tolist() == [2, 8, 16, 0]
