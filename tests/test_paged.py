"""The operators of a serving step over a paged cache, through their public entries, against plain 64-bit forms: rotary positions with the cache write, attention of
single tokens and of packed prompts, sampling; what they refuse (on the CPU), and a run of them together."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

from dooms_b200 import _lib as L
from dooms_b200 import paged

gpu = pytest.mark.gpu
HALF, SINGLE = 2.0 ** -11, 2.0 ** -24      # half a step, relative


# ---------------------------------------------------------------- refusals (no GPU needed)

def fake_cache(**kw):
    c = L.PagedCache()
    c.struct_size = C.sizeof(L.PagedCache)
    c.keys, c.values, c.page_table = 4096, 8192, 12288
    c.n_pages, c.page_size, c.n_sequences, c.max_pages, c.n_head_kv, c.head_dim = 10, 16, 3, 4, 2, 64
    for k, v in kw.items():
        setattr(c, k, v)
    return c


BAD_CACHES = [({"struct_size": 0}, L.INVALID_ARGUMENT), ({"struct_size": 24}, L.INVALID_ARGUMENT), ({"keys": None}, L.INVALID_ARGUMENT), ({"values": 8200}, L.INVALID_ARGUMENT),
              ({"page_table": None}, L.INVALID_ARGUMENT), ({"page_size": 8}, L.INVALID_ARGUMENT), ({"page_size": 24}, L.INVALID_ARGUMENT), ({"page_size": 131072}, L.INVALID_ARGUMENT),
              ({"page_size": -16}, L.INVALID_ARGUMENT), ({"n_pages": 0}, L.INVALID_ARGUMENT), ({"n_sequences": 0}, L.INVALID_ARGUMENT), ({"max_pages": -1}, L.INVALID_ARGUMENT),
              ({"n_head_kv": 0}, L.INVALID_ARGUMENT), ({"n_head_kv": 3}, L.INVALID_ARGUMENT), ({"head_dim": 96}, L.UNSUPPORTED), ({"head_dim": 256}, L.UNSUPPORTED),
              ({"n_pages": 1 << 27, "page_size": 16}, L.INVALID_ARGUMENT)]


def fake_rope(**kw):
    r = L.Rope(C.sizeof(L.Rope), 10000.0, 1, 1, (C.c_int32 * 4)(32))
    for k, v in kw.items():
        setattr(r, k, (C.c_int32 * 4)(*v) if k == "sections" else v)
    return r


def store_code(cache, rope, qkv=16, stride=512, n_head=4, rows=2, seq=16, at=16, pos=16, dt=L.F32, q=32):
    return L.lib().dooms_cuda_rope_store_paged(C.byref(cache), C.byref(rope), qkv, stride, n_head, rows, seq, at, pos, dt, q, None)


def attention_code(cache, dt=L.F32, q=16, seq=16, lengths=16, most=10, out=32, n_head=4, rows=2, scale=0.0, scratch=16, size=1 << 40):
    return L.lib().dooms_cuda_attention_paged(C.byref(cache), dt, q, seq, lengths, most, out, n_head, rows, scale, scratch, size, None)


def prompt_code(cache, q=16, seq=16, start=16, lengths=16, out=32, n_head=4, prompts=2, rows=5, scale=0.0, scratch=16, size=1 << 40):
    return L.lib().dooms_cuda_attention_prompt_paged(C.byref(cache), q, seq, start, lengths, out, n_head, prompts, rows, scale, scratch, size, None)


def sample_code(logits=16, stride=100, rows=2, n=100, t=None, k=None, p=None, m=None, u=16, tokens=16, prob=None):
    return L.lib().dooms_cuda_sample_rows(logits, stride, rows, n, t, k, p, m, u, tokens, prob, None)


@pytest.mark.parametrize("change, code", BAD_CACHES)
def test_bad_caches_are_refused(change, code):
    assert store_code(fake_cache(**change), fake_rope()) == code
    assert attention_code(fake_cache(**change)) == code
    assert prompt_code(fake_cache(**change)) == code
    assert L.lib().dooms_cuda_last_error()


def test_bad_arguments_are_refused_before_a_launch():
    c = fake_cache()
    for rope in (fake_rope(struct_size=0), fake_rope(base=1.0), fake_rope(base=math.nan), fake_rope(base=math.inf), fake_rope(n_axes=0), fake_rope(n_axes=5),
                 fake_rope(sections=(31,)), fake_rope(n_axes=2, sections=(40, -8)), fake_rope(n_axes=3, sections=(10, 10, 11))):
        assert store_code(c, rope) == L.INVALID_ARGUMENT
    for kw in ({"qkv": None}, {"qkv": 20}, {"stride": 508}, {"stride": 514}, {"n_head": 0}, {"n_head": 3}, {"n_head": 130}, {"rows": -1}, {"seq": None}, {"at": None}, {"pos": None},
               {"q": None}, {"q": 24}):
        assert store_code(c, fake_rope(), **kw) == L.INVALID_ARGUMENT, kw
    assert store_code(c, fake_rope(), dt=L.BF16) == L.UNSUPPORTED
    for kw in ({"q": None}, {"q": 8}, {"seq": None}, {"lengths": None}, {"most": -1}, {"out": None}, {"out": 40}, {"n_head": 5}, {"rows": -2}, {"scale": -1.0}, {"scale": math.nan},
               {"scale": math.inf}, {"scratch": None}, {"scratch": 8}):
        assert attention_code(c, **kw) == L.INVALID_ARGUMENT, kw
    assert attention_code(c, dt=L.Q8_0) == L.UNSUPPORTED
    assert attention_code(c, size=64) == L.RESOURCE_EXHAUSTED
    for kw in ({"q": None}, {"q": 8}, {"q": 32}, {"seq": None}, {"start": None}, {"lengths": None}, {"out": None}, {"n_head": 7}, {"prompts": -1}, {"rows": -1}, {"scale": math.nan},
               {"scratch": None}):
        assert prompt_code(c, **kw) == L.INVALID_ARGUMENT, kw
    assert prompt_code(c, size=64) == L.RESOURCE_EXHAUSTED
    for kw in ({"logits": None}, {"stride": 99}, {"rows": -1}, {"n": 0}, {"u": None}, {"tokens": None}):
        assert sample_code(**kw) == L.INVALID_ARGUMENT, kw
    assert sample_code(n=262145, stride=262145) == L.UNSUPPORTED
    assert L.lib().dooms_cuda_attention_paged_scratch_bytes(4, 3, 64) == 0 and L.lib().dooms_cuda_attention_paged_scratch_bytes(4, 2, 96) == 0
    assert L.lib().dooms_cuda_attention_paged_scratch_bytes(14, 2, 64) > 0


def test_calls_without_rows_are_fine_and_touch_nothing():
    c = fake_cache()
    assert store_code(c, fake_rope(), rows=0, qkv=None) == L.OK
    assert attention_code(c, rows=0, q=None) == L.OK
    assert prompt_code(c, prompts=0) == L.OK and prompt_code(c, rows=0) == L.OK
    assert sample_code(rows=0) == L.OK


def test_the_python_face_refuses_other_tensors():
    keys = torch.zeros(4, 16, 2, 64, dtype=torch.float16)
    table = torch.zeros(2, 2, dtype=torch.int32)
    for k, v, t in ((keys.float(), keys, table), (keys, keys[:3], table), (keys, keys.transpose(1, 2), table), (keys, keys, table.long())):
        with pytest.raises(L.DoomsError):
            paged.PagedCache(k, v, t)
    cache = paged.PagedCache(keys, keys.clone(), table)
    ids, q = torch.zeros(3, dtype=torch.int32), torch.zeros(3, 4, 64)
    for bad in ({"q": q.double()}, {"out": q.half()}, {"sequence": ids[:2]}, {"lengths": ids.long()}):
        kw = {"q": q, "sequence": ids, "lengths": ids, "out": q.clone()} | bad
        with pytest.raises(L.DoomsError):
            cache.attention(kw["q"], kw["sequence"], kw["lengths"], 5, kw["out"], torch.zeros(1 << 20))
    with pytest.raises(L.DoomsError):
        cache.rope_store(torch.zeros(3, 500), ids, ids, ids[None], q, 10000.0, True)
    with pytest.raises(L.DoomsError):
        cache.scratch_bytes(5)
    with pytest.raises(L.DoomsError):
        paged.sample_rows(torch.zeros(3, 8, dtype=torch.float16), torch.zeros(3), ids)


def test_overlapping_and_unaligned_memory_is_refused():
    """Blocks read their inputs while others write: what is written may not overlap what is read. An int32 or float off its boundary would fault in the kernel."""
    c, rope, big = fake_cache(), fake_rope(), 1 << 32
    for q, out, scratch in ((16, 16, big), (16, 32, big), (big + 2 * 4 * 64 * 4 - 16, big, 16), (big, 2 * big, big), (2 * big, big + 4096, big)):
        assert attention_code(c, q=q, out=out, scratch=scratch) == L.INVALID_ARGUMENT, (q, out, scratch)
        assert b"overlap" in L.lib().dooms_cuda_last_error()
    for q, out, scratch in ((16, 16, big), (big + 5 * 4 * 64 * 2 - 16, big, 16), (big, 2 * big, big), (2 * big, big + 4096, big)):
        assert prompt_code(c, q=q, out=out, scratch=scratch) == L.INVALID_ARGUMENT, (q, out, scratch)
        assert b"overlap" in L.lib().dooms_cuda_last_error()
    for qkv, q in ((16, 16), (big, big + (512 + 8 * 64) * 4 - 16), (big + 2 * 4 * 64 * 4 - 16, big)):
        assert store_code(c, rope, qkv=qkv, q=q) == L.INVALID_ARGUMENT, (qkv, q)
        assert b"overlap" in L.lib().dooms_cuda_last_error()
    for code in (store_code(c, rope, q=1 << 20, at=18), attention_code(c, q=big, out=2 * big, seq=17), attention_code(fake_cache(page_table=4097), q=big, out=2 * big),
                 prompt_code(c, q=big, out=2 * big, start=22), sample_code(logits=18), sample_code(tokens=17), sample_code(t=33)):
        assert code == L.INVALID_ARGUMENT and b"4 bytes" in L.lib().dooms_cuda_last_error()


def test_the_python_face_refuses_a_scratch_with_gaps():
    keys = torch.zeros(4, 16, 2, 64, dtype=torch.float16)
    cache, ids, q = paged.PagedCache(keys, keys.clone(), torch.zeros(2, 2, dtype=torch.int32)), torch.zeros(3, dtype=torch.int32), torch.zeros(3, 4, 64)
    for scratch in (torch.zeros(1).expand(1 << 24), torch.zeros(1 << 22, 2)[:, 0]):
        with pytest.raises(L.DoomsError, match="scratch"):
            cache.attention(q, ids, ids, 5, q.clone(), scratch)
        with pytest.raises(L.DoomsError, match="scratch"):
            cache.attention_prompt(q.half(), ids, torch.zeros(4, dtype=torch.int32), ids, q.half(), scratch)


# ---------------------------------------------------------------- plain forms in 64 bits

def status():
    flag = C.c_int32()
    code = L.lib().dooms_cuda_kernel_status(None, C.byref(flag))
    return code, flag.value


def cuda(a, dtype=None):
    return torch.as_tensor(np.array(a, order="C"), dtype=dtype).cuda()


class Cache:
    """A paged cache with every sequence's pages in random order, what is not a position of a sequence filled with NaN, and its contents on the host."""

    def __init__(self, lengths, n_head_kv, head_dim, page=16, seed=0, spare=1, fill=math.nan):
        g = np.random.default_rng(seed)
        self.lengths, self.page, self.g = list(lengths), page, g
        need = [-(-n // page) for n in lengths]
        pool = sum(need) + 2
        order = g.permutation(pool).astype(np.int32)
        self.table = np.full((len(need), max(need + [0]) + spare), -7, dtype=np.int32)
        at = 0
        for i, n in enumerate(need):
            self.table[i, :n] = order[at:at + n]
            at += n
        self.host = [np.full((pool, page, n_head_kv, head_dim), fill, dtype=np.float16) for _ in range(2)]
        for i, n in enumerate(lengths):
            for pool_ in self.host:
                self.rows(pool_, i)[self.line(i, n)] = g.standard_normal((n, n_head_kv, head_dim)).astype(np.float16)
        self.upload()

    def upload(self):
        self.keys, self.values, self.d_table = cuda(self.host[0]), cuda(self.host[1]), cuda(self.table)
        self.cache = paged.PagedCache(self.keys, self.values, self.d_table)

    def rows(self, pool, i):
        return pool.reshape(-1, *pool.shape[2:])

    def line(self, i, n):
        j = np.arange(n)
        return self.table[i, j // self.page].astype(np.int64) * self.page + j % self.page

    def sequence(self, i, n):
        return [self.rows(p, i)[self.line(i, n)].astype(np.float64) for p in self.host]

    def scratch(self, n_head):
        return torch.full((self.cache.scratch_bytes(n_head),), 255, dtype=torch.uint8, device="cuda")      # (its contents do not matter)


def attend(q, k, v, scale):
    """q [heads][d], k / v [n][kv heads][d] in 64 bits: outputs, sum_j p_j |v_j|, and the largest sum_i |q_i k_ji| per head."""
    H, K = q.shape[0], k.shape[1]
    out, mass, reach = np.zeros(q.shape), np.zeros(q.shape), np.zeros((H, 1))
    for h in range(H if len(k) else 0):
        kk, vv = k[:, h // (H // K)], v[:, h // (H // K)]
        s = kk @ q[h] * scale
        p = np.exp(s - s.max())
        p /= p.sum()
        out[h], mass[h], reach[h] = p @ vv, p @ np.abs(vv), (np.abs(kk) @ np.abs(q[h])).max()
    return out, mass, reach


def bound(out, mass, reach, d, scale, half):
    """How far a result may be off: scores from d products and sums in 32 bits (each half a step of at most `reach`, and the query in two f16 parts, 2^-22), which move a
    probability by twice that relative; the exponential and the sums in 32 bits (2^-20); with f16 in and out the probabilities and the result rounded to f16."""
    score = scale * reach * ((d + 16) * SINGLE + 2.0 ** -22)
    return mass * (2.0 * score + 2.0 ** -20 + (HALF if half else 0.0)) + np.abs(out) * (HALF if half else SINGLE)


def check_decode(cache, lengths, H, dtype, scale=0.0, most=None, seed=1, idle=(), q_std=1.0, stream=0, sequences=None):
    g = np.random.default_rng(seed)
    D, n = cache.keys.shape[3], len(lengths)
    q = (g.standard_normal((n, H, D)) * q_std).astype(np.float16 if dtype == torch.float16 else np.float32)
    seq = np.arange(n) if sequences is None else np.array(sequences)
    where = np.where(np.isin(np.arange(n), idle), -1, seq).astype(np.int32)
    out = torch.full((n, H, D), 77.0, dtype=dtype, device="cuda")
    cache.cache.attention(cuda(q), cuda(where), cuda(np.array(lengths, np.int32)), max(lengths) if most is None else most, out, cache.scratch(H), scale=scale, stream=stream)
    assert status() == (L.OK, 0)
    got = out.cpu().numpy().astype(np.float64)
    s = scale or 1 / math.sqrt(D)
    for r in range(n):
        if r in idle:
            assert (got[r] == 77.0).all()
            continue
        want, mass, reach = attend(q[r].astype(np.float64), *cache.sequence(seq[r], lengths[r]), s)
        tol = bound(want, mass, reach, D, s, dtype == torch.float16)
        assert (np.abs(got[r] - want) <= tol).all(), (r, lengths[r], np.abs(got[r] - want).max(), tol.min())


# ---------------------------------------------------------------- rotary positions and the cache write

def turned(x, positions, sections, base, neox):
    """x [n][heads][d], positions [axes][n] in 64 bits."""
    d = x.shape[2]
    axis = np.repeat(np.arange(len(sections)), sections)
    angle = positions[axis].T.astype(np.float64) * base ** (-2.0 * np.arange(d // 2) / d)
    c, s = np.cos(angle)[:, None], np.sin(angle)[:, None]
    y = np.empty_like(x)
    one, two = (slice(0, d // 2), slice(d // 2, d)) if neox else (slice(0, d, 2), slice(1, d, 2))
    y[..., one], y[..., two] = x[..., one] * c - x[..., two] * s, x[..., one] * s + x[..., two] * c
    return y


@gpu
@pytest.mark.parametrize("heads, head_dim, neox, dtype, sections, page, n", [
    ((14, 2), 64, True, torch.float32, [32], 16, 1), ((14, 2), 64, False, torch.float16, [8, 12, 12], 32, 37), ((32, 8), 128, False, torch.float32, [64], 16, 5),
    ((40, 8), 128, True, torch.float16, [16, 24, 24], 64, 333), ((3, 3), 128, True, torch.float32, [0, 60, 4, 0], 16, 64), ((64, 1), 64, True, torch.float16, [1, 31], 256, 1500)])
def test_rope_store(heads, head_dim, neox, dtype, sections, page, n):
    H, K = heads
    g = np.random.default_rng(n)
    per = np.diff(np.concatenate([[0], np.sort(g.integers(0, n + 1, 3)), [n]]))          # rows of four sequences (some may have none)
    first = g.integers(0, 100, 4)
    cache = Cache([int(a + b) for a, b in zip(first, per)], K, head_dim, page, seed=n, fill=0.0)
    width = (H + 2 * K) * head_dim
    qkv = torch.full((n, width + 12), math.nan, device="cuda")                            # rows further apart than they are long
    x = g.standard_normal((n, width)).astype(np.float32)
    qkv[:, :width] = cuda(x)
    seq = np.repeat(np.arange(4), per).astype(np.int32)
    at = np.concatenate([np.arange(f, f + p) for f, p in zip(first, per)]).astype(np.int32)
    idle = g.random(n) < 0.1
    positions = g.integers(0, 200000, (len(sections), n)).astype(np.int32)
    q = torch.full((n, H, head_dim), 55.0, dtype=dtype, device="cuda")
    cache.cache.rope_store(qkv[:, :width], cuda(np.where(idle, -3, seq).astype(np.int32)), cuda(at), cuda(positions), q, base=1e6, neox=neox, sections=sections)
    assert status() == (L.OK, 0)
    x64 = x.reshape(n, H + 2 * K, head_dim).astype(np.float64)
    y = np.concatenate([turned(x64[:, :H + K], positions, sections, 1e6, neox), x64[:, H + K:]], axis=1)
    # sine and cosine rounded, two products and a sum rounded: 5 half steps of |u| + |w|, then the stored type's own
    size = np.abs(x64).max()
    got = q.cpu().numpy().astype(np.float64)
    off = np.abs(got - y[:, :H])[~idle]
    assert (off <= 2 * size * 5 * SINGLE + (HALF if dtype == torch.float16 else 0) * np.abs(y[:, :H][~idle])).all()
    assert (got[idle] == 55.0).all()
    for pool, host, part in ((cache.keys, cache.host[0], y[:, H:H + K]), (cache.values, cache.host[1], y[:, H + K:])):
        want = cache.rows(host, 0).astype(np.float64)
        for r in range(n):
            if not idle[r]:
                want[cache.table[seq[r], at[r] // page].astype(np.int64) * page + at[r] % page] = part[r]
        got = cache.rows(pool.cpu().numpy(), 0).astype(np.float64)
        assert (np.abs(got - want) <= np.abs(want) * HALF + 2 * size * 5 * SINGLE + 2.0 ** -25).all()
        same = ~np.isin(np.arange(len(got)), [cache.table[seq[r], at[r] // page] * page + at[r] % page for r in range(n) if not idle[r]])
        assert np.array_equal(got[same], cache.rows(host, 0).astype(np.float64)[same])      # no other position is touched


@gpu
def test_one_axis_is_what_equal_axes_give():
    g = np.random.default_rng(4)
    qkv, seq, at = cuda(g.standard_normal((9, 6 * 64)), torch.float32), cuda(np.zeros(9, np.int32)), cuda(np.arange(9, dtype=np.int32))
    out = []
    for sections in ([32], [10, 11, 11], [8, 8, 8, 8]):
        cache = Cache([9], 1, 64, fill=0.0)
        q = torch.empty(9, 4, 64, device="cuda")
        cache.cache.rope_store(qkv, seq, at, cuda(np.repeat(np.arange(9)[None] * 1000, len(sections), 0).astype(np.int32)), q, base=1e4, neox=True, sections=sections)
        out.append((q, cache.keys, cache.values))
    assert all(torch.equal(a, b) for o in out[1:] for a, b in zip(out[0], o))


@gpu
def test_bad_entries_are_reported_and_not_followed():
    g = np.random.default_rng(3)
    for what in ("sequence", "at", "negative at", "page", "negative page"):
        cache = Cache([40, 40], 2, 64, fill=0.0)
        seq, at = np.array([0, 1, 1], np.int32), np.array([3, 39, 20], np.int32)
        if what == "sequence":
            seq[1] = 2
        elif what == "at":
            at[1] = 16 * cache.table.shape[1]
        elif what == "negative at":
            at[1] = -1
        else:
            cache.table[1, 2] = cache.keys.shape[0] if what == "page" else -1
            cache.upload()
        x = g.standard_normal((3, 8 * 64)).astype(np.float32)
        q = torch.full((3, 4, 64), 9.0, device="cuda")
        cache.cache.rope_store(cuda(x), cuda(seq), cuda(at), cuda(np.zeros((1, 3), np.int32)), q, base=1e4, neox=True)
        assert status() == (L.INTERNAL, 8), what
        assert status() == (L.OK, 0)
        want = [cache.rows(h, 0).copy() for h in cache.host]
        for r in (0, 2):
            for w, a in zip(want, (4, 6)):
                w[cache.table[seq[r], at[r] // 16] * 16 + at[r] % 16] = x[r].reshape(8, 64)[a:a + 2].astype(np.float16)
        assert np.array_equal(cache.rows(cache.keys.cpu().numpy(), 0), want[0]) and np.array_equal(cache.rows(cache.values.cpu().numpy(), 0), want[1])
        assert (q[1] == 9.0).all() and torch.equal(q[0].flatten(), cuda(x[0, :256]))


# ---------------------------------------------------------------- one new token

EDGES = [0, 1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 128, 129, 255, 257, 300, 513]


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("heads, head_dim, page", [((14, 2), 64, 16), ((32, 8), 128, 64), ((40, 8), 128, 16), ((3, 3), 64, 128), ((16, 1), 128, 32), ((18, 2), 64, 16), ((17, 1), 128, 256),
                                                   ((64, 1), 64, 16)])
def test_attention_of_one_token(heads, head_dim, page, dtype):
    H, K = heads
    check_decode(Cache(EDGES, K, head_dim, page, seed=H), EDGES, H, dtype, idle=(4, 11))


@gpu
@pytest.mark.parametrize("lengths", [[1], [7], [2311], [100000], [5000, 1, 0, 4999], [64] * 300, [0, 0, 0]])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_attention_of_one_token_few_and_many_rows(lengths, dtype):
    check_decode(Cache(lengths, 2, 64, 16, seed=len(lengths)), lengths, 6, dtype, most=131072)


@gpu
def test_attention_of_one_token_scales_and_large_queries():
    cache = Cache([100, 37], 2, 128, 32)
    check_decode(cache, [100, 37], 8, torch.float32, scale=0.5)
    check_decode(cache, [100, 37], 8, torch.float32, scale=1e-6, q_std=3e5)          # beyond f16's largest value
    check_decode(cache, [100, 37], 8, torch.float32, q_std=1e-6)
    check_decode(cache, [33, 1, 100], 8, torch.float32, sequences=[0, 1, 0])          # a shared sequence, seen to different lengths


@gpu
def test_attention_of_one_token_infinite_and_tiny_scores():
    cache = Cache([50], 1, 64, 16)
    cache.host[0][cache.table[0, 1]] *= np.float16(100)                               # scores of some hundred: one key takes all
    cache.upload()
    check_decode(cache, [50], 4, torch.float16, q_std=4.0)
    for row in (3, 20):
        cache.host[1].reshape(-1, 64)[cache.line(0, 50)[row]] = np.inf                # an infinity among what is seen comes out, one past the length does not
        cache.upload()
        q = torch.randn(1, 4, 64, device="cuda") * 0.01
        out = torch.empty_like(q)
        one = torch.zeros(1, dtype=torch.int32, device="cuda")
        cache.cache.attention(q, one, one + 3, 50, out, cache.scratch(4))
        assert out.isfinite().all()
        cache.cache.attention(q, one, one + 50, 50, out, cache.scratch(4))
        assert (out == math.inf).all()


@gpu
def test_attention_of_one_token_bad_entries():
    for what in ("sequence", "length", "negative", "page"):
        cache = Cache([40, 40, 40], 2, 64, fill=0.0)
        lengths, seq = np.array([40, 40, 40], np.int32), np.arange(3, dtype=np.int32)
        if what == "sequence":
            seq[1] = 3
        elif what == "length":
            lengths[1] = 41
        elif what == "negative":
            lengths[1] = -2
        else:
            cache.table[1, 1] = 10 ** 6
            cache.upload()
        q = np.random.default_rng(5).standard_normal((3, 6, 64)).astype(np.float32)
        out = torch.zeros(3, 6, 64, device="cuda")
        cache.cache.attention(cuda(q), cuda(seq), cuda(lengths), 40, out, cache.scratch(6))
        assert status() == (L.INTERNAL, 8), what
        for r in (0, 2):
            want, mass, reach = attend(q[r].astype(np.float64), *cache.sequence(r, 40), 0.125)
            assert (np.abs(out[r].cpu().numpy() - want) <= bound(want, mass, reach, 64, 0.125, False)).all()


@gpu
def test_attention_captured_replayed_and_on_another_stream():
    """One graph over the longest length, replayed for other lengths; a scratch that two graphs share; a stream of its own."""
    H, D = 14, 64
    cache = Cache([3000, 900, 40], 2, D)
    g = np.random.default_rng(6)
    q = cuda(g.standard_normal((3, H, D)), torch.float32)
    lengths, seq, out = torch.zeros(3, dtype=torch.int32, device="cuda"), torch.arange(3, dtype=torch.int32, device="cuda"), torch.zeros(3, H, D, device="cuda")
    q16, start, out16 = q.half(), cuda(np.arange(4, dtype=np.int32)), torch.zeros(3, H, D, dtype=torch.float16, device="cuda")
    scratch, side = cache.scratch(H), torch.cuda.Stream()
    graphs = []
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                cache.cache.attention(q, seq, lengths, 3000, out, scratch, stream=side.cuda_stream)
                cache.cache.attention_prompt(q16, seq, start, lengths, out16, scratch, stream=side.cuda_stream)
            graphs.append(graph)
        for i, now in enumerate(([3000, 900, 40], [1, 0, 17], [2999, 16, 33])):
            lengths.copy_(torch.tensor(now, dtype=torch.int32))
            out.fill_(5.0)
            out16.fill_(5.0)
            graphs[i % 2].replay()
            side.synchronize()
            for r, n in enumerate(now):
                for half, have, query in ((False, out, q), (True, out16, q16)):
                    want, mass, reach = attend(query[r].cpu().numpy().astype(np.float64), *cache.sequence(r, n), 0.125)
                    assert (np.abs(have[r].cpu().numpy() - want) <= bound(want, mass, reach, D, 0.125, half)).all()
    assert status() == (L.OK, 0)


@gpu
def test_a_process_whose_first_calls_are_captured():
    """What the first call sets up is set up under a capture too: in a process of its own, all four calls in a graph, then replayed."""
    import subprocess
    import sys
    from pathlib import Path
    code = """
import torch
from dooms_b200 import paged
keys, values = (torch.randn(8, 16, 2, 64, device="cuda").half() for _ in range(2))
cache = paged.PagedCache(keys, values, torch.arange(8, dtype=torch.int32, device="cuda").view(2, 4))
scratch = torch.empty(cache.scratch_bytes(4), dtype=torch.uint8, device="cuda")
seq, at, start = torch.arange(2, dtype=torch.int32, device="cuda"), torch.full((2,), 20, dtype=torch.int32, device="cuda"), torch.arange(3, dtype=torch.int32, device="cuda")
qkv, q, out, q16, out16 = torch.randn(2, 512, device="cuda"), *(torch.zeros(2, 4, 64, device="cuda") for _ in range(2)), *(torch.zeros(2, 4, 64, device="cuda").half() for _ in range(2))
logits, u, tokens = torch.randn(2, 1000, device="cuda"), torch.rand(2, device="cuda"), torch.full((2,), -1, dtype=torch.int32, device="cuda")
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    s = torch.cuda.current_stream().cuda_stream
    cache.rope_store(qkv, seq, at, at[None], q, base=1e4, neox=True, stream=s)
    cache.attention(q, seq, at + 1, 64, out, scratch, stream=s)
    cache.attention_prompt(q16, seq, start, at + 1, out16, scratch, stream=s)
    paged.sample_rows(logits, u, tokens, stream=s)
graph.replay()
torch.cuda.synchronize()
assert (q != 0).any() and (out != 0).all() and (out16 != 0).all() and (tokens >= 0).all()
print("captured")
"""
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300, cwd=Path(__file__).resolve().parent.parent)
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr[-2000:]


# ---------------------------------------------------------------- packed prompts

def check_prompt(cache, new, lengths, H, gaps=(0, 0), scale=0.0, idle=(), every=1, seed=2, sequences=None):
    """Prompt i is the last new[i] of lengths[i] positions; rows in front of the first and behind the last prompt belong to nobody."""
    g = np.random.default_rng(seed)
    D = cache.keys.shape[3]
    start = gaps[0] + np.concatenate([[0], np.cumsum(new)])
    rows = int(start[-1]) + gaps[1]
    q = g.standard_normal((rows, H, D)).astype(np.float16)
    seq = np.arange(len(new)) if sequences is None else np.array(sequences)
    where = np.where(np.isin(np.arange(len(new)), idle), -1, seq).astype(np.int32)
    out = torch.full((rows, H, D), 77.0, dtype=torch.float16, device="cuda")
    cache.cache.attention_prompt(cuda(q), cuda(where), cuda(start.astype(np.int32)), cuda(np.array(lengths, np.int32)), out, cache.scratch(H), scale=scale)
    assert status() == (L.OK, 0)
    got = out.cpu().numpy().astype(np.float64)
    s = scale or 1 / math.sqrt(D)
    assert (got[:start[0]] == 77.0).all() and (got[start[-1]:] == 77.0).all()
    for i, n in enumerate(new):
        if i in idle:
            assert (got[start[i]:start[i + 1]] == 77.0).all()
            continue
        k, v = cache.sequence(seq[i], lengths[i])
        for j in sorted(set(range(0, n, every)) | set(range(max(0, n - 3), n))):
            seen = max(0, lengths[i] - n + j + 1)
            want, mass, reach = attend(q[start[i] + j].astype(np.float64), k[:seen], v[:seen], s)
            tol = bound(want, mass, reach, D, s, True)
            off = np.abs(got[start[i] + j] - want)
            assert (off <= tol).all(), (i, j, seen, off.max(), tol.min())


@gpu
@pytest.mark.parametrize("heads, head_dim, page", [((14, 2), 64, 16), ((32, 8), 128, 32), ((40, 8), 128, 128), ((3, 3), 64, 256), ((16, 1), 128, 16), ((18, 2), 64, 64), ((64, 1), 128, 16),
                                                   ((33, 1), 64, 32)])
def test_attention_of_packed_prompts(heads, head_dim, page):
    H, K = heads
    new = [1, 0, 2, 17, 64, 65, 130, 5, 1, 33]
    cached = [0, 9, 0, 3, 0, 64, 127, 300, 513, 1000]
    lengths = [a + b for a, b in zip(new, cached)]
    check_prompt(Cache(lengths, K, head_dim, page, seed=H), new, lengths, H, gaps=(3, 7), idle=(4,), every=5)


@gpu
@pytest.mark.parametrize("new, cached", [([1], [0]), ([1], [40000]), ([3], [20001]), ([700], [0]), ([257], [1023]), ([1] * 200, [5] * 200), ([0, 0, 0], [4, 0, 9]), ([30, 0, 1000, 0], [0, 5, 0, 0])])
def test_attention_of_few_and_many_prompts(new, cached):
    lengths = [a + b for a, b in zip(new, cached)]
    check_prompt(Cache(lengths, 2, 64, 16, seed=len(new)), new, lengths, 4, gaps=(0, 1), every=41)


@gpu
@pytest.mark.parametrize("longest", [1024, 1025])
@pytest.mark.parametrize("heads, head_dim", [((8, 2), 64), ((5, 1), 128)])
def test_attention_of_prompts_whole_units_and_cut_ones(heads, head_dim, longest):
    """Batches whose longest unit has eight tiles of keys, and nine; more units than there are blocks, and fewer."""
    H, K = heads
    for copies in (1, 12):
        new = [longest, 130, 1, 64, 0, 200] * copies
        lengths = [longest, 900, 700, 64, 5, 333] * copies
        check_prompt(Cache(lengths, K, head_dim, 32, seed=copies), new, lengths, H, gaps=(1, 2), every=97)


@gpu
def test_attention_of_prompts_longer_than_their_lengths():
    """The rows in front of the first position see nothing: zeros."""
    check_prompt(Cache([5, 0, 140], 2, 128, 16), [9, 4, 150], [5, 0, 140], 8)


@gpu
def test_attention_of_prompts_scales_and_shared_sequences():
    cache = Cache([200, 64], 2, 64, 64)
    check_prompt(cache, [50, 20], [200, 64], 6, scale=0.5)
    check_prompt(cache, [10, 10, 5], [100, 64, 200], 6, sequences=[0, 1, 0])


@gpu
@pytest.mark.parametrize("heads, head_dim, page", [((14, 2), 64, 16), ((8, 2), 128, 64), ((3, 3), 64, 256)])
@pytest.mark.parametrize("what", [math.nan, math.inf, -math.inf])
def test_attention_of_prompts_values_that_are_not_finite(heads, head_dim, page, what):
    """Values that are not finite are no concern of the rows in front of their position, in whole units or cut ones, in one column or all of them. A row that sees such a value
    has it in its output: NaN, or the infinity where its probability is far above zero."""
    H, K = heads
    new, cached = [90, 300, 33, 1], [30, 20000, 0, 128]
    lengths = [a + b for a, b in zip(new, cached)]
    for at, column in ((40, 5), (1, None), (85, head_dim - 1)):
        cache = Cache(lengths, K, head_dim, page, seed=H)
        spoilt = [lengths[i] - n + min(at, n - 1) for i, n in enumerate(new)]      # the position of each sequence
        for i, j in enumerate(spoilt):
            cache.rows(cache.host[1], i)[cache.line(i, lengths[i])[j], :, slice(None) if column is None else column] = what
        cache.upload()
        g = np.random.default_rng(at)
        start = np.concatenate([[0], np.cumsum(new)])
        q = g.standard_normal((start[-1], H, head_dim)).astype(np.float16)
        out = torch.full(q.shape, 77.0, dtype=torch.float16, device="cuda")
        cache.cache.attention_prompt(cuda(q), cuda(np.arange(4, dtype=np.int32)), cuda(start.astype(np.int32)), cuda(np.array(lengths, np.int32)), out, cache.scratch(H))
        assert status() == (L.OK, 0)
        got = out.cpu().numpy().astype(np.float64)
        s = 1 / math.sqrt(head_dim)
        for i, n in enumerate(new):
            k, v = cache.sequence(i, lengths[i])
            sane = np.where(np.isfinite(v), v, 0.0)
            for j in sorted({0, min(1, n - 1), max(0, min(at, n - 1) - 1), min(at, n - 1), n - 1}):
                seen = lengths[i] - n + j + 1
                want, mass, reach = attend(q[start[i] + j].astype(np.float64), k[:seen], sane[:seen], s)
                tol = bound(want, mass, reach, head_dim, s, True)
                r = got[start[i] + j]
                if seen > spoilt[i]:
                    hit = np.s_[:, :] if column is None else np.s_[:, column]
                    assert (np.isnan(r[hit]) if math.isnan(what) else ~np.isfinite(r[hit]) if cached[i] > 1000 else r[hit] == what).all(), (i, j)
                    want[hit] = r[hit] = 0.0
                assert (np.abs(r - want) <= tol).all(), (i, j, seen)


@gpu
@pytest.mark.parametrize("heads, head_dim, batch", [((3, 3), 64, 30), ((2, 2), 128, 44), ((14, 2), 64, 40)])
def test_attention_of_prompts_cut_in_two_around_a_value_that_is_not_finite(heads, head_dim, batch):
    """So many units that a cut one is shared by two blocks, at every tile in turn; the position that is not finite is now in the part of the one, now of the other."""
    H, K = heads
    n, at, s = 300, 130, 1 / math.sqrt(head_dim)
    lengths = [900 + 17 * i + n for i in range(batch)]
    cache = Cache(lengths, K, head_dim, 64, seed=H)
    for i in range(batch):
        cache.rows(cache.host[1], i)[cache.line(i, lengths[i])[lengths[i] - n + at], :, i % head_dim] = (math.nan, math.inf)[i % 2]
    cache.upload()
    q = np.random.default_rng(4).standard_normal((batch * n, H, head_dim)).astype(np.float16)
    start = np.arange(batch + 1, dtype=np.int32) * n
    out = torch.full(q.shape, 77.0, dtype=torch.float16, device="cuda")
    cache.cache.attention_prompt(cuda(q), cuda(np.arange(batch, dtype=np.int32)), cuda(start), cuda(np.array(lengths, np.int32)), out, cache.scratch(H))
    assert status() == (L.OK, 0)
    got = out.cpu().numpy().astype(np.float64).reshape(batch, n, H, head_dim)
    assert np.isfinite(got[:, :at]).all()
    for i in range(batch):
        k, v = cache.sequence(i, lengths[i])
        v = np.where(np.isfinite(v), v, 0.0)
        for j in (0, 70, 120, at - 1, at, 299):
            r = got[i, j].copy()
            want, mass, reach = attend(q[i * n + j].astype(np.float64), k[:lengths[i] - n + j + 1], v[:lengths[i] - n + j + 1], s)
            if j >= at:
                assert not np.isfinite(r[:, i % head_dim]).any()
                want[:, i % head_dim] = r[:, i % head_dim] = 0.0
            assert (np.abs(r - want) <= bound(want, mass, reach, head_dim, s, True)).all(), (i, j)


@gpu
def test_a_long_prompt_in_one_call_is_its_pieces():
    """2100 positions at once, and as pieces behind what is cached: the same rows up to the roundings of two results."""
    H, D, n = 10, 128, 2100
    cache = Cache([n], 2, D, 64)
    q = torch.randn(n, H, D, device="cuda").half()
    zero = torch.zeros(1, dtype=torch.int32, device="cuda")
    whole, parts = torch.empty_like(q), torch.empty_like(q)
    cache.cache.attention_prompt(q, zero, cuda(np.array([0, n], np.int32)), zero + n, whole, cache.scratch(H))
    for a, b in ((0, 1), (1, 700), (700, 1212), (1212, 2099), (2099, 2100)):
        cache.cache.attention_prompt(q[a:b], zero, cuda(np.array([0, b - a], np.int32)), zero + b, parts[a:b], cache.scratch(H))
    assert status() == (L.OK, 0)
    k, v = (torch.from_numpy(x).cuda() for x in cache.sequence(0, n))
    for h in (0, 7):
        s = q[:, h].double() @ k[:, h // 5].T / math.sqrt(D)
        p = torch.softmax(s.masked_fill(torch.ones_like(s, dtype=torch.bool).triu(1), -math.inf), -1)
        want, mass = p @ v[:, h // 5], p @ v[:, h // 5].abs()
        reach = (q[:, h].double().abs() @ k[:, h // 5].abs().T).amax(1, keepdim=True)
        tol = torch.from_numpy(bound(want.cpu().numpy(), mass.cpu().numpy(), reach.cpu().numpy(), D, 1 / math.sqrt(D), True)).cuda()
        assert ((whole[:, h] - want).abs() <= tol).all() and ((parts[:, h] - want).abs() <= tol).all()


@gpu
def test_attention_of_prompts_bad_entries():
    for what in ("sequence", "length", "negative", "page", "start", "descending"):
        cache = Cache([40, 40, 40], 2, 64, fill=0.0)
        lengths, seq, start = np.array([40, 40, 40], np.int32), np.arange(3, dtype=np.int32), np.array([0, 10, 20, 30], np.int32)
        ok = (0, 2)
        if what == "sequence":
            seq[1] = 3
        elif what == "length":
            lengths[1] = 16 * cache.table.shape[1] + 1
        elif what == "negative":
            lengths[1] = -2
        elif what == "page":
            cache.table[1, 1] = -5
            cache.upload()
        elif what == "start":
            start[3], ok = 31, (0, 1)
        else:
            start[2], ok = 5, (0,)
        q = np.random.default_rng(5).standard_normal((30, 6, 64)).astype(np.float16)
        out = torch.zeros(30, 6, 64, dtype=torch.float16, device="cuda")
        cache.cache.attention_prompt(cuda(q), cuda(seq), cuda(start), cuda(lengths), out, cache.scratch(6))
        assert status() == (L.INTERNAL, 8), what
        for i in ok:
            k, v = cache.sequence(i, 40)
            for j in range(5 if what == "descending" else 10):
                want, mass, reach = attend(q[10 * i + j].astype(np.float64), k[:31 + j], v[:31 + j], 0.125)
                assert (np.abs(out[10 * i + j].cpu().numpy() - want) <= bound(want, mass, reach, 64, 0.125, True)).all(), what


# ---------------------------------------------------------------- sampling

def chain(x, t, k, p, m, u):
    """(token, probability) of one row in 64 bits, from the definition."""
    x = np.asarray(x, dtype=np.float32).astype(np.float64)
    there = [i for i in range(len(x)) if x[i] == x[i]]
    if not there or max(x[i] for i in there) == -math.inf:
        return (there[0] if there else 0), 0.0
    order = sorted((i for i in there if x[i] > -math.inf), key=lambda i: (-x[i], i))
    if not t > 0:
        return order[0], 1.0
    if k > 0:
        order = order[:k]
    g = np.array([0.0 if x[i] == x[order[0]] else x[order[0]] - x[i] for i in order])      # (an infinity is no distance from itself)
    mass = np.exp(-g)
    keep = len(order)
    if p < 1:
        ahead = np.concatenate([[0.0], np.cumsum(mass)[:-1]])
        keep = max(1, int((ahead < float(np.float32(p)) * mass.sum()).sum()))
    if m > 0:
        keep = max(1, min(keep, int((mass >= float(np.float32(m))).sum())))
    w = np.exp(-g[:keep] / float(np.float32(t)))
    at = int((np.cumsum(w) <= float(np.float32(u)) * w.sum()).sum())
    at = min(at, int((w > 0).sum()) - 1)
    return order[at], w[at] / w.sum()


def check_sample(x, t, k, p, m, u, stride=0):
    x = np.asarray(x, dtype=np.float32)
    rows, n = x.shape
    d = torch.full((rows, n + stride), math.inf, device="cuda")
    d[:, :n] = cuda(x)
    t, p, m, u = (np.broadcast_to(np.asarray(a, dtype=np.float32), rows) for a in (t, p, m, u))
    k = np.broadcast_to(np.asarray(k, dtype=np.int32), rows)
    tokens, prob = torch.full((rows,), -9, dtype=torch.int32, device="cuda"), torch.full((rows,), -9.0, device="cuda")
    paged.sample_rows(d[:, :n], cuda(u), tokens, prob, cuda(t), cuda(k), cuda(p), cuda(m))
    want = [chain(x[r], t[r], k[r], p[r], m[r], u[r]) for r in range(rows)]
    assert tokens.tolist() == [w[0] for w in want]
    # weights of 2^-46 of the largest, a sum of n of them, one rounding to f32
    assert (np.abs(prob.cpu().numpy() - np.array([w[1] for w in want])) <= 2.0 ** -46 * n + 2.0 ** -24).all()


FILTERS = {"chat": (0.8, 40, 0.95, 0.05), "open": (1.1, 0, 1.0, 0.0), "nucleus": (0.7, 0, 0.9, 0.0), "wide": (1.0, 3000, 0.999, 0.0001), "min_p": (1.5, 0, 1.0, 0.02), "greedy": (0.0, 0, 1.0, 0.0),
           "one": (1.0, 1, 1.0, 0.0), "tiny top_p": (1.0, 0, 1e-6, 0.0), "min_p 1": (1.0, 0, 1.0, 1.0), "cold": (0.01, 0, 1.0, 0.0), "hot": (50.0, 0, 0.99, 0.0)}


@gpu
@pytest.mark.parametrize("name", FILTERS)
@pytest.mark.parametrize("n", [1, 2, 33, 1000, 2049, 8191, 40000])
def test_sampling(n, name):
    g = np.random.default_rng(n)
    rows = 12
    x = g.standard_normal((rows, n)) * np.array([0.01, 0.5, 2.5, 8.0])[np.arange(rows) % 4][:, None] + g.standard_normal((rows, 1)) * 20
    check_sample(x, *FILTERS[name], u=np.concatenate([[0.0, 1 - 2.0 ** -24, 0.5], g.random(rows - 3)]), stride=n % 3)


@gpu
@pytest.mark.parametrize("n", [128256, 151936, 262144])
def test_sampling_whole_vocabularies(n):
    g = np.random.default_rng(n)
    names = list(FILTERS)
    rows = 2 * len(names)
    x = g.standard_normal((rows, n)) * np.where(np.arange(rows) < len(names), 2.5, 0.05)[:, None]
    t, k, p, m = (np.array([FILTERS[names[r % len(names)]][i] for r in range(rows)]) for i in range(4))
    check_sample(x, t, k.astype(int), p, m, g.random(rows))


@gpu
@pytest.mark.parametrize("name", ["chat", "open", "nucleus", "wide", "min_p", "hot"])
def test_sampling_equal_logits(name):
    """Many equal values: counted out in the order of their indices, over every block of a row."""
    g = np.random.default_rng(1)
    u = g.random(6)
    check_sample(np.zeros((6, 30000)), *FILTERS[name], u=u)
    check_sample(np.where(g.random((6, 30000)) < 0.5, 3.0, -0.0), *FILTERS[name], u=u)
    check_sample(torch.from_numpy(g.standard_normal((6, 50000)) * 0.3).bfloat16().float().numpy(), *FILTERS[name], u=u)
    check_sample(g.integers(-3, 4, (6, 20000)) * 0.0, *FILTERS[name], u=u)
    check_sample(g.integers(-3, 4, (6, 20000)) * 1.0, *FILTERS[name], u=u)


@gpu
@pytest.mark.parametrize("name", ["chat", "open", "nucleus", "greedy"])
def test_sampling_masked_logits(name):
    g = np.random.default_rng(2)
    n = 5000
    x = g.standard_normal((8, n)) * 3
    x[0, g.permutation(n)[:4990]] = -np.inf
    x[1, :] = -np.inf
    x[1, 4321] = -5.0
    x[2, :] = -np.inf                        # nothing to draw: the first
    x[3, :] = np.nan                         # no number at all
    x[4, 100:] = np.nan
    x[5, g.permutation(n)[:4000]] = np.finfo(np.float32).min
    x[6, :] = -np.inf
    x[6, :7] = np.nan                        # the first number
    x[7, :] = np.finfo(np.float32).min       # the type's lowest value is a number like any other
    check_sample(x, *FILTERS[name], u=g.random(8))


@gpu
def test_sampling_large_logits_and_defaults():
    g = np.random.default_rng(3)
    with np.errstate(over="ignore"):
        x = g.standard_normal((3, 700)).astype(np.float32) * 1e38
    check_sample(x, 1.0, 0, 1.0, 0.0, g.random(3))
    x[:, 99] = np.inf                        # an infinity takes all (the third row has two of them, which share)
    d, u, tokens = cuda(x), g.random(3).astype(np.float32), torch.zeros(3, dtype=torch.int32, device="cuda")
    paged.sample_rows(d, cuda(u), tokens)
    assert tokens.tolist() == [chain(x[r], 1.0, 0, 1.0, 0.0, u[r])[0] for r in range(3)]
    x, u = g.standard_normal((5, 3001)).astype(np.float32), g.random(5).astype(np.float32)
    tokens = torch.zeros(5, dtype=torch.int32, device="cuda")
    paged.sample_rows(cuda(x), cuda(u), tokens)
    assert tokens.tolist() == [chain(x[r], 1.0, 0, 1.0, 0.0, u[r])[0] for r in range(5)]


@gpu
def test_sampling_is_the_host_samplers_chain():
    """The host sampler's draws come from the same distribution: its first 4000 against the device's for 4000 random numbers, per token within five standard deviations."""
    g = np.random.default_rng(7)
    x, n, draws = (g.standard_normal(200) * 2).astype(np.float32), 200, 4000
    s = L.Sampling(C.sizeof(L.Sampling), 0.8, 30, 0.9, 1.0, 11)
    host = np.empty(draws, dtype=np.int32)
    L.check(L.lib().dooms_cuda_sample(x.ctypes.data, n, C.byref(s), draws, host.ctypes.data))
    tokens = torch.empty(draws, dtype=torch.int32, device="cuda")
    f = lambda v: torch.full((draws,), v, device="cuda")  # noqa: E731
    paged.sample_rows(cuda(x).expand(draws, n).contiguous(), cuda(g.random(draws), torch.float32), tokens, None, f(0.8), torch.full((draws,), 30, dtype=torch.int32, device="cuda"), f(0.9))
    a, b = np.bincount(host, minlength=n), np.bincount(tokens.cpu().numpy(), minlength=n)
    assert ((a > 0) == (b > 0)).mean() > 0.97 and set(np.nonzero(b)[0]) <= set(np.argsort(-x)[:30])
    assert (np.abs(a - b) <= 5 * np.sqrt(a + b + 1)).all()


@gpu
def test_sampling_twice_gives_the_same_and_rows_do_not_touch_one_another():
    g = np.random.default_rng(8)
    x, u = cuda(g.standard_normal((100, 20000)) * 0.2, torch.float32), cuda(g.random(100), torch.float32)
    out = [torch.zeros(100, dtype=torch.int32, device="cuda") for _ in range(3)]
    paged.sample_rows(x, u, out[0])
    paged.sample_rows(x, u, out[1])
    for r in range(0, 100, 7):
        paged.sample_rows(x[r:r + 1], u[r:r + 1], out[2][r:r + 1])
    assert torch.equal(out[0], out[1]) and torch.equal(out[0][::7], out[2][::7])


@gpu
@pytest.mark.parametrize("rows, n", [(75, 20000), (160, 17000), (400, 5000)])
def test_sampling_batches_of_mixed_rows(rows, n):
    """More rows than there are blocks for eight each: rows that a bound leaves little of and rows that need a total go in two launches, also under a capture."""
    g = np.random.default_rng(rows)
    names = list(FILTERS)
    kind = [names[i] for i in g.integers(0, len(names), rows)]
    x = (g.standard_normal((rows, n)) * g.choice([0.05, 1.0, 2.5, 6.0], rows)[:, None]).astype(np.float32)
    t, p, m = (np.array([FILTERS[name][i] for name in kind], dtype=np.float32) for i in (0, 2, 3))
    k, u = np.array([FILTERS[name][1] for name in kind], dtype=np.int32), g.random(rows).astype(np.float32)
    check_sample(x, t, k, p, m, u)
    d = [cuda(a) for a in (x, u, t, k, p, m)]
    tokens, prob = torch.full((rows,), -9, dtype=torch.int32, device="cuda"), torch.zeros(rows, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        d[0].mul_(1.0)                         # what the sampling reads is made by the kernel in front of it, and read by the one behind it
        paged.sample_rows(d[0], d[1], tokens, prob, *d[2:], stream=torch.cuda.current_stream().cuda_stream)
        copy = tokens.clone()
    for _ in range(3):
        tokens.fill_(-9)
        graph.replay()
    assert copy.tolist() == [chain(x[r], t[r], k[r], p[r], m[r], u[r])[0] for r in range(rows)]


@gpu
@pytest.mark.parametrize("offset", [1, 2, 3, 4])
def test_sampling_rows_that_do_not_begin_on_16_bytes(offset):
    g = np.random.default_rng(offset)
    x = g.standard_normal((6, 5001)).astype(np.float32) * 3
    flat = torch.full((offset + 6 * 5003,), math.inf, device="cuda")
    rows = flat[offset:].view(6, 5003)[:, :5001]
    rows.copy_(cuda(x))
    t, k, p, m, u = (np.array(a) for a in zip(*[FILTERS[n] + (g.uniform(),) for n in ("chat", "open", "nucleus", "wide", "min_p", "greedy")]))
    tokens = torch.full((6,), -9, dtype=torch.int32, device="cuda")
    paged.sample_rows(rows, cuda(u, torch.float32), tokens, None, cuda(t, torch.float32), cuda(k, torch.int32), cuda(p, torch.float32), cuda(m, torch.float32))
    assert tokens.tolist() == [chain(x[r], t[r], int(k[r]), p[r], m[r], u[r])[0] for r in range(6)]


# ---------------------------------------------------------------- large pools, many rows, calls at once

@gpu
def test_positions_of_a_pool_beyond_32_bits():
    """Pools of more than 2^32 bytes and 2^31 values, in the largest pages: rows written and read at their end are those that were meant."""
    H, K, D, page, n = 8, 8, 128, 65536, 65600
    pages = (1 << 31) // (K * D * page) + 3                  # 2^31 values and three pages
    keys, values = (torch.empty(pages, page, K, D, dtype=torch.float16, device="cuda") for _ in range(2))
    cache = paged.PagedCache(keys, values, torch.tensor([[pages - 1, pages - 2], [0, 1]], dtype=torch.int32, device="cuda"))
    small = Cache([n], K, D, 4096, seed=3)                   # the same sequence in small pages
    line = torch.from_numpy(small.line(0, n)).cuda()
    for mine, other in ((keys, small.keys), (values, small.values)):
        mine[pages - 1] = other.view(-1, K, D)[line[:page]]
        mine[pages - 2, :n - page] = other.view(-1, K, D)[line[page:]]
        mine[0].zero_()
    scratch = small.scratch(H)
    new, ids = 3, torch.zeros(3, dtype=torch.int32, device="cuda")
    qkv = torch.randn(new, (H + 2 * K) * D, device="cuda")
    at = torch.tensor([n - 1, n - 2, n - 3], dtype=torch.int32, device="cuda")
    outs = []
    for c in (cache, small.cache):
        q = torch.empty(new, H, D, device="cuda")
        c.rope_store(qkv, ids, at, at[None], q, base=1e6, neox=True)
        one, some = torch.zeros_like(q), torch.zeros(new, H, D, dtype=torch.float16, device="cuda")
        c.attention(q, ids, at + 1, n, one, scratch)
        c.attention_prompt(q.half(), ids[:1], torch.tensor([0, new], dtype=torch.int32, device="cuda"), at[:1] + 1, some, scratch)
        outs.append((q, one, some))
    assert status() == (L.OK, 0)
    for a, b in zip(*outs):
        assert torch.equal(a, b)
    assert (keys[0] == 0).all() and (keys[pages - 2, n - page - 3:n - page] == small.keys.view(-1, K, D)[line[n - 3:]]).all()


@gpu
def test_more_rows_than_threads():
    """Batches of thousands of short sequences."""
    lengths = [1 + i % 3 for i in range(2500)]
    cache = Cache(lengths, 1, 64, 16, seed=8)
    check_decode(cache, lengths, 2, torch.float16, idle=range(0, 2500, 7))
    check_prompt(cache, [i % 2 for i in range(2500)], lengths, 2, idle=range(0, 2500, 7))


@gpu
def test_calls_at_once_on_two_streams():
    """Every operator on two streams at the same time, each with its own scratch and outputs: what each gives is what it gives alone."""
    H, K, D, V = 16, 4, 128, 30000
    g = np.random.default_rng(12)

    def side(seed):
        lengths = [5000, 17, 900, 64]
        cache = Cache([n + 1 for n in lengths], K, D, 16, seed=seed)
        stream, scratch = torch.cuda.Stream(), cache.scratch(H)
        seq, at = torch.arange(4, dtype=torch.int32, device="cuda"), cuda(np.array(lengths, np.int32))
        qkv, logits, u = torch.randn(4, (H + 2 * K) * D, device="cuda"), torch.randn(64, V, device="cuda") * 2, torch.rand(64, device="cuda")
        top_k = cuda(g.choice([0, 40], 64), torch.int32)
        pq, start = torch.randn(2400, H, D, device="cuda").half(), cuda(np.array([0, 900, 910, 1100, 1164], np.int32))

        def run():
            q, out, pout = torch.empty(4, H, D, device="cuda"), torch.zeros(4, H, D, device="cuda"), torch.zeros_like(pq)
            tokens, prob = torch.zeros(64, dtype=torch.int32, device="cuda"), torch.zeros(64, device="cuda")
            s = stream.cuda_stream
            cache.cache.rope_store(qkv, seq, at, at[None], q, base=1e4, neox=True, stream=s)
            cache.cache.attention(q, seq, at + 1, 5001, out, scratch, stream=s)
            cache.cache.attention_prompt(pq, seq, start, at + 1, pout, scratch, stream=s)
            paged.sample_rows(logits, u, tokens, prob, top_k=top_k, stream=s)
            return q, out, pout, tokens, prob
        return stream, run
    sides = [side(1), side(2)]
    torch.cuda.synchronize()
    alone = []
    for stream, run in sides:
        with torch.cuda.stream(stream):
            alone.append(run())
        torch.cuda.synchronize()
    results = [[], []]
    for _ in range(10):
        for i, (stream, run) in enumerate(sides):
            with torch.cuda.stream(stream):
                results[i].append(run())
    torch.cuda.synchronize()
    assert status() == (L.OK, 0)
    for i in range(2):
        for result in results[i]:
            assert all(torch.equal(a, b) for a, b in zip(result, alone[i]))


# ---------------------------------------------------------------- together

@gpu
def test_a_serving_run():
    """Two prompts (one with an image's positions) stored and attended in one packed call, then three steps of both sequences and a third that idles at first: the cache that
    store leaves is the one that attention reads, and what is sampled is what the next step takes."""
    H, K, D, V, page = 6, 2, 64, 500, 16
    g = np.random.default_rng(9)
    pool, prompts, sections = 16, [37, 21], [8, 12, 12]
    table = g.permutation(pool)[:15].reshape(3, 5).astype(np.int32)
    keys, values = (torch.full((pool, page, K, D), math.nan, dtype=torch.float16, device="cuda") for _ in range(2))
    cache = paged.PagedCache(keys, values, cuda(table))
    scratch = torch.empty(cache.scratch_bytes(H), dtype=torch.uint8, device="cuda")
    embed = cuda(g.standard_normal((V, (H + 2 * K) * D)), torch.float32)
    head = cuda(g.standard_normal((H * D, V)) * 0.1, torch.float32)
    tokens = [g.integers(0, V, n) for n in prompts] + [np.array([], dtype=np.int64)]
    seen = [[], [], []]                       # (positions [3], token) of everything stored so far

    def expected(i, upto):
        rows = embed[torch.tensor([t for _, t in seen[i][:upto]])].cpu().numpy().astype(np.float64).reshape(upto, H + 2 * K, D)
        pos = np.array([p for p, _ in seen[i][:upto]]).T.reshape(3, upto)
        y = turned(rows[:, :H + K], pos, sections, 1e4, True)
        k = y[:, H:].astype(np.float32).astype(np.float16).astype(np.float64)
        return y[:, :H], k, rows[:, H + K:].astype(np.float16).astype(np.float64)

    def compare(out, i, upto, half):
        q, k, v = expected(i, upto)
        want, mass, reach = attend(q[-1], k, v, 0.125)
        # the query rounded to f16 moves a score by half a step of each product; a key one f16 step off (its rotation rounds differently) by a step
        extra = mass * 2 * 0.125 * reach * (HALF * (3 if half else 2))
        assert (np.abs(out.cpu().numpy().astype(np.float64) - want) <= bound(want, mass, reach, D, 0.125, half) + extra).all()

    def place(i, t):
        n = len(seen[i])
        image = i == 0 and 10 <= n < 26
        seen[i].append(((10, 10 + (n - 10) // 4, 10 + (n - 10) % 4) if image else (n, n, n), int(t)))
        return i, n, seen[i][-1][0], int(t)
    rows = [place(i, t) for i in range(2) for t in tokens[i]]
    q = torch.empty(len(rows), H, D, dtype=torch.float16, device="cuda")
    cache.rope_store(embed[torch.tensor([r[3] for r in rows])], cuda(np.array([r[0] for r in rows], np.int32)), cuda(np.array([r[1] for r in rows], np.int32)),
                     cuda(np.array([r[2] for r in rows], np.int32).T), q, base=1e4, neox=True, sections=sections)
    out = torch.empty_like(q)
    cache.attention_prompt(q, cuda(np.arange(2, dtype=np.int32)), cuda(np.array([0, 37, 58], np.int32)), cuda(np.array(prompts, np.int32)), out, scratch)
    for i, last in ((0, 36), (1, 57)):
        for back in (0, 5, 20):
            compare(out[last - back], i, prompts[i] - back, True)
    state = torch.stack([out[36].float(), out[57].float(), torch.zeros(H, D, device="cuda")])
    for step in range(3):
        logits = state.flatten(1) @ head
        picked, u = torch.zeros(3, dtype=torch.int32, device="cuda"), g.random(3).astype(np.float32)
        paged.sample_rows(logits, cuda(u), picked, None, torch.full((3,), 0.9, device="cuda"), torch.full((3,), 20, dtype=torch.int32, device="cuda"))
        for i in range(3):
            assert picked[i] == chain(logits[i].cpu().numpy(), 0.9, 20, 1.0, 0.0, u[i])[0]
        active = [0, 1, 2] if step else [0, 1]
        rows = [place(i, picked[i]) for i in active]
        seq = np.array([i if i in active else -1 for i in range(3)], np.int32)
        at = np.array([len(seen[i]) - 1 for i in range(3)], np.int32)
        pos = np.array([seen[i][-1][0] if i in active else (0, 0, 0) for i in range(3)], np.int32).T
        q = torch.zeros(3, H, D, device="cuda")
        cache.rope_store(embed[picked.long()], cuda(seq), cuda(at), cuda(pos), q, base=1e4, neox=True, sections=sections)
        out = torch.zeros(3, H, D, device="cuda")
        cache.attention(q, cuda(seq), cuda(at + 1), 80, out, scratch)
        for i in active:
            compare(out[i], i, len(seen[i]), False)
        assert 2 in active or (out[2] == 0).all()
        state = out
    assert status() == (L.OK, 0)
