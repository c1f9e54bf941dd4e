"""The 4-bit key/value cache (module w4a16_kv): written bytes and values read back bit for bit, attention against
64 bits, and refusals.

Attention's tolerance, element by element: half a unit in the last place of the output's type (2^-11 of an fp16
result, 2^-8 of a bf16 one, 2^-25 of a subnormal one), and 2^-10 of sum p |v| / sum p for what is rounded inside (a
probability times its value's scale to fp16, 2^-11, and fp32 sums and exponentials, well under as much again).
The lse is held in fp32 from fp32 scores: 2^-16 of (1 + |lse|).
"""
from __future__ import annotations

import ctypes
import os

import numpy as np
import pytest
import torch

from tests import _kv4
from tests._helpers import PKG, torch_cuda

SIZES = [(64, 64), (128, 64), (128, 128)]
DTYPES = [torch.float16, torch.bfloat16]


def kv():
    import w4a16_kv
    return w4a16_kv


def values(rng, shape, dtype, spread=1.0):
    x = rng.standard_normal(shape, dtype=np.float32) * spread
    x *= np.where(rng.random(shape[-2:]) > 0.95, 6, 1).astype(np.float32)           # a few channels larger than the rest
    return torch.from_numpy(x + 0.5 * rng.standard_normal(shape[-2:], dtype=np.float32)).to(dtype)


def filled(rng, lens, P, H, D, G, dtype=torch.float16, spare=3, junk=True):
    """A cache (numpy, built by the restated format) whose sequences' pages lie in random order among junk, and the table."""
    width = max(1, -(-max([*lens, 1]) // P))
    pages = width * len(lens) + spare
    cache = rng.integers(0, 256, (pages, H, _kv4.page_bytes(P, D, G)), dtype=np.uint8) if junk else np.zeros(
        (pages, H, _kv4.page_bytes(P, D, G)), np.uint8)
    if junk:                                                     # scales and zeros of unwritten places: NaN and infinities
        cache[:, :, P * D:].view(np.uint16)[...] = rng.choice(np.array([0x7E00, 0x7C00, 0xFC00, 0xFFFF], np.uint16), (pages, H, 4 * D // G * P))
    table = rng.permutation(pages)[:width * len(lens)].reshape(len(lens), width).astype(np.int32)
    for b, n in enumerate(lens):
        if n:
            t = np.arange(n)
            _kv4.write(cache, values(rng, (n, H, D), dtype).float().numpy(), values(rng, (n, H, D), dtype).float().numpy(),
                       table[b, t // P].astype(np.int64) * P + t % P, G, P)
    return cache, table


def check(out, lse, ref, dtype):
    want, want_lse, spread = ref
    got = out.double().cpu().numpy()
    u = 2.0**-11 if dtype == torch.float16 else 2.0**-8
    nan = np.isnan(want)
    assert np.array_equal(np.isnan(got), nan)
    err = np.abs(got - want)[~nan] - (u * np.abs(want) + 2.0**-10 * spread + 2.0**-25)[~nan]
    assert err.size == 0 or err.max() <= 0, f"{err.max():.3g} over the tolerance"
    assert np.array_equal(want[~nan] == 0, (got == 0)[~nan]) or (want[~nan] != 0).all() or (got[(want == 0) & ~nan] == 0).all()
    if lse is not None:
        gl = lse.double().cpu().numpy()
        ok = ~np.isnan(want_lse) & np.isfinite(want_lse)
        assert np.array_equal(np.isneginf(gl), np.isneginf(want_lse))
        assert (np.abs(gl - want_lse)[ok] <= 2.0**-16 * (1 + np.abs(want_lse[ok]))).all()


def attend(q, cache, table, lens, G, P, q_start=None, device="cuda", **kw):
    """(out, lse) of the op and the 64-bit reference."""
    dev = lambda x, t: None if x is None else torch.as_tensor(np.asarray(x), dtype=t).to(device)  # noqa: E731
    out, lse = kv().kv4_attention(q.to(device), torch.from_numpy(cache).to(device), dev(table, torch.int32), dev(lens, torch.int32), G,
                                  q_start=dev(q_start, torch.int32), return_lse=True, **kw)
    kw.pop("max_q", None)
    return out, lse, _kv4.attention(q, cache, table, lens, G, P, q_start, **kw)


# ------------------------------------------------------------------------------------- on the CPU


def test_format_error_is_half_a_step():
    """|s (q - z) - x| <= s / 2 (and the clamp's share of it) in 64 bits for anything that fp16 holds."""
    rng = np.random.default_rng(1)
    x = (rng.standard_normal((200, 128)) * 10.0 ** rng.uniform(-3, 3, (200, 1)) + rng.choice([0, 0, 30, -5], (200, 1))).astype(np.float16)
    for G in (64, 128):
        q, s, z = _kv4.quantise(x, G)
        assert (np.abs(z.astype(float)) <= 97).all() and (z.astype(float) * 8 == np.rint(z.astype(float) * 8)).all()
        back = (q.reshape(200, -1, G) - z.astype(np.float64)[..., None]) * s.astype(np.float64)[..., None]
        assert (np.abs(back - x.reshape(200, -1, G).astype(np.float64)) <= s.astype(np.float64)[..., None] * 0.5001).all()
        # q - z is exact in fp16, which the matrix instructions' operands rest on
        d = q.reshape(200, -1, G) - z.astype(np.float64)[..., None]
        assert (d.astype(np.float16).astype(np.float64) == d).all()


def test_restated_bytes_round_trip():
    rng = np.random.default_rng(2)
    for D, G in SIZES:
        cache = np.zeros((3, 2, _kv4.page_bytes(32, D, G)), np.uint8)
        k, v = (rng.standard_normal((40, 2, D)).astype(np.float16) for _ in range(2))
        slots = rng.permutation(96)[:40]
        _kv4.write(cache, k, v, slots, G, 32)
        for x, got in zip((k, v), _kv4.read(cache, slots, D, G, 32)):
            q, s, z = _kv4.quantise(x, G)
            want = (q.reshape(40, 2, -1, G) - z.astype(float)[..., None]) * s.astype(float)[..., None]
            assert np.array_equal(got, want.reshape(40, 2, D))


def test_refuses_host_tensors():
    pytest.importorskip("w4a16_kv")
    c = torch.zeros(1, 1, _kv4.page_bytes(16, 64, 64), dtype=torch.uint8)
    k, slots = torch.zeros(1, 1, 64).half(), torch.zeros(1, dtype=torch.int64)
    for call in (lambda: kv().kv4_write(c, k, k, slots, 64), lambda: kv().kv4_read(c, slots, 64, 64),
                 lambda: kv().kv4_attention(k, c, torch.zeros(1, 1).int(), torch.ones(1).int(), 64)):
        with pytest.raises(RuntimeError, match="must be CUDA"):
            call()
    with pytest.raises(RuntimeError, match="unsupported sizes"):
        kv().kv4_cache(1, 24, 1, 64, 64, device="cpu")
    assert kv().kv4_cache(2, 32, 3, 128, 64, device="cpu").shape == (2, 3, _kv4.page_bytes(32, 128, 64))


class Cache(ctypes.Structure):
    _fields_ = [("data", ctypes.c_void_p)] + [(n, ctypes.c_int64) for n in ("pages", "page_size", "kv_heads", "head_dim", "group_size")]


class Args(ctypes.Structure):
    _fields_ = [("q", ctypes.c_void_p), ("out", ctypes.c_void_p), ("lse", ctypes.c_void_p)] + \
               [(n, ctypes.c_int64) for n in ("q_token_stride", "q_head_stride", "tokens", "heads", "batch")] + \
               [("block_table", ctypes.c_void_p), ("table_width", ctypes.c_int64), ("table_stride", ctypes.c_int64),
                ("seq_lens", ctypes.c_void_p), ("q_start", ctypes.c_void_p), ("max_q", ctypes.c_int64), ("window", ctypes.c_int64),
                ("scale", ctypes.c_float), ("bf16", ctypes.c_int32), ("causal", ctypes.c_int32)]


@pytest.fixture(scope="module")
def lib():
    path = os.path.join(PKG, "libw4a16_hip.so")
    if not os.path.exists(path):
        pytest.skip("library not built")
    L = ctypes.CDLL(path)
    L.w4a16_last_error.restype = ctypes.c_char_p
    L.w4a16_kv4_page_bytes.restype = L.w4a16_kv4_attention_workspace.restype = ctypes.c_int64
    L.w4a16_kv4_page_bytes.argtypes = [ctypes.c_int64] * 3
    L.w4a16_kv4_write.argtypes = [ctypes.c_void_p] * 3 + [ctypes.c_int] + [ctypes.c_int64] * 5 + [ctypes.c_void_p] * 2
    L.w4a16_kv4_read.argtypes = [ctypes.c_void_p] * 2 + [ctypes.c_int64, ctypes.c_int] + [ctypes.c_void_p] * 3
    L.w4a16_kv4_attention_workspace.argtypes = [ctypes.c_void_p] * 3
    L.w4a16_kv4_attention.argtypes = [ctypes.c_void_p] * 4 + [ctypes.c_int64] + [ctypes.c_void_p] * 2
    return L


def test_c_entry_points_refuse_before_any_device_work(lib):
    assert lib.w4a16_kv4_page_bytes(64, 128, 128) == 64 * 136 and lib.w4a16_kv4_page_bytes(16, 128, 64) == 16 * 144
    assert [lib.w4a16_kv4_page_bytes(*x) for x in ((8, 128, 128), (24, 128, 128), (4112, 128, 128), (16, 96, 64), (16, 64, 128))] == [0] * 5
    ok = dict(data=4096, pages=2, page_size=16, kv_heads=2, head_dim=128, group_size=64)
    p = 4096                                                     # never dereferenced: every call is refused on the host
    bad = [(dict(head_dim=80), b"head size"), (dict(group_size=32), b"group size"), (dict(head_dim=64, group_size=128), b"divide"),
           (dict(page_size=20), b"page size"), (dict(kv_heads=0), b"kv_heads"), (dict(pages=-1), b"range"), (dict(data=4100), b"aligned"),
           (dict(data=None), b"null")]
    for change, word in bad:
        c = Cache(**{**ok, **change})
        a, lim = Args(p, p, None, 256, 128, 1, 2, 1, p, 1, 1, p, None, 1, 0, 1.0, 0, 1), (ctypes.c_int32 * 4)(256, 163840, 1024, 950)
        assert lib.w4a16_kv4_write(ctypes.byref(c), p, p, 0, 1, 256, 128, 256, 128, p, None) == 1
        assert word in lib.w4a16_last_error() and lib.w4a16_last_error().startswith(b"kv4_write")
        assert lib.w4a16_kv4_read(ctypes.byref(c), p, 1, 0, p, p, None) == 1 and word in lib.w4a16_last_error()
        assert lib.w4a16_kv4_attention_workspace(ctypes.byref(c), ctypes.byref(a), lim) == -1 and word in lib.w4a16_last_error()
        assert lib.w4a16_kv4_attention(ctypes.byref(c), ctypes.byref(a), lim, None, 0, p, None) == 1 and word in lib.w4a16_last_error()
    c = Cache(**ok)
    assert lib.w4a16_kv4_write(ctypes.byref(c), None, p, 0, 1, 256, 128, 256, 128, p, None) == 1 and b"null" in lib.w4a16_last_error()
    assert lib.w4a16_kv4_write(ctypes.byref(c), p + 1, p, 0, 1, 256, 128, 256, 128, p, None) == 1 and b"aligned" in lib.w4a16_last_error()
    assert lib.w4a16_kv4_write(ctypes.byref(c), p, p, 0, -1, 256, 128, 256, 128, p, None) == 1
    assert lib.w4a16_kv4_read(ctypes.byref(c), p, 1, 0, p + 2, p, None) == 1 and b"aligned" in lib.w4a16_last_error()
    assert lib.w4a16_kv4_write(ctypes.byref(c), None, None, 0, 0, 0, 0, 0, 0, None, None) == 0        # nothing to do
    names = [f[0] for f in Args._fields_]
    good = dict(zip(names, (p, p, None, 256, 128, 1, 2, 1, p, 1, 1, p, None, 1, 0, 1.0, 0, 1)))
    lim = (ctypes.c_int32 * 4)(256, 163840, 1024, 950)
    assert lib.w4a16_kv4_attention_workspace(ctypes.byref(c), ctypes.byref(Args(**good)), lim) >= 0
    for change, word in [(dict(heads=3), b"multiple"), (dict(scale=0.0), b"scale"), (dict(scale=float("nan")), b"scale"), (dict(scale=-1.0), b"scale"),
                         (dict(tokens=2), b"one query"), (dict(max_q=0), b"range"), (dict(window=-1), b"range"), (dict(q=None), b"null"),
                         (dict(seq_lens=None), b"null"), (dict(block_table=None), b"null"), (dict(out=p + 4), b"aligned"), (dict(lse=p + 2), b"aligned"),
                         (dict(batch=2, tokens=2, table_stride=0), b"overlap"), (dict(table_width=1 << 27), b"range")]:
        a = Args(**{**good, **change})
        assert lib.w4a16_kv4_attention(ctypes.byref(c), ctypes.byref(a), lim, None, 0, p, None) == 1, change
        assert word in lib.w4a16_last_error(), (change, lib.w4a16_last_error())


# ------------------------------------------------------------------------------------- on the GPU


def laid_out(x, layout):
    """x [T, H, D] on the GPU as a user may hold it: contiguous, slices of a fused projection, at odd element offsets, or
    with the heads outermost."""
    T, H, D = x.shape
    if layout == "fused":
        whole = torch.full((T, 3 * H + 1, D), float("nan"), dtype=x.dtype, device="cuda")
        whole[:, H:2 * H] = x.cuda()
        return whole[:, H:2 * H]
    if layout == "odd":
        whole = torch.full((T, H * (D + 3) + 1), float("nan"), dtype=x.dtype, device="cuda")
        view = whole[:, 1:].view(T, H, D + 3)[..., :D] if whole[:, 1:].is_contiguous() else whole[:, 1:].unflatten(1, (H, D + 3))[..., :D]
        view.copy_(x.cuda())
        return view
    if layout == "heads":
        return x.cuda().transpose(0, 1).contiguous().transpose(0, 1)
    return x.cuda().contiguous()


def slot_cases(rng, kind, T, total):
    if kind == "run":                                            # one run from an odd place
        return np.arange(5, 5 + T)
    if kind == "aligned":
        return np.arange(16, 16 + T)
    s = rng.permutation(total)[:T]
    if kind == "holes":                                          # padding and slots outside the cache
        s[::3] = rng.choice([-1, -2**40, total, 2**40], s[::3].shape)
    return s


@pytest.mark.gpu
@pytest.mark.parametrize("D,G", SIZES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,H,P,kind,layout", [(1, 1, 16, "random", "plain"), (1, 8, 64, "run", "fused"), (37, 3, 32, "run", "odd"),
                                               (70, 2, 16, "holes", "heads"), (130, 5, 48, "aligned", "plain"),
                                               (64, 2, 128, "random", "fused"), (100, 1, 64, "run", "plain"), (200, 2, 16, "aligned", "odd")])
def test_write_gives_the_formats_bytes(D, G, dtype, T, H, P, kind, layout):
    torch_cuda()
    rng = np.random.default_rng(T * 100 + D + G)
    pages = -(-(T + 32) // P) + 2
    slots = slot_cases(rng, kind, T, pages * P).astype(np.int64)
    k, v = values(rng, (T, H, D), dtype), values(rng, (T, H, D), dtype, 0.1)
    want = np.full((pages, H, _kv4.page_bytes(P, D, G)), 0xA5, np.uint8)
    cache = torch.from_numpy(want.copy()).cuda()
    kv().kv4_write(cache, laid_out(k, layout), laid_out(v, layout), torch.from_numpy(slots).cuda(), G)
    _kv4.write(want, k.float().numpy(), v.float().numpy(), slots, G, P)
    assert np.array_equal(cache.cpu().numpy(), want)             # and nothing beside those tokens
    rk, rv = kv().kv4_read(cache, torch.from_numpy(slots).cuda(), D, G, dtype)
    for got, exact in zip((rk, rv), _kv4.read(want, slots, D, G, P)):
        assert got.shape == (T, H, D) and got.is_contiguous()
        assert np.array_equal(_kv4.bits(got), _kv4.bits(torch.from_numpy(exact).float().to(dtype)))


@pytest.mark.gpu
@pytest.mark.parametrize("D,G", SIZES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("run", [False, True])
def test_write_of_unusual_values(D, G, dtype, run):
    torch_cuda()
    rows = [0.0, -0.0, 1.0, -3.5, 65504.0, float("inf"), float("-inf"), float("nan"), 6e-8, 1e-5, 2.0**-14]
    T = 32
    rng = np.random.default_rng(5)
    x = np.zeros((T, 1, D), np.float32)
    for i in range(T):
        x[i, 0] = rows[i % len(rows)]                            # a constant group
        if i >= len(rows):
            x[i, 0] = rng.standard_normal(D) * 10.0 ** rng.integers(-4, 4)
            x[i, 0, rng.integers(0, D, 2)] = rows[i % len(rows)]
    if dtype == torch.bfloat16:
        x[-1] *= 1e30
    with np.errstate(over="ignore"):
        k = torch.from_numpy(x).to(dtype)
    v = k.flip(0).contiguous()
    slots = np.arange(T) + 16 if run else rng.permutation(64)[:T]
    want = np.zeros((4, 1, _kv4.page_bytes(16, D, G)), np.uint8)
    cache = torch.from_numpy(want.copy()).cuda()
    kv().kv4_write(cache, k.cuda(), v.cuda(), torch.from_numpy(slots).cuda(), G)
    _kv4.write(want, k.float().numpy(), v.float().numpy(), slots, G, 16)
    assert np.array_equal(cache.cpu().numpy(), want)
    rk, _ = kv().kv4_read(cache, torch.from_numpy(slots).cuda(), D, G, torch.float16)
    nan = torch.isnan(k.float().view(T, -1, G)).any(-1, keepdim=True).expand(T, D // G, G).reshape(T, 1, D)
    assert torch.equal(torch.isnan(rk.cpu()), nan)


@pytest.mark.gpu
@pytest.mark.parametrize("D,G", SIZES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind,T", [("run", 1), ("run", 90), ("random", 33), ("holes", 50), ("aligned", 128)])
def test_read_of_any_bytes(D, G, dtype, kind, T):
    torch_cuda()
    rng = np.random.default_rng(T + D)
    P, H = 32, 3
    cache = rng.integers(0, 256, (8, H, _kv4.page_bytes(P, D, G)), dtype=np.uint8)
    side = cache[:, :, P * D:].view(np.uint16).reshape(8, H, 4, D // G, P)
    for zero in (1, 3):                                          # zeros as the format has them; scales of any bits
        side[:, :, zero] = (rng.integers(-97 * 8, 97 * 8, side[:, :, zero].shape) / 8).astype(np.float16).view(np.uint16)
    slots = slot_cases(rng, kind, T, 8 * P).astype(np.int64)
    with np.errstate(invalid="ignore"):
        want = _kv4.read(cache, slots, D, G, P)
    for got, exact in zip(kv().kv4_read(torch.from_numpy(cache).cuda(), torch.from_numpy(slots).cuda(), D, G, dtype), want):
        ref = torch.from_numpy(exact).float().to(dtype)
        nan = torch.isnan(ref)
        assert torch.equal(torch.isnan(got.cpu()), nan)
        assert np.array_equal(_kv4.bits(got.cpu().masked_fill(nan, 0)), _kv4.bits(ref.masked_fill(nan, 0)))


@pytest.mark.gpu
@pytest.mark.parametrize("D,G", SIZES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("Hq,H,P,lens,window", [
    (1, 1, 16, [1], 0), (4, 1, 64, [15, 16, 17], 0), (8, 2, 16, [0, 63, 64, 65, 0, 1], 0), (12, 4, 32, [100, 7], 0), (16, 1, 64, [700], 0),
    (8, 1, 16, [129, 1000], 0), (5, 1, 48, [333], 0), (8, 2, 16, [0, 500, 3, 64], 50), (4, 4, 128, [257, 128], 1), (32, 2, 16, [90, 2], 64)])
def test_attention_of_single_tokens(D, G, dtype, Hq, H, P, lens, window):
    torch_cuda()
    rng = np.random.default_rng(sum(lens) + Hq)
    cache, table = filled(rng, lens, P, H, D, G, dtype)
    q = values(rng, (len(lens), Hq, D), dtype)
    out, lse, ref = attend(q, cache, table, lens, G, P, window=window)
    assert out.shape == q.shape and out.dtype == dtype and lse.dtype == torch.float32
    check(out, lse, ref, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("D,G", SIZES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("Hq,H,P,lens,counts,window,causal", [
    (4, 1, 16, [20, 3], [2, 3], 0, True), (8, 1, 32, [150, 0, 40], [2, 0, 1], 0, True), (2, 2, 16, [70, 90], [5, 8], 30, True),
    (4, 2, 64, [200], [40], 0, True), (1, 1, 16, [129], [129], 0, True), (4, 1, 16, [65, 0, 30, 1], [65, 0, 17, 1], 0, True),
    (8, 2, 32, [300, 10], [33, 10], 0, True), (3, 1, 48, [100, 260], [100, 50], 0, True), (4, 4, 16, [190, 40], [190, 40], 21, True),
    (4, 1, 16, [5, 50], [20, 60], 0, True), (4, 2, 16, [90, 33], [40, 20], 0, False), (4, 2, 16, [90, 33], [3, 2], 0, False),
    (6, 2, 16, [140], [60], 17, False), (64, 1, 16, [40], [3], 0, True)])
def test_attention_of_several_tokens(D, G, dtype, Hq, H, P, lens, counts, window, causal):
    torch_cuda()
    rng = np.random.default_rng(sum(lens) + Hq + sum(counts))
    cache, table = filled(rng, lens, P, H, D, G, dtype)
    start = np.concatenate([[0], np.cumsum(counts)])
    q = values(rng, (int(start[-1]), Hq, D), dtype)
    out, lse, ref = attend(q, cache, table, lens, G, P, start, max_q=max(counts), window=window, causal=causal)
    check(out, lse, ref, dtype)
    again, lse2, _ = attend(q, cache, table, lens, G, P, start, window=window, causal=causal)     # max_q left to the op
    check(again, lse2, ref, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("q_len,told", [(1, 1), (7, 1), (40, 3), (150, 1)])
def test_attention_holds_for_any_max_q(q_len, told):
    """max_q selects the kernel; queries past it are computed too."""
    torch_cuda()
    rng = np.random.default_rng(q_len)
    lens, counts = [q_len + 30, 9], [q_len, 2]
    cache, table = filled(rng, lens, 16, 2, 128, 64)
    q = values(rng, (q_len + 2, 8, 128), torch.float16)
    out, lse, ref = attend(q, cache, table, lens, 64, 16, [0, q_len, q_len + 2], max_q=told)
    check(out, lse, ref, torch.float16)


@pytest.mark.gpu
@pytest.mark.parametrize("q_len", [1, 4, 60])
@pytest.mark.parametrize("D,G", SIZES)
def test_attention_never_sees_what_is_masked(q_len, D, G):
    """Pages that the table does not name, entries outside the cache, and places past the end hold NaN, infinities or
    nothing; a length past the table is cut."""
    torch_cuda()
    rng = np.random.default_rng(q_len)
    P, lens = 16, [75, 200, 64]
    cache, table = filled(rng, lens, P, 2, D, G)
    table[0, 1], table[0, 3] = -1, 10**6                         # holes in the first sequence
    table[2, :] = -7                                             # the third has no page: its rows see nothing
    told = [75, 200, 10**6]
    start = np.arange(4) * q_len
    q = values(rng, (3 * q_len, 4, D), torch.float16)
    out, lse, ref = attend(q, cache, table, told, G, P, start, max_q=q_len)
    check(out, lse, ref, torch.float16)
    assert not torch.isnan(out).any() and (out[2 * q_len:] == 0).all() and torch.isneginf(lse[2 * q_len:]).all()
    out, lse, ref = attend(q, cache, table, [-5, 0, 0], G, P, start, max_q=q_len)
    assert (out == 0).all() and torch.isneginf(lse).all()


@pytest.mark.gpu
@pytest.mark.parametrize("q_len", [1, 30])
@pytest.mark.parametrize("where", ["q", "k", "v"])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_attention_passes_on_nan(q_len, where, value):
    """A NaN that a row attends to makes that row NaN, and no other row; infinities in q do too."""
    torch_cuda()
    rng = np.random.default_rng(3)
    P, H, D, G, n = 16, 2, 128, 128, 50
    k, v = (values(rng, (n, H, D), torch.float16) for _ in range(2))
    q = values(rng, (q_len, 8, D), torch.float16)
    if where == "q":
        q[0, 5, 17] = value
    elif value == value:
        pytest.skip("infinities saturate when they are written")
    else:
        (k if where == "k" else v)[n - 1, 1, 40] = value         # seen by the last query alone, in KV head 1
    cache = np.zeros((5, H, _kv4.page_bytes(P, D, G)), np.uint8)
    _kv4.write(cache, k.float().numpy(), v.float().numpy(), np.arange(n), G, P)
    out, lse, _ = attend(q, cache, np.arange(4, dtype=np.int32)[None], [n], G, P, [0, q_len], max_q=q_len)
    nan = torch.isnan(out).cpu()
    want = torch.zeros_like(nan)
    if where == "q":
        want[0, 5] = True
    else:
        want[-1, 4:] = True
    assert torch.equal(nan, want)


@pytest.mark.gpu
@pytest.mark.parametrize("q_len", [1, 24])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size,scale", [(1.0, 40.0), (3000.0, 1e-6), (1e-4, 1.0), (1.0, 1e-30), (60.0, 1.0)])
def test_attention_of_sharp_and_flat_scores(q_len, dtype, size, scale):
    """Scores of thousands, where one key wins, and of nothing, where all weigh the same; large and tiny values."""
    torch_cuda()
    rng = np.random.default_rng(9)
    P, H, D, G, n = 32, 1, 128, 64, 300
    k, v = (values(rng, (n, H, D), dtype, size) for _ in range(2))
    cache = np.zeros((10, H, _kv4.page_bytes(P, D, G)), np.uint8)
    _kv4.write(cache, k.float().numpy(), v.float().numpy(), np.arange(n), G, P)
    q = values(rng, (q_len, 4, D), dtype, size)
    table = np.arange(10, dtype=np.int32)[None]
    out, lse = kv().kv4_attention(q.cuda(), torch.from_numpy(cache).cuda(), torch.from_numpy(table).cuda(),
                                  torch.tensor([n], dtype=torch.int32).cuda(), G, q_start=torch.tensor([0, q_len], dtype=torch.int32).cuda(),
                                  scale=scale, return_lse=True)
    want, want_lse, spread = _kv4.attention(q, cache, table, [n], G, P, [0, q_len], scale=scale)
    # fp32 scores: 2^-21 of the sum of |q k| moves a probability by as much again, times the spread of the values
    mag = scale * float(np.abs(q.double().numpy()).max()) * float(np.abs(_kv4.read(cache, np.arange(n), D, G, P)[0]).max()) * D
    u = 2.0**-11 if dtype == torch.float16 else 2.0**-8
    top = np.abs(_kv4.read(cache, np.arange(n), D, G, P)[1]).max()
    tol = u * np.abs(want) + 2.0**-10 * spread + 2.0**-25 + min(1.0, 2.0**-21 * mag) * top
    got = out.double().cpu().numpy()
    big = np.abs(want) > 65504 if dtype == torch.float16 else np.zeros_like(want, bool)
    assert (np.abs(got - want) <= tol)[~big].all()
    assert (np.abs(lse.double().cpu().numpy() - want_lse) <= 2.0**-16 * (1 + np.abs(want_lse)) + 2.0**-21 * mag).all()


@pytest.mark.gpu
@pytest.mark.parametrize("q_len", [3, 50])
@pytest.mark.parametrize("D,G", SIZES)
@pytest.mark.parametrize("least,most", [(-40, 0), (-9, 3), (-20, 100)])
def test_attention_rows_of_very_different_sizes(q_len, D, G, least, most):
    """One huge query costs the queries that share its workgroup nothing (bf16, whose range is beyond fp16's)."""
    torch_cuda()
    rng = np.random.default_rng(q_len + D + G + most)
    cache, table = filled(rng, [200], 16, 2, D, G, torch.bfloat16)
    size = 2.0 ** rng.integers(least, most + 1, (q_len, 4, 1))
    size[0, 0], size[1, 0] = 2.0**most, 2.0**least
    q = (values(rng, (q_len, 4, D), torch.float32) * torch.from_numpy(size).float()).to(torch.bfloat16)
    out, lse, ref = attend(q, cache, table, [200], G, 16, [0, q_len], max_q=q_len)
    check(out, lse, ref, torch.bfloat16)


@pytest.mark.gpu
@pytest.mark.parametrize("D,G", SIZES)
@pytest.mark.parametrize("Hq,H,P,counts,window", [(8, 1, 16, [2, 2, 1, 2], 0), (8, 1, 64, [3, 1, 3, 0], 0), (16, 2, 64, [4, 4, 4, 4], 600),
                                                  (8, 1, 32, [5, 2, 8, 1], 0), (4, 1, 16, [17, 3, 20, 1], 300)])
def test_attention_shares_of_ragged_sequences(D, G, Hq, H, P, counts, window):
    """8 to 80 rows, with and without sets of them, over contexts that workgroups share: every row once, from all its keys."""
    torch_cuda()
    rng = np.random.default_rng(D + G + sum(counts))
    lens = [1300, 3, 740, 65]
    cache, table = filled(rng, lens, P, H, D, G)
    start = np.concatenate([[0], np.cumsum(counts)])
    q = values(rng, (int(start[-1]), Hq, D), torch.float16)
    out, lse, ref = attend(q, cache, table, lens, G, P, start, max_q=max(counts), window=window)
    check(out, lse, ref, torch.float16)


@pytest.mark.gpu
@pytest.mark.parametrize("q_len", [1, 6, 70])
@pytest.mark.parametrize("D,G", SIZES)
def test_attention_keeps_nan_of_no_weight(q_len, D, G):
    """A value that is no number makes its group NaN for every row that sees it, however little its key weighs, and for no other."""
    torch_cuda()
    rng = np.random.default_rng(q_len + D)
    P, n = 32, 150
    k, v = (values(rng, (n, 1, D), torch.float16) for _ in range(2))
    q = values(rng, (q_len, 2, D), torch.float16)
    at = n - max(1, q_len // 2)                                  # seen by the later rows only
    k[at] = -60 * q[-1, 0]                                       # at least for the last row its weight is 0 in fp32
    v[at, 0, D - 1] = float("nan")
    cache = np.zeros((5, 1, _kv4.page_bytes(P, D, G)), np.uint8)
    _kv4.write(cache, k.float().numpy(), v.float().numpy(), np.arange(n), G, P)
    table = np.arange(5, dtype=np.int32)[None]
    out, _, _ = attend(q, cache, table, [n], G, P, [0, q_len], max_q=q_len)
    sees = np.arange(n - q_len, n)[:, None, None] >= at
    group = np.arange(D) // G == (D - 1) // G
    assert np.array_equal(np.isnan(out.float().cpu().numpy()), np.broadcast_to(sees & group, out.shape))


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["fused", "odd", "heads"])
@pytest.mark.parametrize("q_len", [1, 50])
def test_attention_takes_any_strides(layout, q_len):
    torch_cuda()
    rng = np.random.default_rng(4)
    cache, table = filled(rng, [70], 16, 2, 128, 128)
    q = values(rng, (q_len, 8, 128), torch.float16)
    wide = torch.full((1, 40), -1, dtype=torch.int32).cuda()     # the table, a slice of a wider one at an odd offset
    wide[:, 3:3 + table.shape[1]] = torch.from_numpy(table).cuda()
    args = (torch.from_numpy(cache).cuda(), wide[:, 3:3 + table.shape[1]], torch.tensor([70], dtype=torch.int32).cuda(), 128)
    start = torch.tensor([0, q_len], dtype=torch.int32).cuda()
    out = kv().kv4_attention(laid_out(q, layout), *args, q_start=start, max_q=q_len)
    assert torch.equal(out, kv().kv4_attention(q.cuda(), *args, q_start=start, max_q=q_len))


@pytest.mark.gpu
@pytest.mark.parametrize("n,q_len", [(6000, 1), (20000, 1), (5000, 3), (9000, 40), (4100, 300)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_over_long_contexts(n, q_len, dtype):
    """Contexts long enough to be split over workgroups; the result is the same twice, bit for bit."""
    torch_cuda()
    P, H, D, G = 64, 2, 128, 128
    g = torch.Generator(device="cuda").manual_seed(n)
    cache = kv().kv4_cache(-(-n // P) + 1, P, H, D, G)
    k, v = (torch.randn(n, H, D, device="cuda", generator=g).to(dtype) for _ in range(2))
    kv().kv4_write(cache, k, v, torch.arange(n, device="cuda"), G)
    q = (torch.randn(q_len, 8, D, device="cuda", generator=g) * 1.5).to(dtype)
    table = torch.arange(cache.shape[0], dtype=torch.int32, device="cuda")[None]
    args = (q, cache, table, torch.tensor([n], dtype=torch.int32, device="cuda"), G)
    start = torch.tensor([0, q_len], dtype=torch.int32, device="cuda")
    out, lse = kv().kv4_attention(*args, q_start=start, max_q=q_len, return_lse=True)
    hk, hv = (x.double() for x in kv().kv4_read(cache, torch.arange(n, device="cuda"), D, G, torch.float16))
    x = torch.einsum("ihd,thd->hit", q.double(), hk.repeat_interleave(4, 1)) * D**-0.5
    pos = torch.arange(n - q_len, n, device="cuda")
    x = x.masked_fill(torch.arange(n, device="cuda") > pos[:, None], float("-inf"))
    p = x.softmax(-1)
    ref = (torch.einsum("hit,thd->ihd", p, hv.repeat_interleave(4, 1)), x.logsumexp(-1).t(),
           torch.einsum("hit,thd->ihd", p, hv.abs().repeat_interleave(4, 1)))
    # the values were read back rounded to fp16: 2^-11 of each more, in keys as in values
    want, wl, spread = (t.cpu().numpy() for t in ref)
    check(out, None, (want, wl, spread * 2), dtype)
    again, _ = kv().kv4_attention(*args, q_start=start, max_q=q_len, return_lse=True)
    assert torch.equal(out, again)


@pytest.mark.gpu
@pytest.mark.parametrize("q_len", [1, 40])
def test_cache_past_32_bit_offsets(q_len):
    torch = torch_cuda()
    P, H, D, G, n = 64, 8, 128, 128, 150
    page = _kv4.page_bytes(P, D, G) * H
    pages = (1 << 32) // page + 100
    cache = torch.empty(pages, H, page // H, dtype=torch.uint8, device="cuda")
    table = torch.tensor([[pages - 1, (1 << 31) // page + 1, pages - 40]], dtype=torch.int32, device="cuda")
    small = torch.zeros(3, H, page // H, dtype=torch.uint8, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(1)
    k, v = (torch.randn(n, H, D, device="cuda", generator=g).half() for _ in range(2))
    t = torch.arange(n, device="cuda")
    q = torch.randn(q_len, 32, D, device="cuda", generator=g).half()
    lens, start = torch.tensor([n], dtype=torch.int32, device="cuda"), torch.tensor([0, q_len], dtype=torch.int32, device="cuda")
    got = []
    for c, tab in ((cache, table), (small, torch.arange(3, dtype=torch.int32, device="cuda")[None])):
        slots = tab[0, t // P].long() * P + t % P
        kv().kv4_write(c, k, v, slots, G)
        got.append((*kv().kv4_read(c, slots, D, G), kv().kv4_attention(q, c, tab, lens, G, q_start=start, max_q=q_len)))
    for a, b in zip(*got):
        assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("q_len,n", [(1, 3000), (48, 900)])
def test_other_streams_and_graphs(q_len, n):
    """The calls run on the current stream, and a captured graph replays them on what its inputs then hold."""
    torch = torch_cuda()
    P, H, D, G = 16, 2, 128, 128
    g = torch.Generator(device="cuda").manual_seed(1)
    make = lambda *s: torch.randn(*s, device="cuda", generator=g).half()  # noqa: E731
    k, v, q = make(n, H, D), make(n, H, D), make(q_len, 8, D)
    cache = kv().kv4_cache(-(-n // P), P, H, D, G)
    table = torch.arange(cache.shape[0], dtype=torch.int32, device="cuda")[None]
    lens, start = torch.tensor([n], dtype=torch.int32, device="cuda"), torch.tensor([0, q_len], dtype=torch.int32, device="cuda")
    slots = torch.arange(n, device="cuda")

    def step():
        kv().kv4_write(cache, k, v, slots, G)
        return kv().kv4_attention(q, cache, table, lens, G, q_start=start, max_q=q_len)

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        cache.zero_()
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for i in range(4):
        k.copy_(make(n, H, D))
        q.copy_(make(q_len, 8, D))
        cache.zero_()
        graph.replay()
        torch.cuda.synchronize()
        again = captured.clone()
        cache.zero_()
        assert torch.equal(again, step()), i


@pytest.mark.gpu
@pytest.mark.parametrize("q_len", [1, 40])
def test_rows_of_no_sequence_are_not_written(lib, q_len):
    """Queries before the first sequence's and past the last one's, with whatever the workspace held before."""
    torch = torch_cuda()
    P, H, D, G, n, before, after = 64, 2, 128, 128, 9000, 3, 7
    g = torch.Generator(device="cuda").manual_seed(5)
    cache = kv().kv4_cache(-(-n // P), P, H, D, G)
    k, v = (torch.randn(n, H, D, device="cuda", generator=g).half() for _ in range(2))
    kv().kv4_write(cache, k, v, torch.arange(n, device="cuda"), G)
    q = torch.randn(before + q_len + after, 8, D, device="cuda", generator=g).half()
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    table, lens = torch.arange(cache.shape[0], dtype=torch.int32, device="cuda")[None], i32(n)
    want, want_lse = kv().kv4_attention(q[before:before + q_len], cache, table, lens, G, q_start=i32(0, q_len), max_q=q_len, return_lse=True)
    start, out, lse = i32(before, before + q_len), torch.full_like(q, 7), torch.full(q.shape[:2], 9.0, device="cuda")
    c = Cache(cache.data_ptr(), cache.shape[0], P, H, D, G)
    a = Args(q.data_ptr(), out.data_ptr(), lse.data_ptr(), q.stride(0), q.stride(1), q.shape[0], 8, 1, table.data_ptr(), table.shape[1],
             table.stride(0), lens.data_ptr(), start.data_ptr(), q_len, 0, D**-0.5, 0, 1)
    lim = (ctypes.c_int32 * 4)(256, 163840, 1024, 950)
    size = lib.w4a16_kv4_attention_workspace(ctypes.byref(c), ctypes.byref(a), lim)
    assert size > 0
    workspace, counters = torch.full((size // 4 + 4,), 5, dtype=torch.int32, device="cuda"), torch.zeros(4096, dtype=torch.int32, device="cuda")
    assert lib.w4a16_kv4_attention(ctypes.byref(c), ctypes.byref(a), lim, workspace.data_ptr(), size, counters.data_ptr(),
                                   torch.cuda.current_stream().cuda_stream) == 0, lib.w4a16_last_error()
    torch.cuda.synchronize()
    assert torch.equal(out[before:-after], want) and torch.equal(lse[before:-after], want_lse)
    for rows in (slice(0, before), slice(before + q_len, None)):
        assert (out[rows] == 7).all() and (lse[rows] == 9).all()
    assert (counters == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("q_len", [1, 40, 200])
def test_a_table_much_wider_than_its_sequences(q_len):
    """A table for the longest context that a server allows, 2^26 tokens here, and short sequences."""
    torch_cuda()
    rng = np.random.default_rng(q_len)
    lens, P, H, D, G = [300, 201], 64, 8, 128, 128
    cache, table = filled(rng, lens, P, H, D, G)
    wide = np.full((2, (1 << 26) // P), -1, np.int32)
    wide[:, :table.shape[1]] = table
    q = values(rng, (2 * q_len, 32, D), torch.float16)
    out, lse, ref = attend(q, cache, wide, lens, G, P, [0, q_len, 2 * q_len], max_q=q_len)
    check(out, lse, ref, torch.float16)


@pytest.mark.gpu
def test_attention_of_a_long_prompt():
    """132001 tokens with themselves, 32 heads on 8: rows here and there against 64 bits."""
    torch = torch_cuda()
    n, P, H, D, G = 132001, 64, 8, 64, 64
    g = torch.Generator(device="cuda").manual_seed(2)
    cache = kv().kv4_cache(-(-n // P), P, H, D, G)
    k, v = (torch.randn(n, H, D, device="cuda", generator=g).half() for _ in range(2))
    slots = torch.arange(n, device="cuda")
    kv().kv4_write(cache, k, v, slots, G)
    q = torch.randn(n, 32, D, device="cuda", generator=g).half()
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    out = kv().kv4_attention(q, cache, torch.arange(cache.shape[0], dtype=torch.int32, device="cuda")[None], i32(n), G, q_start=i32(0, n), max_q=n)
    hk, hv = (x.double() for x in kv().kv4_read(cache, slots, D, G, torch.float16))
    for i in (0, 1, 63, 64, 4099, 65535, 65536, 131071, 131072, n - 1):
        for h in (0, 13, 31):
            p = (hk[:i + 1, h // 4] @ q[i, h].double() * D**-0.5).softmax(0)
            want, spread = p @ hv[:i + 1, h // 4], p @ hv[:i + 1, h // 4].abs()
            # the values were read back rounded to fp16: 2^-11 of each more, in keys as in values
            check(out[i, h], None, (want.cpu().numpy(), None, 2 * spread.cpu().numpy()), torch.float16)


@pytest.mark.gpu
def test_empty_calls():
    torch = torch_cuda()
    c = kv().kv4_cache(2, 16, 2, 128, 64)
    none = torch.zeros(0, dtype=torch.int64, device="cuda")
    x = torch.zeros(0, 2, 128, dtype=torch.half, device="cuda")
    kv().kv4_write(c, x, x, none, 64)
    assert (c == 0).all()
    k, v = kv().kv4_read(c, none, 128, 64)
    assert k.shape == v.shape == (0, 2, 128)
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")  # noqa: E731
    assert kv().kv4_attention(x, c, i32(0, 1), i32(0), 64).shape == (0, 2, 128)
    out, lse = kv().kv4_attention(torch.ones(3, 4, 128, device="cuda").half(), c, i32(3, 0), i32(3) + 5, 64, return_lse=True)
    assert (out == 0).all() and torch.isneginf(lse).all()        # no pages at all
    empty = kv().kv4_cache(0, 16, 2, 128, 64)
    kv().kv4_write(empty, x.new_ones(1, 2, 128), x.new_ones(1, 2, 128), none.new_zeros(1), 64)
    k, _ = kv().kv4_read(empty, none.new_zeros(1), 128, 64)
    assert (k == 0).all()


@pytest.mark.gpu
def test_refusals():
    torch = torch_cuda()
    c = kv().kv4_cache(2, 16, 2, 128, 64)
    x = torch.zeros(1, 2, 128, dtype=torch.half, device="cuda")
    s = torch.zeros(1, dtype=torch.int64, device="cuda")
    t, n = torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.ones(1, dtype=torch.int32, device="cuda")
    bad = [(lambda: kv().kv4_write(c, x.float(), x.float(), s, 64), "fp16 or bf16"), (lambda: kv().kv4_write(c, x, x.bfloat16(), s, 64), "same dtype"),
           (lambda: kv().kv4_write(c, x, x[:, :1], s, 64), "same sizes"), (lambda: kv().kv4_write(c, x[:, :1], x[:, :1], s, 64), "heads"),
           (lambda: kv().kv4_write(c, x, x, s.int(), 64), "int64"), (lambda: kv().kv4_write(c, x, x, s.expand(2), 64), "contiguous|tokens"),
           (lambda: kv().kv4_write(c, x, x, s, 32), "unsupported"), (lambda: kv().kv4_write(c, x, x, s, 128), "last size"),
           (lambda: kv().kv4_write(c.transpose(0, 1), x, x, s, 64), "contiguous"), (lambda: kv().kv4_write(c.char(), x, x, s, 64), "uint8"),
           (lambda: kv().kv4_write(c, x.transpose(1, 2).contiguous().transpose(1, 2), x, s, 64), "contiguous in the head"),
           (lambda: kv().kv4_read(c, s, 128, 64, torch.float32), "fp16 or bf16"), (lambda: kv().kv4_read(c, s[None], 128, 64), "slots must be"),
           (lambda: kv().kv4_attention(x.float(), c, t, n, 64), "fp16 or bf16"), (lambda: kv().kv4_attention(x[:, :1], c, t, n, 64), "multiple"),
           (lambda: kv().kv4_attention(x, c, t.long(), n, 64), "int32"), (lambda: kv().kv4_attention(x, c, t, n.expand(2), 64), "block_table"),
           (lambda: kv().kv4_attention(x.expand(2, 2, 128), c, t, n, 64), "one query per sequence"),
           (lambda: kv().kv4_attention(x, c, t, n, 64, q_start=n), "q_start"), (lambda: kv().kv4_attention(x, c, t, n, 64, scale=0.0), "scale"),
           (lambda: kv().kv4_attention(x, c, t, n, 64, scale=float("inf")), "scale"), (lambda: kv().kv4_attention(x, c, t, n, 64, window=-1), "window"),
           (lambda: kv().kv4_attention(x, c, t, n, 64, max_q=-1), "max_q"), (lambda: kv().kv4_attention(x, c[0], t, n, 64), "cache must be")]
    for call, word in bad:
        with pytest.raises(RuntimeError, match=word):
            call()
    assert (c == 0).all()
