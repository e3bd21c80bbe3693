"""Head norm + rotation, the paged KV cache and attention over it, on the device against the 64-bit definitions."""
import ctypes as C
import time

import numpy as np
import pytest

import magnetron_b200 as mb
from magnetron_b200.attention import DeviceArray
from oracle import attention_oracle as A
from oracle import mag_oracle as O
from tests.attention_cases import DTYPES, HALF_STEP, Paged, bits_of, check_attention

pytestmark = pytest.mark.gpu


def raw_bits(t):
    return t.to_bits()


# ---- head norm + rotation -------------------------------------------------------------------------------------------------

def run_norm_rope(gpu, dt, tokens, hq, hk, dim, rotary, interleaved, norm, far, factor=1.0, fused=True, in_place=False, seed=0, pad=0):
    rng = np.random.default_rng(seed)
    width = (hq + 2 * hk) * dim + pad
    buf = bits_of(dt, rng.standard_normal((tokens, width)))
    t = mb.Tensor.from_bits(gpu, dt, buf)
    q = t.as_strided((tokens, hq, dim), (width, dim, 1), pad)
    k = t.as_strided((tokens, hk, dim), (width, dim, 1), pad + hq * dim)
    wq, wk = (bits_of(dt, 1 + 0.3 * rng.standard_normal(dim)) for _ in range(2))
    twq, twk = mb.Tensor.from_bits(gpu, dt, wq), mb.Tensor.from_bits(gpu, dt, wk)
    pos = rng.integers(0, far, tokens).astype(np.int32)
    pos[0] = far - 1
    freq = (1e6 ** (-np.arange(rotary // 2) / max(1, rotary // 2))).astype(np.float32)
    dpos, dfreq = DeviceArray(gpu, pos), DeviceArray(gpu, freq)
    rope = mb.Rope(dpos, dfreq, rotary, interleaved=interleaved, factor=factor) if rotary else None
    outs = mb.qk_norm_rope(q, k, rope, q if in_place else None, k if in_place else None, q_weight=twq if norm else None, k_weight=twk if norm else None, eps=1e-6)
    after = raw_bits(t)
    for got, first, heads, w in ((outs[0], pad, hq, wq), (outs[1], pad + hq * dim, hk, wk)):
        x = O.bits_to_f64(dt, buf[:, first:first + heads * dim].reshape(tokens, heads, dim))
        want, size = A.norm_rope(x, O.bits_to_f64(dt, w) if norm else None, 1e-6, pos, freq, rotary, interleaved, np.float64(np.float32(factor)))
        g = O.bits_to_f64(dt, raw_bits(got))
        # one rounding of the result; the mean of squares, its root and the products: (dim + 32) fp32 roundings of the parts, the
        # sines' errors (angle reduced in fp64, fraction in fp32) among them; half the least subnormal step
        tol = HALF_STEP[dt] * np.abs(want) + (dim + 32) * 2.0 ** -24 * size + 2.0 ** -25 * (dt == mb.FLOAT16)
        assert (np.abs(g - want) <= tol).all(), float((np.abs(g - want) / tol).max())
    if not in_place:
        assert np.array_equal(after, buf)                                # inputs are not touched
    else:
        assert np.array_equal(after[:, :pad], buf[:, :pad])
        assert np.array_equal(after[:, pad + (hq + hk) * dim:], buf[:, pad + (hq + hk) * dim:])   # v beside them neither


@pytest.mark.parametrize("name", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("dim,rotary,interleaved", [(128, 128, False), (128, 128, True), (128, 64, False), (64, 64, False), (80, 40, False),
                                                    (96, 48, True), (256, 256, False), (256, 64, True), (8, 2, False), (64, 22, False), (64, 22, True), (128, 0, False)])
def test_norm_rope_layouts(gpu, name, dim, rotary, interleaved):
    run_norm_rope(gpu, DTYPES[name], 5, 4, 2, dim, rotary, interleaved, True, 40000)


@pytest.mark.parametrize("tokens,hq,hk", [(1, 16, 8), (1, 1, 1), (3, 5, 1), (257, 16, 8), (2000, 7, 3)])
def test_norm_rope_sizes(gpu, tokens, hq, hk):
    run_norm_rope(gpu, mb.BFLOAT16, tokens, hq, hk, 128, 128, False, True, 131072, factor=1.2)
    run_norm_rope(gpu, mb.FLOAT16, tokens, hq, hk, 64, 64, True, False, 1 << 20)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("pad", [0, 1, 3, 8])
def test_norm_rope_alignment_and_in_place(gpu, pad, in_place):
    run_norm_rope(gpu, mb.BFLOAT16, 33, 4, 2, 128, 128, False, True, 5000, pad=pad, in_place=in_place)


def test_norm_rope_far_positions_and_rows_of_extremes(gpu):
    run_norm_rope(gpu, mb.FLOAT32, 64, 2, 1, 64, 64, False, False, 2 ** 31 - 1)
    # a row of zeros stays zero (eps keeps the root finite), a NaN stays in its row, without a rotation beside the norm
    x = np.zeros((3, 2, 64), np.float32)
    x[1, 1, 5] = np.nan
    x[2, 0] = 3e18                                                        # squares sum to about 6e38 / 64: past the fp32 range
    t = mb.Tensor.from_bits(gpu, mb.FLOAT32, bits_of(mb.FLOAT32, x))
    w = mb.Tensor.from_bits(gpu, mb.FLOAT32, bits_of(mb.FLOAT32, np.ones(64)))
    out, none = mb.qk_norm_rope(t, None, None, q_weight=w)
    got = out.to_bits().view(np.float32)
    assert none is None and (got[0] == 0).all() and (got[1, 0] == 0).all() and np.isnan(got[1, 1]).all()


# ---- the cache, written and read ------------------------------------------------------------------------------------------

def write_and_check(gpu, dt, bits, q_lens, kv_lens, *, kv_heads, dim, page, pad_rows=0, strided=True, offset=0, spread=1.0, seed=0):
    p = Paged(gpu, dt, bits, q_lens, kv_lens, kv_heads=kv_heads, dim=dim, page=page, seed=seed)
    rng = np.random.default_rng(seed + 1)
    tokens = sum(q_lens) + pad_rows
    width = 2 * kv_heads * dim + offset
    x = rng.standard_normal((tokens, width)) * np.exp(spread * rng.standard_normal((tokens, 1)))
    if dt == mb.FLOAT16:
        x = np.clip(x, -65504, 65504)
    buf = bits_of(dt, x)
    t = mb.Tensor.from_bits(gpu, dt, buf)
    k = t.as_strided((tokens, kv_heads, dim), (width, dim, 1), offset)
    v = t.as_strided((tokens, kv_heads, dim), (width, dim, 1), offset + kv_heads * dim)
    want = {(n, "pool"): p.pool[n].copy() for n in ("k", "v")} | {(n, "exps"): p.exps[n].copy() for n in p.exps}
    at = 0
    for b, n in enumerate(q_lens):
        for i in range(n):
            pos = kv_lens[b] - n + i
            if pos >= 0:
                page_id, slot = p.tables[b][pos // page], pos % page
                for j, name in enumerate(("k", "v")):
                    row = buf[at + i, offset + j * kv_heads * dim:offset + (j + 1) * kv_heads * dim].reshape(kv_heads, dim)
                    if bits == 8:
                        codes, exps = A.quantise(O.bits_to_f64(dt, row), dt)
                        want[name, "pool"][page_id, :, slot], want[name, "exps"][page_id, :, slot] = codes, exps
                    else:
                        want[name, "pool"][page_id, :, slot] = row
        at += n
    mb.kv_cache_write(p.cache, p.batch, k, v)
    mb.synchronize(gpu)
    got = p.download()
    for key, w in want.items():                                           # bit for bit, all other rows as they were
        assert np.array_equal(got[key], w), (key, np.argwhere(got[key] != w)[:4].tolist())


@pytest.mark.parametrize("name", ["bf16", "fp16"])
@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("kv_heads,dim,page", [(1, 64, 16), (8, 128, 16), (3, 80, 32), (2, 96, 64), (1, 256, 16), (12, 16, 128)])
def test_cache_write(gpu, name, bits, kv_heads, dim, page):
    write_and_check(gpu, DTYPES[name], bits, [1, 0, 37, 5, 1], [20, 7, 37, 3, 257], kv_heads=kv_heads, dim=dim, page=page, pad_rows=3, spread=2.0)


@pytest.mark.parametrize("offset", [0, 1, 8])
def test_cache_write_alignment(gpu, offset):
    for bits in (16, 8):
        write_and_check(gpu, mb.BFLOAT16, bits, [1] * 70, list(range(1, 71)), kv_heads=2, dim=128, page=16, offset=offset)


def test_cache_write_many_sequences(gpu):
    q = [1 + (i * 7) % 3 for i in range(1300)]                            # three levels of the search for a token's sequence
    write_and_check(gpu, mb.BFLOAT16, 8, q, [n + (i % 5) for i, n in enumerate(q)], kv_heads=1, dim=64, page=16)
    write_and_check(gpu, mb.FLOAT16, 16, [9000], [9000], kv_heads=2, dim=64, page=64)


@pytest.mark.parametrize("name", ["bf16", "fp16"])
def test_eight_bit_rows_of_every_kind(gpu, name):
    """Every finite 16-bit pattern in a row of its own, with zeros, and beside a larger one; infinities and NaN."""
    dt = DTYPES[name]
    patterns = np.arange(65536, dtype=np.uint16)
    rows = np.zeros((2 * 65536, 1, 16), np.uint16)
    rows[:65536, 0, 3] = patterns
    rows[65536:, 0, 0] = patterns
    rows[65536:, 0, 9] = np.roll(patterns, 977)
    n = rows.shape[0]
    p = Paged(gpu, dt, 8, [n], [n], kv_heads=1, dim=16, page=1024)
    t = mb.Tensor.from_bits(gpu, dt, rows)
    mb.kv_cache_write(p.cache, p.batch, t, t)
    got = p.download()
    with np.errstate(invalid="ignore"):
        codes, exps = A.quantise(O.bits_to_f64(dt, rows), dt)
    pos = np.arange(n)
    at = np.asarray(p.tables[0])[pos // 1024], slice(None), pos % 1024
    assert np.array_equal(got["k", "exps"][at], exps) and np.array_equal(got["k", "pool"][at], codes)
    # read back: exactly code * 2^e in the type; every finite row stays finite
    cu = DeviceArray(gpu, np.array([0, n], np.int32))
    k, v = mb.Tensor(gpu, dt, rows.shape), mb.Tensor(gpu, dt, rows.shape)
    mb.kv_cache_read(p.cache, p.batch, cu, k, v)
    back = O.bits_to_f64(dt, k.to_bits())
    want = O.bits_to_f64(dt, bits_of(dt, A.dequantise(codes, exps)))
    finite = np.isfinite(O.bits_to_f64(dt, rows)).all(-1)
    assert np.array_equal(back[finite], want[finite]) and np.isfinite(back[finite]).all() and np.isnan(back[~finite]).all()


@pytest.mark.parametrize("name", ["bf16", "fp16"])
@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("kv_heads,dim,page", [(1, 64, 16), (8, 128, 32), (3, 80, 16), (1, 256, 64)])
def test_cache_read(gpu, name, bits, kv_heads, dim, page):
    dt = DTYPES[name]
    kv = [1, 0, 33, 16, 400]
    p = Paged(gpu, dt, bits, [1] * 5, kv, kv_heads=kv_heads, dim=dim, page=page, seed=3)
    take = [1, 0, 20, 16, 400]                                            # the third sequence only in part
    cu = DeviceArray(gpu, np.concatenate([[0], np.cumsum(take)]).astype(np.int32))
    rows = sum(take) + 4                                                  # rows behind the last sequence stay as they were
    before = np.full((rows, 2 * kv_heads * dim + 8), 0x1234, np.uint16)
    t = mb.Tensor.from_bits(gpu, dt, before)
    w = before.shape[1]
    k, v = t.as_strided((rows, kv_heads, dim), (w, dim, 1), 0), t.as_strided((rows, kv_heads, dim), (w, dim, 1), kv_heads * dim)
    mb.kv_cache_read(p.cache, p.batch, cu, k, v)
    after = t.to_bits()
    want = before.copy()
    at = 0
    for b, n in enumerate(take):
        for j, side in enumerate(("k", "v")):
            want[at:at + n, j * kv_heads * dim:(j + 1) * kv_heads * dim] = bits_of(dt, p.rows(side, b, n)).reshape(n, kv_heads * dim)
        at += n
    assert np.array_equal(after, want)


# ---- attention ------------------------------------------------------------------------------------------------------------

def attend(gpu, p, heads, *, scale=None, causal=True, window=0, seed=5, lse=True, fused=False, pad_rows=0, q_scale=1.0, check=True):
    rng = np.random.default_rng(seed)
    tokens = sum(p.q_lens) + pad_rows
    width = heads * p.dim + (64 if fused else 0)
    qb = bits_of(p.dtype, rng.standard_normal((tokens, width)) * q_scale)
    t = mb.Tensor.from_bits(gpu, p.dtype, qb)
    q = t.as_strided((tokens, heads, p.dim), (width, p.dim, 1), 32 if fused else 0)
    out = mb.Tensor.from_bits(gpu, p.dtype, np.full((tokens, heads, p.dim), 0x1234, np.uint16))
    l = mb.Tensor.from_bits(gpu, mb.FLOAT32, np.full((tokens, heads), 0x41414141, np.uint32)) if lse else None
    mb.paged_attention(q, p.cache, p.batch, out, lse=l, scale=scale, causal=causal, window=window)
    got = out.to_bits()
    mb.synchronize(gpu)
    off = 32 if fused else 0
    qh = qb[:, off:off + heads * p.dim].reshape(tokens, heads, p.dim)
    gl = l.to_bits().view(np.float32) if lse else None
    n = sum(p.q_lens)
    if check:
        assert (got[n:] == 0x1234).all()                                  # rows behind the last sequence belong to nobody
        check_attention(p, qh, got, None if gl is None else gl.astype(np.float64), scale=scale, causal=causal, window=window)
    return qh, got, gl


SHAPES = {
    "decode": ([1, 1, 1, 1], [1, 16, 17, 300]),
    "empty": ([1, 0, 2, 0, 1], [0, 0, 40, 9, 31]),
    "few": ([2, 4, 3], [50, 4, 129]),
    "short_cache": ([5, 3, 40], [2, 0, 17]),                              # more new tokens than cached ones: rows that see nothing
    "prompts": ([33, 130, 1, 64], [33, 130, 1, 64]),
    "chunk": ([70, 1, 128], [400, 257, 128]),
}


@pytest.mark.parametrize("name", ["bf16", "fp16"])
@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("shape", list(SHAPES))
@pytest.mark.parametrize("heads,kv_heads,dim,page", [(4, 2, 64, 16), (8, 1, 128, 32)])
def test_attention_shapes(gpu, name, bits, shape, heads, kv_heads, dim, page):
    q, kv = SHAPES[shape]
    p = Paged(gpu, DTYPES[name], bits, q, kv, kv_heads=kv_heads, dim=dim, page=page, seed=11)
    attend(gpu, p, heads, pad_rows=2)


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("dim", [16, 32, 48, 64, 80, 96, 112, 128])
def test_attention_head_dims(gpu, bits, dim):
    p = Paged(gpu, mb.BFLOAT16, bits, [1, 3, 90], [77, 30, 200], kv_heads=2, dim=dim, page=16, seed=dim)
    attend(gpu, p, 6, fused=True)
    p = Paged(gpu, mb.FLOAT16, bits, [1, 1], [77, 30], kv_heads=2, dim=dim, page=32, seed=dim)
    attend(gpu, p, 6)


@pytest.mark.parametrize("group", [1, 2, 3, 5, 7, 8, 16, 33])
def test_attention_groups(gpu, group):
    p = Paged(gpu, mb.BFLOAT16, 16, [1, 2, 50], [200, 2, 90], kv_heads=2, dim=64, page=16, seed=group)
    attend(gpu, p, 2 * group)
    p = Paged(gpu, mb.FLOAT16, 8, [1, 1], [200, 65], kv_heads=1, dim=128, page=16, seed=group)
    attend(gpu, p, group)


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("window", [1, 7, 16, 100, 128, 1000])
def test_attention_window(gpu, bits, window):
    p = Paged(gpu, mb.BFLOAT16, bits, [1, 1, 150, 4], [300, 5, 400, 260], kv_heads=2, dim=64, page=16, seed=window)
    attend(gpu, p, 4, window=window)
    p = Paged(gpu, mb.BFLOAT16, bits, [1, 1], [2300, 1], kv_heads=1, dim=128, page=64, seed=window)
    attend(gpu, p, 4, window=window)


@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31, 2 ** 62, 2 ** 63 - 1])
@pytest.mark.parametrize("q_lens,kv_lens", [([1, 1], [700, 90]), ([60], [300])])
def test_attention_windows_beyond_all_positions(gpu, window, q_lens, kv_lens):
    p = Paged(gpu, mb.BFLOAT16, 16, q_lens, kv_lens, kv_heads=2, dim=64, page=16, seed=2)
    q = mb.Tensor.from_bits(gpu, mb.BFLOAT16, bits_of(mb.BFLOAT16, np.random.default_rng(2).standard_normal((sum(q_lens), 4, 64))))
    want = mb.paged_attention(q, p.cache, p.batch).to_bits()
    assert np.array_equal(mb.paged_attention(q, p.cache, p.batch, window=window).to_bits(), want)


@pytest.mark.parametrize("bits", [16, 8])
def test_attention_to_all_cached_rows(gpu, bits):
    """Without the causal mask: any number of new tokens over any number of cached ones (cross attention)."""
    p = Paged(gpu, mb.FLOAT16, bits, [1, 200, 3, 7], [130, 60, 0, 512], kv_heads=2, dim=64, page=16, seed=2)
    attend(gpu, p, 4, causal=False)


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("page", [16, 64, 512])
def test_attention_long_caches_are_split(gpu, bits, page):
    p = Paged(gpu, mb.BFLOAT16, bits, [1, 1, 2], [9001, 300, 4100], kv_heads=1, dim=128, page=page, seed=4)
    attend(gpu, p, 8)
    p = Paged(gpu, mb.FLOAT16, bits, [40, 1], [6000, 33], kv_heads=1, dim=64, page=page, seed=4)
    attend(gpu, p, 4)


@pytest.mark.parametrize("bits,dim", [(16, 64), (8, 128)])
@pytest.mark.parametrize("window", [0, 90])
def test_attention_more_pieces_of_work_than_multiprocessors(gpu, bits, dim, window):
    """Sequences of one and of two tiles, short and long, none and one new token: every CTA takes several of them in turn."""
    rng = np.random.default_rng(4)
    q = [int(n) for n in rng.integers(20, 330, 60)]
    q[7], q[31], q[32] = 0, 1, 1
    kv = [n + int(x) for n, x in zip(q, rng.integers(0, 300, 60))]
    kv[3], kv[40] = 10, 0
    p = Paged(gpu, mb.BFLOAT16, bits, q, kv, kv_heads=4, dim=dim, page=16, seed=12)
    attend(gpu, p, 8, window=window)


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("q_lens,kv_lens,heads,kv_heads,causal,window", [
    ([1200], [1200], 1, 1, True, 0),                        # rows of a tile that end before its last part begins
    ([1300], [1900], 1, 1, True, 0),
    ([200], [3300], 8, 1, True, 0),                         # 7 units: many parts each
    ([330, 1, 40, 700], [2500, 900, 4000, 1400], 6, 2, True, 0),
    ([330, 1, 40, 700], [2500, 900, 4000, 1400], 6, 2, False, 0),
    ([900, 60], [2600, 3000], 2, 2, True, 1500),
    ([64] * 20, [1500] * 20, 16, 4, True, 0),               # 80 units of one round
    ([50] * 25, [1300] * 25, 32, 8, True, 0),               # a round and a rest
])
def test_attention_units_in_parts(gpu, bits, q_lens, kv_lens, heads, kv_heads, causal, window):
    p = Paged(gpu, mb.BFLOAT16, bits, q_lens, kv_lens, kv_heads=kv_heads, dim=64, page=32, seed=len(q_lens) + kv_lens[0])
    attend(gpu, p, heads, causal=causal, window=window)


def test_attention_pieces_longer_than_the_wait_limit(gpu):
    """The limit is on waits for something that does not come, not on how long a sequence may be."""
    L = mb.lib()
    p = Paged(gpu, mb.BFLOAT16, 16, [9600], [90000], kv_heads=8, dim=16, page=64, seed=6)
    q = mb.Tensor.from_bits(gpu, mb.BFLOAT16, bits_of(mb.BFLOAT16, np.random.default_rng(6).standard_normal((9600, 8, 16))))
    want = mb.paged_attention(q, p.cache, p.batch).to_bits()
    old = L.magb200_get_wait_limit_ns()
    mb.check(L.magb200_set_wait_limit_ns(1_000_000))
    try:
        assert np.array_equal(mb.paged_attention(q, p.cache, p.batch).to_bits(), want)
    finally:
        mb.check(L.magb200_set_wait_limit_ns(old))


@pytest.mark.parametrize("bits", [16, 8])
def test_attention_scales_and_sharp_rows(gpu, bits):
    """A negative scale, no scale at all, and scores so far apart that one weight takes all."""
    p = Paged(gpu, mb.BFLOAT16, bits, [1, 20, 140], [500, 20, 300], kv_heads=2, dim=64, page=16, seed=6)
    for scale, q_scale in ((-0.2, 1.0), (0.0, 1.0), (0.125, 30.0)):
        attend(gpu, p, 4, scale=scale, q_scale=q_scale)


@pytest.mark.parametrize("name,k_scale,v_scale", [("bf16", 1e-20, 1e30), ("bf16", 1.0, 1e-30), ("bf16", 1.0, 3e5), ("fp16", 1e-3, 1e3), ("fp16", 1.0, 1e-5), ("fp16", 1.0, 8e3)])
@pytest.mark.parametrize("bits", [16, 8])
def test_attention_ranges_of_rows(gpu, name, k_scale, v_scale, bits):
    """Rows far from one, where 8-bit exponents reach past what one factor of the type can hold."""
    p = Paged(gpu, DTYPES[name], bits, [1, 5, 130], [100, 60, 160], kv_heads=1, dim=64, page=16, seed=8, k_scale=k_scale, v_scale=v_scale)
    attend_relative(gpu, p, 2, v_scale)


def attend_relative(gpu, p, heads, v_scale):
    qh, got, lse = attend(gpu, p, heads, check=False)
    g = O.bits_to_f64(p.dtype, got)
    q = O.bits_to_f64(p.dtype, qh)
    u = HALF_STEP[p.dtype]
    at = 0
    for b, n in enumerate(p.q_lens):
        out, _, spread, size = A.attention(q[at:at + n], p.rows("k", b), p.rows("v", b), p.dim ** -0.5, True, 0)
        weight = 2 * p.dim * 2.0 ** -24 * size + 2.0 ** -22 + p.kv_lens[b] * 2.0 ** -24
        # as check_attention, and in fp16 weights under 2^-14 and results under 2^-14 are rounded to multiples of 2^-24
        largest = np.abs(p.rows("v", b)).max()
        small = 2.0 ** -25 * (1 + p.kv_lens[b] * min(largest, 65504.0)) if p.dtype == mb.FLOAT16 else 0.0
        tol = u * np.abs(out) + (u + 2 * weight[..., None]) * spread + small
        # rows of 8e3 in fp16 hold some infinities (a value past 65504): 0 * inf is NaN for every row of the definition above, while
        # the kernel may leave a column finite whose infinity no row sees; all other elements are held to the bound
        fine = np.isfinite(out) & np.isfinite(tol)
        err = np.abs(g[at:at + n] - out)
        assert (err[fine] <= tol[fine]).all(), (b, float((err / tol)[fine].max()))
        assert fine.all() or not np.isfinite(largest)
        at += n


@pytest.mark.parametrize("bits", [16, 8])
def test_attention_rows_at_the_top_of_fp16(gpu, bits):
    """V rows up to 65504, whose exponent (8) one fp16 factor cannot hold; few and many rows."""
    p = Paged(gpu, mb.FLOAT16, bits, [1, 5, 130], [100, 60, 160], kv_heads=1, dim=64, page=16, seed=8, v_scale=8e3, clip=65504.0)
    assert np.abs(p.rows("v", 0)).max() > 57344
    attend_relative(gpu, p, 2, 8e3)


@pytest.mark.parametrize("bits", [16, 8])
def test_sequences_share_pages(gpu, bits):
    p = Paged(gpu, mb.BFLOAT16, bits, [1, 2, 90], [100, 120, 190], kv_heads=2, dim=64, page=16, seed=9, share=5)
    attend(gpu, p, 4)


def test_results_repeat_bit_for_bit(gpu):
    p = Paged(gpu, mb.BFLOAT16, 8, [1, 1, 300], [9000, 700, 2000], kv_heads=1, dim=128, page=32, seed=1)
    first = attend(gpu, p, 8)
    for _ in range(3):
        again = attend(gpu, p, 8, check=False)
        assert np.array_equal(first[1], again[1]) and np.array_equal(first[2], again[2])


@pytest.mark.parametrize("bits", [16, 8])
def test_nan_keys_reach_only_the_rows_that_see_them(gpu, bits):
    """K of one cached token is NaN: rows before it are untouched by it, it and later rows are NaN."""
    p = Paged(gpu, mb.BFLOAT16, bits, [200], [200], kv_heads=1, dim=64, page=16, seed=3)
    clean = attend(gpu, p, 2)
    page, slot = p.tables[0][77 // 16], 77 % 16
    if bits == 8:
        p.exps["k"][page, 0, slot] = A.NAN_EXPONENT
        p.pool["k"][page, 0, slot] = 0
    else:
        p.pool["k"][page, 0, slot, 7] = 0x7FFF
    p.upload()
    hit = attend(gpu, p, 2, check=False)
    assert np.array_equal(hit[1][:77], clean[1][:77]) and np.isnan(O.bits_to_f64(mb.BFLOAT16, hit[1][77:])).all()


def test_bad_pages_and_offsets_are_reported_not_followed(gpu):
    """The kernels check what they read from device memory: bad entries are skipped and reported, the device stays usable."""
    for field in ("pages", "cu_q", "kv_len"):
        p = Paged(gpu, mb.BFLOAT16, 16, [3, 40], [90, 100], kv_heads=2, dim=64, page=16, seed=5)
        if field == "pages":
            p.tables[1][2], p.tables[0][0] = 10 ** 6, -7
        q = [3, 40] if field != "cu_q" else [3, 400]
        kv = [90, 100] if field != "kv_len" else [90, 10 ** 6]
        p.batch = mb.KVBatch.from_lists(gpu, q, kv, p.tables)
        p.batch.struct.max_q = 40
        qt = mb.Tensor.from_bits(gpu, mb.BFLOAT16, np.zeros((43, 4, 64), np.uint16))
        out = mb.paged_attention(qt, p.cache, p.batch)
        with pytest.raises(mb.MagB200Error) as e:
            mb.synchronize(gpu)
        assert e.value.code == mb.ERR_INVALID_ARG and "paged cache" in str(e.value)
        mb.synchronize(gpu)                                               # reported once
        if field != "cu_q":
            kt = mb.Tensor.from_bits(gpu, mb.BFLOAT16, np.zeros((43, 2, 64), np.uint16))
            before = p.download()
            mb.kv_cache_write(p.cache, p.batch, kt, kt)
            if field == "kv_len":
                with pytest.raises(mb.MagB200Error):
                    mb.synchronize(gpu)
                after = p.download()
                assert np.array_equal(before["k", "pool"][p.tables[1]], after["k", "pool"][p.tables[1]])
            else:
                mb.synchronize(gpu)                                       # the write touches only the sound last pages
        del out
        good = Paged(gpu, mb.BFLOAT16, 16, [3, 40], [90, 100], kv_heads=2, dim=64, page=16, seed=5)
        attend(gpu, good, 4)


def test_lengths_that_no_memory_holds_are_reported(gpu):
    """32 sequences of 2^31 rows each by way of one page: their groups of 16 rows are 2^32, more than a call walks."""
    n, page, width = 32, 1 << 20, 2047
    cache = mb.KVCache(gpu, mb.BFLOAT16, 1, page, 1, 16)
    batch = mb.KVBatch(n, width, cu_q=DeviceArray(gpu, np.arange(n + 1, dtype=np.int32)), kv_len=DeviceArray(gpu, np.full(n, width * page, np.int32)),
                       pages=DeviceArray(gpu, np.zeros((n, width), np.int32)), max_q=1)
    q = mb.Tensor.from_bits(gpu, mb.BFLOAT16, np.zeros((n, 1, 16), np.uint16))
    out = mb.Tensor.from_bits(gpu, mb.BFLOAT16, np.full((n, 1, 16), 0x1234, np.uint16))
    mb.paged_attention(q, cache, batch, out)
    with pytest.raises(mb.MagB200Error) as e:
        mb.synchronize(gpu)
    assert e.value.code == mb.ERR_INVALID_ARG
    assert (out.to_bits() == 0x1234).all()


def test_recorded_calls_follow_the_lengths_in_memory(gpu):
    """A graph of write + attention replayed while the sequences grow, beside eager calls and a second graph."""
    dt, heads, hk, dim, page = mb.BFLOAT16, 4, 2, 64, 16
    p = Paged(gpu, dt, 8, [1, 1], [700, 100], kv_heads=hk, dim=dim, page=page, seed=7)
    lens = [600, 20]
    kv_len, cu = DeviceArray(gpu, np.asarray(lens, np.int32)), DeviceArray(gpu, np.array([0, 1, 2], np.int32))
    table = np.zeros((2, 44), np.int32)
    for b in range(2):
        table[b, :len(p.tables[b])] = p.tables[b]
    dtable = DeviceArray(gpu, table)
    batch = mb.KVBatch(2, 44, cu_q=cu, kv_len=kv_len, pages=dtable, max_q=1, max_kv=700)
    p.batch = batch
    rng = np.random.default_rng(1)
    qb, kvb = bits_of(dt, rng.standard_normal((2, heads, dim))), bits_of(dt, rng.standard_normal((2, 2 * hk, dim)))
    q, kv = mb.Tensor.from_bits(gpu, dt, qb), mb.Tensor.from_bits(gpu, dt, kvb)
    k, v = kv.as_strided((2, hk, dim), (2 * hk * dim, dim, 1), 0), kv.as_strided((2, hk, dim), (2 * hk * dim, dim, 1), hk * dim)
    out, out2 = mb.Tensor(gpu, dt, (2, heads, dim)), mb.Tensor(gpu, dt, (2, heads, dim))
    mb.paged_attention(q, p.cache, batch, out)
    mb.synchronize(gpu)
    L, graphs = mb.lib(), []
    for o in (out, out2):
        mb.check(L.magb200_graph_begin_capture(gpu))
        mb.kv_cache_write(p.cache, batch, k, v)
        mb.paged_attention(q, p.cache, batch, o)
        g = C.c_void_p()
        mb.check(L.magb200_graph_end_capture(gpu, C.byref(g)))
        graphs.append(g)
    for step in range(3):
        kv_len.update(np.asarray([n + 1 + 33 * step for n in lens], np.int32))
        mb.check(L.magb200_graph_launch(gpu, graphs[0]))
        mb.check(L.magb200_graph_launch(gpu, graphs[1]))
        eager = mb.paged_attention(q, p.cache, batch)
        got = out.to_bits()
        p.kv_lens = [n + 1 + 33 * step for n in lens]
        down = p.download()
        p.pool, p.exps = {n: down[n, "pool"] for n in ("k", "v")}, {n: down[n, "exps"] for n in ("k", "v")}
        check_attention(p, qb, got)
        assert np.array_equal(got, out2.to_bits()) and np.array_equal(got, eager.to_bits())
    for g in graphs:
        mb.check(L.magb200_graph_destroy(g))


def test_first_call_cannot_be_recorded_before_the_workspace_exists(gpu):
    """After a shutdown the device has no workspace: recording refuses, an eager call makes it, recording then works."""
    L = mb.lib()
    mb.check(L.magb200_device_shutdown(gpu))
    mb.check(L.magb200_device_init(gpu))
    p = Paged(gpu, mb.BFLOAT16, 16, [1], [40], kv_heads=1, dim=64, page=16)
    q = mb.Tensor.from_bits(gpu, mb.BFLOAT16, np.zeros((1, 2, 64), np.uint16))
    out = mb.Tensor(gpu, mb.BFLOAT16, (1, 2, 64))
    mb.check(L.magb200_graph_begin_capture(gpu))
    with pytest.raises(mb.MagB200Error) as e:
        mb.paged_attention(q, p.cache, p.batch, out)
    g = C.c_void_p()
    mb.check(L.magb200_graph_end_capture(gpu, C.byref(g)))
    mb.check(L.magb200_graph_destroy(g))
    assert "once before" in str(e.value)
    attend(gpu, p, 2)


@pytest.mark.parametrize("tokens", [1, 200])
def test_operators_keep_their_place_between_matmuls(gpu, tokens):
    """Runs of matmuls that may overlap one another, the operators right behind and before them, without a wait in between; results
    that the next matmul takes as its weight among them. Against the same calls with a wait after each."""
    dt, heads, hk, dim, page = mb.BFLOAT16, 8, 8, 64, 16
    width = heads * dim
    rng = np.random.default_rng(tokens)
    x = mb.Tensor.from_bits(gpu, dt, bits_of(dt, rng.standard_normal((tokens, 2048))))
    ws = [mb.Tensor.from_bits(gpu, dt, bits_of(dt, rng.standard_normal((2048, width)) * 0.02)) for _ in range(3)]
    p = Paged(gpu, dt, 16, [tokens], [tokens + 40], kv_heads=hk, dim=dim, page=page, seed=3)
    dpos, dfreq = DeviceArray(gpu, np.arange(tokens, dtype=np.int32)), DeviceArray(gpu, np.ones(dim // 2, np.float32))
    rope, cu = mb.Rope(dpos, dfreq, dim), DeviceArray(gpu, np.array([0, tokens + 40], np.int32))

    def run(wait):
        results = []
        for _ in range(4):
            q, k, v = ((x @ w).view((tokens, heads, dim)) for w in ws)
            wait()
            mb.qk_norm_rope(q, k, rope, q, k)
            wait()
            mb.kv_cache_write(p.cache, p.batch, k, v)
            wait()
            o = mb.paged_attention(q, p.cache, p.batch)
            wait()
            y = o.view((tokens, width)) @ ws[0].T                              # the attention's result as x
            z = ws[1] @ o.view((tokens, width)).T      # and as the weight
            wait()
            rk, rv = mb.Tensor(gpu, dt, (tokens + 40, hk, dim)), mb.Tensor(gpu, dt, (tokens + 40, hk, dim))
            mb.kv_cache_read(p.cache, p.batch, cu, rk, rv)
            wait()
            s = o.view((tokens, width)) @ rk.view((tokens + 40, width)).T      # rows of the cache as the weight
            results += [y, z, s]
        return [t.to_bits() for t in results]

    want = run(lambda: mb.synchronize(gpu))
    got = run(lambda: None)
    assert all(np.array_equal(a, b) for a, b in zip(want, got))


def test_on_a_stream_of_the_callers(gpu):
    torch = pytest.importorskip("torch")
    p = Paged(gpu, mb.BFLOAT16, 8, [40, 1], [90, 100], kv_heads=2, dim=64, page=16, seed=4)
    q = mb.Tensor.from_bits(gpu, mb.BFLOAT16, bits_of(mb.BFLOAT16, np.random.default_rng(4).standard_normal((41, 4, 64))))
    want = mb.paged_attention(q, p.cache, p.batch).to_bits()
    stream = torch.cuda.Stream(gpu)
    mb.check(mb.lib().magb200_set_stream(gpu, stream.cuda_stream))
    try:
        out = mb.paged_attention(q, p.cache, p.batch)
        stream.synchronize()
        assert np.array_equal(out.to_bits(), want)
    finally:
        mb.check(mb.lib().magb200_set_stream(gpu, None))


# ---- a run of them as a layer uses them -----------------------------------------------------------------------------------

@pytest.mark.parametrize("bits", [16, 8])
def test_a_layers_attention_block_prompt_then_tokens(gpu, bits):
    """Grouped q/k/v projection, head norm + rotation in place, cache write, attention and the output projection: two prompts, then
    single tokens. Each step is checked against the 64-bit definition of the same inputs as it found them on the device."""
    dt, hidden, heads, hk, dim, page = mb.BFLOAT16, 256, 4, 2, 64, 16
    rng = np.random.default_rng(0)
    weights = [mb.Tensor.from_bits(gpu, dt, bits_of(dt, rng.standard_normal((n * dim, hidden)) * 0.06)) for n in (heads, hk, hk)]
    wo = mb.Tensor.from_bits(gpu, dt, bits_of(dt, rng.standard_normal((hidden, heads * dim)) * 0.06))
    gains = [mb.Tensor.from_bits(gpu, dt, bits_of(dt, 1 + 0.1 * rng.standard_normal(dim))) for _ in range(2)]
    freq = (1e4 ** (-np.arange(dim // 2) / (dim // 2))).astype(np.float32)
    dfreq = DeviceArray(gpu, freq)
    p = Paged(gpu, dt, bits, [1, 1], [120, 60], kv_heads=hk, dim=dim, page=page, seed=1)
    done = [0, 0]
    for q_lens in ([70, 9], [1, 1], [1, 0], [3, 1]):
        kv_lens = [d + n for d, n in zip(done, q_lens)]
        tokens = sum(q_lens)
        x = mb.Tensor.from_bits(gpu, dt, bits_of(dt, rng.standard_normal((tokens, hidden))))
        outs = [mb.Tensor(gpu, dt, (tokens, w.shape[0])) for w in weights]
        ys = [w.T.view_struct() for w in weights]
        rs = [o.view_struct() for o in outs]
        arr = C.POINTER(mb.View) * 3
        mb.check(mb.lib().magb200_matmul_grouped(gpu, C.byref(x.view_struct()), 3, arr(*[C.pointer(y) for y in ys]), arr(*[C.pointer(r) for r in rs])))
        q, k, v = (o.view((tokens, n, dim)) for o, n in zip(outs, (heads, hk, hk)))
        pos = np.concatenate([np.arange(d, d + n) for d, n in zip(done, q_lens)]).astype(np.int32)
        dpos = DeviceArray(gpu, pos)
        raw = [O.bits_to_f64(dt, t.to_bits()) for t in (q, k)]
        mb.qk_norm_rope(q, k, mb.Rope(dpos, dfreq, dim), q, k, q_weight=gains[0], k_weight=gains[1])
        for t, r, g in ((q, raw[0], gains[0]), (k, raw[1], gains[1])):
            want, size = A.norm_rope(r, O.bits_to_f64(dt, g.to_bits()), 1e-6, pos, freq, dim, False, 1.0)
            got = O.bits_to_f64(dt, t.to_bits())
            assert (np.abs(got - want) <= HALF_STEP[dt] * np.abs(want) + (dim + 32) * 2.0 ** -24 * size).all()
        p.q_lens, p.kv_lens = q_lens, kv_lens
        p.batch = mb.KVBatch.from_lists(gpu, q_lens, kv_lens, p.tables)
        mb.kv_cache_write(p.cache, p.batch, k, v)
        o = mb.paged_attention(q, p.cache, p.batch)
        y = o.view((tokens, heads * dim)) @ wo.T
        down = p.download()
        p.pool = {n: down[n, "pool"] for n in ("k", "v")}
        p.exps = {n: down[n, "exps"] for n in ("k", "v")} if bits == 8 else {}
        check_attention(p, q.to_bits(), o.to_bits())
        ob = O.bits_to_f64(dt, o.to_bits()).reshape(tokens, -1)
        wf = O.bits_to_f64(dt, wo.to_bits())
        assert (np.abs(O.bits_to_f64(dt, y.to_bits()) - ob @ wf.T) <= (2.0 ** -8 + heads * dim * 2.0 ** -24) * (np.abs(ob) @ np.abs(wf).T)).all()
        done = kv_lens


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("q_lens", [[1], [2], [4], [40]])
def test_query_rows_at_the_top_of_bf16(gpu, bits, q_lens):
    """Rows whose largest element lies in [2^127, 2^128), against keys so small that their scores are ordinary numbers: of either
    sign, beside rows of ordinary size, in tiles of 8, 16 and 32 rows and of 256."""
    heads, n = 8, q_lens[0]
    p = Paged(gpu, mb.BFLOAT16, bits, q_lens, [90], kv_heads=1, dim=64, page=16, seed=14)
    rng = np.random.default_rng(14)
    for page, slot in ((p.tables[0][i // 16], i % 16) for i in range(90)):
        element, lift = int(rng.integers(8, 16)), int(rng.integers(0, 3))      # 1 .. 1.875 times 2^-124 .. 2^-122, and zeros beside it
        if bits == 8:
            p.pool["k"][page, 0, slot], p.exps["k"][page, 0, slot] = 0, -124 + lift
            p.pool["k"][page, 0, slot, 5] = 0x30 + element                      # exponent field 7: 1.fff
        else:
            p.pool["k"][page, 0, slot] = 0
            p.pool["k"][page, 0, slot, 5:6] = bits_of(mb.BFLOAT16, [element * 2.0 ** (-127 + lift)])
    p.upload()
    q = rng.standard_normal((n, heads, 64)).astype(np.float32)
    q[:, 0, 5], q[:, 1, 5], q[:, 2, 5], q[:, 3, 5] = 2.0 ** 127, -1.9 * 2.0 ** 127, 2.0 ** 126, 1.5 * 2.0 ** 127
    q[:, 3, 9] = -2.0 ** 127
    qb = bits_of(mb.BFLOAT16, q)
    got = mb.paged_attention(mb.Tensor.from_bits(gpu, mb.BFLOAT16, qb), p.cache, p.batch).to_bits()
    check_attention(p, qb, got)


@pytest.mark.parametrize("name,bits", [("fp16", 16), ("fp16", 8), ("bf16", 8), ("bf16", 16)])
@pytest.mark.parametrize("q_lens,kv_lens", [([1], [30000]), ([8], [30000]), ([16], [30000]), ([20], [30000]), ([300], [900]), ([1, 20, 300], [700, 9000, 900])])
@pytest.mark.parametrize("gap", [20.5, 24.7, 28.3])
def test_many_small_weights_beside_a_large_one(gpu, name, bits, q_lens, kv_lens, gap):
    """The first cached token's weight is 2^gap times that of every other one; all elements of the output but the first come from the
    others, however small their weights are. fp16 weights under 2^-21 of the largest (of the tensor cores' tiles; 2^-29 in the streaming
    kernel) are off by up to 2^-32 of it, the others by half a step."""
    dt, dim = DTYPES[name], 16
    p = Paged(gpu, dt, bits, q_lens, kv_lens, kv_heads=1, dim=dim, page=128, seed=15)
    for b, n in enumerate(kv_lens):
        k, v = np.zeros((n, dim)), np.ones((n, dim))
        k[0, 0] = 16.0
        v[0, 1:], v[1:, 0] = 0.0, 0.0
        pos = np.arange(n)
        at = np.asarray(p.tables[b])[pos // p.page], 0, pos % p.page
        for side, rows in (("k", k), ("v", v)):
            if bits == 8:
                p.pool[side][at], p.exps[side][at] = A.quantise(rows, dt)
            else:
                p.pool[side][at] = bits_of(dt, rows)
    p.upload()
    tokens = sum(q_lens)
    q = np.zeros((tokens, 2, dim))
    q[:, :, 0] = 1.0
    q[:, 1, 1] = 1.0
    qb, scale = bits_of(dt, q), gap * np.log(2.0) / 16
    lse = mb.Tensor(gpu, mb.FLOAT32, (tokens, 2))
    out = mb.paged_attention(mb.Tensor.from_bits(gpu, dt, qb), p.cache, p.batch, lse=lse, scale=scale)
    got = out.to_bits()
    if gap > 21 and dt == mb.FLOAT16 and 2 * max(q_lens) > 16:
        at = 0
        for b, n in enumerate(q_lens):
            want = A.attention(O.bits_to_f64(dt, qb[at:at + n]), p.rows("k", b), p.rows("v", b), scale, True, 0)[0]
            assert (np.abs(O.bits_to_f64(dt, got[at:at + n]) - want) <= kv_lens[b] * 2.0 ** -32 + 2.0 ** -10 * want + 2.0 ** -25).all()
            at += n
    else:
        check_attention(p, qb, got, lse.to_bits().view(np.float32).astype(np.float64), scale=scale)


def batch_of(gpu, cu, kv_lens, tables, max_q=0):
    """A batch with offsets as they are, sound or not."""
    width = max(len(t) for t in tables)
    table = np.full((len(tables), width), -1, np.int32)
    for b, t in enumerate(tables):
        table[b, :len(t)] = t
    return mb.KVBatch(len(tables), width, cu_q=DeviceArray(gpu, np.asarray(cu, np.int32)), kv_len=DeviceArray(gpu, np.asarray(kv_lens, np.int32)),
                      pages=DeviceArray(gpu, table), max_q=max_q)


BAD_OFFSETS = [([0, 3, 400], 0, [0]),                     # past the rows
               ([0, 3, 43], 20, [0]),                     # more new tokens than max_q
               ([0, 43, 3], 0, [0]),                      # descending
               ([-2, 3, 43], 0, [1]),                     # before the rows
               ([43, 43, 0], 0, []),                      # no row belongs to anyone
               ([0, 0, 2 ** 31 - 1], 0, []), ([2 ** 31 - 1, -2 ** 31, 0], 0, [])]


def reported(gpu, words):
    with pytest.raises(mb.MagB200Error) as e:
        mb.synchronize(gpu)
    assert e.value.code == mb.ERR_INVALID_ARG and words in str(e.value)
    mb.synchronize(gpu)                                                   # once


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("cu,max_q,sound", BAD_OFFSETS)
def test_offsets_that_do_not_fit_are_reported_by_the_write(gpu, bits, cu, max_q, sound):
    """The sequences in `sound` are written as they should be, the others not at all."""
    p = Paged(gpu, mb.BFLOAT16, bits, [3, 40], [90, 100], kv_heads=2, dim=64, page=16, seed=5)
    rows = bits_of(mb.BFLOAT16, np.random.default_rng(3).standard_normal((43, 2, 64)))
    t = mb.Tensor.from_bits(gpu, mb.BFLOAT16, rows)
    mb.kv_cache_write(p.cache, batch_of(gpu, cu, [90, 100], p.tables, max_q), t, t)
    reported(gpu, "offsets")
    want = {(n, "pool"): p.pool[n].copy() for n in ("k", "v")} | {(n, "exps"): p.exps[n].copy() for n in p.exps}
    for b in sound:
        for i in range(cu[b], cu[b + 1]):
            pos = p.kv_lens[b] - (cu[b + 1] - i)
            at = p.tables[b][pos // 16], slice(None), pos % 16
            for n in ("k", "v"):
                if bits == 8:
                    want[n, "pool"][at], want[n, "exps"][at] = A.quantise(O.bits_to_f64(mb.BFLOAT16, rows[i]), mb.BFLOAT16)
                else:
                    want[n, "pool"][at] = rows[i]
    got = p.download()
    assert all(np.array_equal(got[key], w) for key, w in want.items())


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("cu,max_q,sound", [c for c in BAD_OFFSETS if not c[1]])
def test_offsets_that_do_not_fit_are_reported_by_the_read(gpu, bits, cu, max_q, sound):
    p = Paged(gpu, mb.BFLOAT16, bits, [3, 40], [90, 100], kv_heads=2, dim=64, page=16, seed=5)
    before = np.full((43, 2, 64), 0x1234, np.uint16)
    k, v = mb.Tensor.from_bits(gpu, mb.BFLOAT16, before), mb.Tensor.from_bits(gpu, mb.BFLOAT16, before)
    mb.kv_cache_read(p.cache, p.batch, DeviceArray(gpu, np.asarray(cu, np.int32)), k, v)
    reported(gpu, "offsets")
    for name, t in (("k", k), ("v", v)):
        want = before.copy()
        for b in sound:
            want[cu[b]:cu[b + 1]] = bits_of(mb.BFLOAT16, p.rows(name, b, cu[b + 1] - cu[b]))
        assert np.array_equal(t.to_bits(), want)


def test_bad_offsets_among_many_sequences_are_reported(gpu):
    """A sequence without tokens of its own, far from every token's, with more sequences than the grid has threads."""
    n = 2000
    cu = np.zeros(n + 1, np.int32)
    cu[1:] = 2
    cu[1500] = 1                                                          # down and up again, within the rows
    table = DeviceArray(gpu, np.zeros((n, 1), np.int32))
    batch = mb.KVBatch(n, 1, cu_q=DeviceArray(gpu, cu), kv_len=DeviceArray(gpu, np.full(n, 2, np.int32)), pages=table)
    cache = mb.KVCache(gpu, mb.BFLOAT16, 1, 16, 1, 16)
    rows = mb.Tensor.from_bits(gpu, mb.BFLOAT16, np.zeros((2, 1, 16), np.uint16))
    mb.kv_cache_write(cache, batch, rows, rows)
    reported(gpu, "offsets")
    out = mb.Tensor(gpu, mb.BFLOAT16, (2, 1, 16)), mb.Tensor(gpu, mb.BFLOAT16, (2, 1, 16))
    mb.kv_cache_read(cache, batch, DeviceArray(gpu, cu), *out)
    reported(gpu, "offsets")


def test_pages_and_lengths_that_do_not_fit_are_reported_by_write_and_read(gpu):
    """A bad page that a write or a read has to touch, and more rows asked for than are cached: the rest is done."""
    p = Paged(gpu, mb.BFLOAT16, 16, [3, 40], [90, 100], kv_heads=2, dim=64, page=16, seed=5)
    rows = bits_of(mb.BFLOAT16, np.random.default_rng(3).standard_normal((43, 2, 64)))
    t = mb.Tensor.from_bits(gpu, mb.BFLOAT16, rows)
    tables = [list(x) for x in p.tables]
    tables[1][4] = 10 ** 6                                                # positions 64 .. 79 of sequence 1, whose new tokens are 60 .. 99
    want = p.pool["k"].copy()
    for i in range(43):
        b, pos = (0, 87 + i) if i < 3 else (1, 57 + i)
        if not (b == 1 and 64 <= pos < 80):
            want[p.tables[b][pos // 16], :, pos % 16] = rows[i]
    mb.kv_cache_write(p.cache, batch_of(gpu, [0, 3, 43], [90, 100], tables), t, t)
    reported(gpu, "a page")
    assert np.array_equal(p.download()["k", "pool"], want)
    p.pool["k"] = want
    before = np.full((200, 2, 64), 0x1234, np.uint16)
    for bad, cu, words in ((tables, [0, 90, 190], "a page"), (p.tables, [0, 90, 195], "a length")):
        k, v = mb.Tensor.from_bits(gpu, mb.BFLOAT16, before), mb.Tensor.from_bits(gpu, mb.BFLOAT16, before)
        mb.kv_cache_read(p.cache, batch_of(gpu, [0, 3, 43], [90, 100], bad), DeviceArray(gpu, np.asarray(cu, np.int32)), k, v)
        reported(gpu, words)
        expect = before.copy()
        expect[:190] = np.concatenate([bits_of(mb.BFLOAT16, p.rows("k", 0, 90)), bits_of(mb.BFLOAT16, p.rows("k", 1, 100))])
        if bad is tables:
            expect[90 + 64:90 + 80] = 0x1234
        assert np.array_equal(k.to_bits(), expect)


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("q_lens", [[2, 1], [2, 70]])
def test_negative_lengths_are_reported(gpu, bits, q_lens):
    """A sequence with new tokens and a negative length: reported by all operators; its rows see nothing, the others are as ever. Without
    new tokens its length is nobody's business."""
    p = Paged(gpu, mb.BFLOAT16, bits, q_lens, [90, 100], kv_heads=2, dim=64, page=16, seed=5)
    tokens = sum(q_lens)
    rows = mb.Tensor.from_bits(gpu, mb.BFLOAT16, bits_of(mb.BFLOAT16, np.random.default_rng(3).standard_normal((tokens, 2, 64))))
    q = mb.Tensor.from_bits(gpu, mb.BFLOAT16, bits_of(mb.BFLOAT16, np.random.default_rng(4).standard_normal((tokens, 4, 64))))
    want = mb.paged_attention(q, p.cache, p.batch).to_bits()
    cu = [0, q_lens[0], tokens]
    bad = batch_of(gpu, cu, [90, -3], p.tables)
    out = mb.paged_attention(q, p.cache, bad)
    reported(gpu, "a length")
    got = out.to_bits()
    assert np.array_equal(got[:q_lens[0]], want[:q_lens[0]]) and (got[q_lens[0]:] == 0).all()
    before = p.download()
    mb.kv_cache_write(p.cache, batch_of(gpu, cu, [-1, -3], p.tables), rows, rows)
    reported(gpu, "a length")
    after = p.download()
    assert all(np.array_equal(before[key], after[key]) for key in before)
    mb.kv_cache_read(p.cache, bad, DeviceArray(gpu, np.array([0, 0, 1], np.int32)), rows, mb.Tensor(gpu, mb.BFLOAT16, (tokens, 2, 64)))
    reported(gpu, "a length")
    idle = batch_of(gpu, [0, tokens, tokens], [90, -3], p.tables)
    mb.kv_cache_write(p.cache, idle, rows, rows)
    mb.paged_attention(q, p.cache, idle, mb.Tensor(gpu, mb.BFLOAT16, (tokens, 4, 64)))
    mb.synchronize(gpu)


@pytest.mark.parametrize("name", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("dim", [8, 64, 96, 128, 256])
@pytest.mark.parametrize("pad", [0, 1])
def test_norm_of_rows_whose_squares_leave_fp32(gpu, name, dim, pad):
    """Rows so large or so small that the squares of their elements overflow or underflow, beside ordinary ones."""
    dt = DTYPES[name]
    rng = np.random.default_rng(dim)
    powers = {"fp16": [15, 0, -14, -20, -24]}.get(name, [126, 100, 64, 63, 0, -40, -50, -51, -64, -100, -126, -140 if name == "fp32" else -130])
    x = rng.uniform(1.0, 1.9, (len(powers) + 1, 3, dim)) * rng.choice([-1.0, 1.0], (len(powers) + 1, 3, dim))
    x[:-1] *= np.exp2(np.asarray(powers, np.float64))[:, None, None]
    x[:, 1, 1:] *= 2.0 ** -9                                               # one element makes the mean
    x[-1, 2] = 0.0
    buf = np.zeros((len(powers) + 1, 3 * dim + pad), np.uint32 if dt == mb.FLOAT32 else np.uint16)
    buf[:, pad:] = bits_of(dt, x).reshape(len(powers) + 1, -1)
    t = mb.Tensor.from_bits(gpu, dt, buf).as_strided((len(powers) + 1, 3, dim), (3 * dim + pad, dim, 1), pad)
    w = bits_of(dt, rng.uniform(0.5, 1.5, dim))
    given = O.bits_to_f64(dt, bits_of(dt, x))
    for eps in (1e-6, 0.0, 1.0):
        got = O.bits_to_f64(dt, mb.qk_norm_rope(t, None, None, q_weight=mb.Tensor.from_bits(gpu, dt, w), eps=eps)[0].to_bits())
        eps32 = np.float64(np.float32(eps))
        with np.errstate(invalid="ignore"):
            want = A.norm_rope(given, O.bits_to_f64(dt, w), eps32, None, None, 0, False, 1.0)[0]
        # one rounding of the result; the mean of squares, its root and the products: dim + 32 roundings of fp32; where they are
        # subnormal half a step of fp32 for each of the two products, the first times a weight below 1.5, and half one of the result
        least = {"fp16": 2.0 ** -25, "bf16": 2.0 ** -134, "fp32": 0.0}[name] + 2.5 * 2.0 ** -150
        tol = HALF_STEP[dt] * np.abs(want) + (dim + 32) * 2.0 ** -24 * np.abs(want) + least
        some = np.isfinite(want)                                          # a row of zeros with eps 0 has no norm
        assert np.isfinite(got[some]).all() and (np.abs(got - want)[some] <= tol[some]).all(), (eps, np.argwhere(~(np.abs(got - want) <= tol))[:4].tolist())
        assert some[:-1].all() and np.isnan(got[~some]).all()


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("q_lens", [[1, 2], [3, 70]])
def test_attention_takes_rows_of_a_bad_page_for_zeros(gpu, bits, q_lens):
    p = Paged(gpu, mb.BFLOAT16, bits, q_lens, [90, 200], kv_heads=2, dim=64, page=16, seed=5)
    tables = [list(t) for t in p.tables]
    tables[0][1], tables[1][9] = 10 ** 6, -7
    for b, i in ((0, 1), (1, 9)):
        for n in ("k", "v"):
            p.pool[n][p.tables[b][i]] = 0
            if bits == 8:
                p.exps[n][p.tables[b][i]] = 0
    p.upload()
    tokens = sum(q_lens)
    qb = bits_of(mb.BFLOAT16, np.random.default_rng(4).standard_normal((tokens, 4, 64)))
    q, lse, want_lse = mb.Tensor.from_bits(gpu, mb.BFLOAT16, qb), mb.Tensor(gpu, mb.FLOAT32, (tokens, 4)), mb.Tensor(gpu, mb.FLOAT32, (tokens, 4))
    want = mb.paged_attention(q, p.cache, p.batch, lse=want_lse).to_bits()
    check_attention(p, qb, want)
    got = mb.paged_attention(q, p.cache, batch_of(gpu, [0, q_lens[0], tokens], [90, 200], tables), lse=lse)
    reported(gpu, "a page")
    assert np.array_equal(got.to_bits(), want) and np.array_equal(lse.to_bits(), want_lse.to_bits())


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("limit", [1, 3, 20, 147])
def test_attention_under_a_limit_of_ctas(gpu, bits, limit):
    """Units whole and in parts, beside single tokens, on fewer multiprocessors than there are."""
    L = mb.lib()
    mb.check(L.magb200_set_cta_limit(gpu, limit))
    try:
        for q_lens, kv_lens, heads, hk in (([330, 1, 40, 700], [2500, 900, 4000, 1400], 6, 2), ([200], [3300], 8, 1), ([50] * 8, [1300] * 8, 16, 8)):
            attend(gpu, Paged(gpu, mb.BFLOAT16, bits, q_lens, kv_lens, kv_heads=hk, dim=64, page=32, seed=limit), heads)
    finally:
        mb.check(L.magb200_set_cta_limit(gpu, 0))


def test_the_attention_leaves_multiprocessors_free(gpu):
    """The limit of CTAs shows in the time: 128 units on four multiprocessors, so on all of them."""
    L = mb.lib()
    p = Paged(gpu, mb.BFLOAT16, 16, [4096], [4096], kv_heads=8, dim=64, page=64)
    q = mb.Tensor.from_bits(gpu, mb.BFLOAT16, bits_of(mb.BFLOAT16, np.random.default_rng(1).standard_normal((4096, 8, 64))))
    out = mb.Tensor(gpu, mb.BFLOAT16, (4096, 8, 64))

    def ms(limit):
        mb.check(L.magb200_set_cta_limit(gpu, limit))
        times = []
        for _ in range(5):
            mb.synchronize(gpu)
            t = time.perf_counter()
            for _ in range(10):
                mb.paged_attention(q, p.cache, p.batch, out)
            mb.synchronize(gpu)
            times.append(time.perf_counter() - t)
        return min(times)

    try:
        assert ms(4) > 5 * ms(0)                                          # 37 times fewer
    finally:
        mb.check(L.magb200_set_cta_limit(gpu, 0))


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("batch", [33, 64, 65, 200])
@pytest.mark.parametrize("window", [0, 50])
def test_decode_batches_of_more_sequences_than_lanes(gpu, bits, batch, window):
    """Single tokens of many sequences, none of some, lengths from none on: the sequences behind the first 32 are counted first and
    searched afterwards, and pieces end anywhere in the line of all of them."""
    rng = np.random.default_rng(batch + window)
    q = [int(n) for n in rng.integers(0, 3, batch)]
    kv = [int(n) for n in np.exp(rng.uniform(0.0, np.log(700.0), batch))]
    q[0], q[31], q[32], q[-1], kv[5], kv[40 % batch], kv[-1] = 1, 0, 1, 1, 0, 0, 2000
    p = Paged(gpu, mb.BFLOAT16, bits, q, kv, kv_heads=3, dim=64, page=16, seed=batch)
    attend(gpu, p, 6, window=window, pad_rows=1)


def test_decode_batch_of_a_thousand_sequences(gpu):
    p = Paged(gpu, mb.FLOAT16, 16, [1] * 1000, [1 + (i * 37) % 90 for i in range(1000)], kv_heads=1, dim=32, page=16, seed=3)
    attend(gpu, p, 2)


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("tokens,rows", [(9600, [0, 1, 127, 128, 255, 256, 4863, 9471, 9472, 9599]), (600, [0, 255, 256, 599]), (20, [0, 19])])
def test_rows_behind_90000_cached_ones(gpu, bits, tokens, rows):
    """Long walks of the tensor cores' kernel, units whole and in parts, against the definition: the first and last rows of tiles, with
    the rounding that check_attention counts. Scores spread by 4, so that a row is made of a few of its cached rows, wherever they are."""
    p = Paged(gpu, mb.BFLOAT16, bits, [tokens], [90000], kv_heads=2, dim=16, page=64, seed=6)
    qb = bits_of(mb.BFLOAT16, np.random.default_rng(6).standard_normal((tokens, 4, 16)) * 4)
    got = O.bits_to_f64(mb.BFLOAT16, mb.paged_attention(mb.Tensor.from_bits(gpu, mb.BFLOAT16, qb), p.cache, p.batch).to_bits())
    q, k, v, u = O.bits_to_f64(mb.BFLOAT16, qb), p.rows("k", 0), p.rows("v", 0), HALF_STEP[mb.BFLOAT16]
    for r in rows:
        n = 90000 - tokens + r + 1
        want, _, spread, size = A.attention(q[r:r + 1], k[:n], v[:n], 0.25, True, 0)
        weight = 2 * 16 * 2.0 ** -24 * size + 2.0 ** -22 + n * 2.0 ** -24
        tol = u * np.abs(want) + (u + 2 * weight[..., None]) * spread + 2.0 ** -25
        assert (tol < np.abs(want).max() / 8).all()                        # what a row of other places would be off by
        assert (np.abs(got[r:r + 1] - want) <= tol).all(), (r, float((np.abs(got[r:r + 1] - want) / tol).max()))


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("q_lens,kv_lens,heads,hk,window", [
    ([64] + [1] * 45, [6000] + [40 + 7 * i for i in range(45)], 32, 8, 0),      # a chunk on a long context beside many single tokens
    ([1] * 20 + [300, 20, 90] + [1] * 30, [90] * 20 + [2500, 1300, 1700] + [200] * 30, 12, 12, 0),
    ([1] * 20 + [300, 20, 90] + [1] * 30, [90] * 20 + [2500, 1300, 1700] + [200] * 30, 12, 12, 1100),
    ([200] * 20 + [1] * 20, [1300] * 40, 8, 8, 0),                              # a round and a rest beside single tokens
    ([100, 1, 30] + [1] * 120, [9000, 3, 5000] + [50] * 120, 4, 4, 0),          # more single tokens than the chunks' rows
])
def test_units_are_cut_beside_single_tokens(gpu, bits, q_lens, kv_lens, heads, hk, window):
    """Few units of many rows in a batch of many sequences, which the host's bound counts as a unit each."""
    p = Paged(gpu, mb.BFLOAT16, bits, q_lens, kv_lens, kv_heads=hk, dim=64, page=32, seed=len(q_lens))
    attend(gpu, p, heads, window=window)


def test_a_chunk_takes_no_longer_beside_single_tokens(gpu):
    """16 units on 100000 cached rows use all multiprocessors, whatever else is in the batch."""
    def ms(singles):
        n = 1 + singles
        p = Paged(gpu, mb.BFLOAT16, 16, [64] + [1] * singles, [100000] + [16] * singles, kv_heads=8, dim=64, page=256)
        q = mb.Tensor.from_bits(gpu, mb.BFLOAT16, np.zeros((63 + n, 64, 64), np.uint16))
        out = mb.Tensor(gpu, mb.BFLOAT16, (63 + n, 64, 64))
        times = []
        for _ in range(5):
            mb.synchronize(gpu)
            t = time.perf_counter()
            for _ in range(10):
                mb.paged_attention(q, p.cache, p.batch, out)
            mb.synchronize(gpu)
            times.append(time.perf_counter() - t)
        return min(times)

    assert ms(60) < 3 * ms(0)                                             # 9 times with every unit whole


@pytest.mark.parametrize("bits", [16, 8])
def test_caches_beyond_32_bits(gpu, bits):
    """Pools of more than 2^31 elements (and, with 16 bits, 2^32 bytes); the sequences lie in their first and last pages."""
    dt, pages, page, hk, dim = mb.BFLOAT16, 17000, 128, 8, 128
    cache = mb.KVCache(gpu, dt, pages, page, hk, dim, bits)
    try:
        tables = [[pages - 1, 0, pages - 3], [pages - 2, pages - 5]]
        q_lens, kv_lens = [300, 130], [300, 130]
        rng = np.random.default_rng(bits)
        kb, vb, qb = (bits_of(dt, rng.standard_normal((430, n, dim))) for n in (hk, hk, 2 * hk))
        k, v, q = (mb.Tensor.from_bits(gpu, dt, x) for x in (kb, vb, qb))
        batch = batch_of(gpu, [0, 300, 430], kv_lens, tables)
        mb.kv_cache_write(cache, batch, k, v)
        rk, rv = mb.Tensor(gpu, dt, (430, hk, dim)), mb.Tensor(gpu, dt, (430, hk, dim))
        mb.kv_cache_read(cache, batch, DeviceArray(gpu, np.array([0, 300, 430], np.int32)), rk, rv)
        back = []
        for got, raw in ((rk, kb), (rv, vb)):
            want = raw if bits == 16 else bits_of(dt, A.dequantise(*A.quantise(O.bits_to_f64(dt, raw), dt)))
            assert np.array_equal(got.to_bits(), want)
            back.append(O.bits_to_f64(dt, want))
        many = O.bits_to_f64(dt, mb.paged_attention(q, cache, batch).to_bits())
        at = np.array([299, 429])                                          # the last new tokens alone: the streaming kernel
        few = mb.paged_attention(mb.Tensor.from_bits(gpu, dt, qb[at]), cache, batch_of(gpu, [0, 1, 2], kv_lens, tables), None)
        few = O.bits_to_f64(dt, few.to_bits())
        for b, rows in enumerate((slice(0, 300), slice(300, 430))):
            want, _, spread, size = A.attention(O.bits_to_f64(dt, qb[rows]), back[0][rows], back[1][rows], dim ** -0.5, True, 0)
            weight = 2 * dim * 2.0 ** -24 * size + 2.0 ** -22 + kv_lens[b] * 2.0 ** -24
            tol = HALF_STEP[dt] * np.abs(want) + (HALF_STEP[dt] + 2 * weight[..., None]) * spread + 2.0 ** -25
            assert (np.abs(many[rows] - want) <= tol).all() and (np.abs(few[b] - want[-1]) <= tol[-1]).all()
        mb.synchronize(gpu)
    finally:
        del cache
        mb.check(mb.lib().magb200_pool_trim(gpu))
