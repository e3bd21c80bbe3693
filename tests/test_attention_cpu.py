"""Refusals and host-side decisions of the operators around the KV cache: no device is touched."""
import ctypes as C

import numpy as np
import pytest

import magnetron_b200 as mb
from oracle import attention_oracle as A
from oracle import mag_oracle as O

BASE = 1 << 40          # never dereferenced: every call here is refused on the host
POOL = [(1 << 44) + (i << 40) for i in range(4)]


def tensor(shape, dtype=mb.BFLOAT16, strides=None, at=BASE, offset=0):
    return mb.Tensor(0, dtype, shape, strides, base_ptr=at, offset=offset)


def cache(**kw):
    a = dict(dtype=mb.BFLOAT16, pages=10, page_size=16, kv_heads=2, head_dim=64, bits=16, k=POOL[0], v=POOL[1], k_exp=POOL[2], v_exp=POOL[3]) | kw
    return mb.KVCache(0, a["dtype"], a["pages"], a["page_size"], a["kv_heads"], a["head_dim"], a["bits"], k=a["k"], v=a["v"], k_exp=a["k_exp"], v_exp=a["v_exp"])


def batch(**kw):
    a = dict(batch=2, max_pages=4, cu_q=BASE, kv_len=BASE, pages=BASE, max_q=0, max_kv=0) | kw
    return mb.KVBatch(a["batch"], a["max_pages"], cu_q=a["cu_q"], kv_len=a["kv_len"], pages=a["pages"], max_q=a["max_q"], max_kv=a["max_kv"])


def refused(code, fn, *a, **kw):
    with pytest.raises(mb.MagB200Error) as e:
        fn(*a, **kw)
    assert e.value.code == code, e.value
    return str(e.value)


Q = (6, 4, 64)
FAR = BASE + (1 << 30)


def test_a_sound_call_gets_as_far_as_the_device():
    if mb.device_count() > 0:
        pytest.skip("a device is present")
    code = mb.ERR_NO_DEVICE
    refused(code, mb.paged_attention, tensor(Q), cache(), batch(), tensor(Q, at=FAR))
    refused(code, mb.kv_cache_write, cache(bits=8), batch(), tensor((6, 2, 64)), tensor((6, 2, 64)))
    refused(code, mb.kv_cache_read, cache(), batch(), BASE, tensor((6, 2, 64)), tensor((6, 2, 64), at=FAR))
    refused(code, mb.qk_norm_rope, tensor(Q), tensor((6, 2, 64), at=FAR), mb.Rope(BASE, BASE, 64), tensor(Q), tensor((6, 2, 64), at=FAR))


@pytest.mark.parametrize("change", [dict(page_size=24), dict(page_size=8), dict(page_size=0), dict(head_dim=72), dict(head_dim=8), dict(head_dim=0), dict(bits=4),
                                    dict(dtype=mb.FLOAT32), dict(dtype=7), dict(pages=0), dict(pages=1 << 40), dict(kv_heads=0), dict(k=BASE + 2), dict(v=BASE + 8),
                                    dict(bits=8, k_exp=BASE + 4)])
def test_refused_caches(change):
    rows = tensor((6, 2, 64))
    for call in (lambda c: mb.kv_cache_write(c, batch(), rows, rows), lambda c: mb.kv_cache_read(c, batch(), BASE, rows, tensor((6, 2, 64), at=FAR)),
                 lambda c: mb.paged_attention(tensor(Q), c, batch(), tensor(Q, at=FAR))):
        refused(mb.ERR_INVALID_ARG, call, cache(**change))


def test_refused_null_pools():
    for name in ("k", "v", "k_exp", "v_exp"):
        c = cache(bits=8)
        setattr(c.struct, name, None)
        refused(mb.ERR_INVALID_ARG, mb.kv_cache_write, c, batch(), tensor((6, 2, 64)), tensor((6, 2, 64)))


@pytest.mark.parametrize("change", [dict(batch=0), dict(batch=-1), dict(max_pages=0), dict(max_q=-1), dict(max_kv=-1), dict(cu_q=None), dict(kv_len=None), dict(pages=None)])
def test_refused_batches(change):
    rows = tensor((6, 2, 64))
    refused(mb.ERR_INVALID_ARG, mb.kv_cache_write, cache(), batch(**change), rows, rows)
    refused(mb.ERR_INVALID_ARG, mb.paged_attention, tensor(Q), cache(), batch(**change), tensor(Q, at=FAR))


def test_refused_rows_of_the_cache():
    ok = tensor((6, 2, 64))
    for k in (tensor((6, 3, 64)), tensor((5, 2, 64)), tensor((6, 2, 32)), tensor((6, 128))):
        refused(mb.ERR_SHAPE, mb.kv_cache_write, cache(), batch(), k, ok)
    refused(mb.ERR_INVALID_ARG, mb.kv_cache_write, cache(), batch(), tensor((6, 2, 64), mb.FLOAT16), ok)
    refused(mb.ERR_INVALID_ARG, mb.kv_cache_write, cache(), batch(), tensor((6, 2, 64), strides=(256, 128, 2)), ok)
    refused(mb.ERR_INVALID_ARG, mb.kv_cache_read, cache(), batch(), None, ok, tensor((6, 2, 64), at=FAR))
    refused(mb.ERR_INVALID_ARG, mb.kv_cache_read, cache(), batch(), BASE, ok, ok)                              # both results in one place
    refused(mb.ERR_INVALID_ARG, mb.kv_cache_read, cache(), batch(), BASE, tensor((6, 2, 64), strides=(64, 64, 1)), tensor((6, 2, 64), at=FAR))


def test_refused_attention_calls():
    out = tensor(Q, at=FAR)

    def call(q=tensor(Q), c=cache(), b=batch(), o=out, **kw):
        mb.paged_attention(q, c, b, o, **kw)

    refused(mb.ERR_INVALID_ARG, call, c=cache(head_dim=144), q=tensor((6, 4, 144)), o=tensor((6, 4, 144), at=FAR))
    refused(mb.ERR_SHAPE, call, q=tensor((6, 3, 64)), o=tensor((6, 3, 64), at=FAR))                             # 3 heads over 2
    refused(mb.ERR_SHAPE, call, q=tensor((6, 4, 80)), o=tensor((6, 4, 80), at=FAR))
    refused(mb.ERR_SHAPE, call, o=tensor((5, 4, 64), at=FAR))
    refused(mb.ERR_INVALID_ARG, call, q=tensor(Q, mb.FLOAT16))
    refused(mb.ERR_INVALID_ARG, call, q=tensor(Q, mb.FLOAT32), o=tensor(Q, mb.FLOAT32, at=FAR))
    refused(mb.ERR_INVALID_ARG, call, q=tensor(Q, offset=4))                                                    # 8 bytes off
    refused(mb.ERR_INVALID_ARG, call, q=tensor(Q, strides=(300, 64, 1)))
    refused(mb.ERR_INVALID_ARG, call, o=tensor(Q))                                                              # out is q
    refused(mb.ERR_INVALID_ARG, call, o=tensor(Q, at=FAR, strides=(0, 64, 1)))
    for scale in (float("nan"), float("inf")):
        refused(mb.ERR_INVALID_ARG, call, scale=scale)
    refused(mb.ERR_INVALID_ARG, call, window=-1)
    refused(mb.ERR_INVALID_ARG, call, window=5, causal=False)
    refused(mb.ERR_SHAPE, call, lse=tensor((6, 4), mb.BFLOAT16, at=2 * FAR))
    refused(mb.ERR_SHAPE, call, lse=tensor((6, 5), mb.FLOAT32, at=2 * FAR))
    refused(mb.ERR_SHAPE, call, lse=tensor((6, 4), mb.FLOAT32, strides=(8, 1), at=2 * FAR))
    refused(mb.ERR_INVALID_ARG, call, lse=tensor((6, 4), mb.FLOAT32, at=FAR))                                   # lse inside out


def test_refused_norms_and_rotations():
    q, k, rope = tensor(Q), tensor((6, 2, 64), at=FAR), mb.Rope(BASE, BASE, 64)

    def call(q=q, k=k, rope=rope, qo=tensor(Q, at=4 * FAR), ko=tensor((6, 2, 64), at=8 * FAR), **kw):
        mb.qk_norm_rope(q, k, rope, qo, ko, **kw)

    refused(mb.ERR_INVALID_ARG, call, q=tensor((6, 4, 60)), qo=tensor((6, 4, 60), at=4 * FAR))
    refused(mb.ERR_INVALID_ARG, call, q=tensor((6, 4, 264)), qo=tensor((6, 4, 264), at=4 * FAR))
    refused(mb.ERR_SHAPE, call, qo=tensor((6, 5, 64), at=4 * FAR))
    refused(mb.ERR_SHAPE, call, k=tensor((5, 2, 64), at=FAR), ko=tensor((5, 2, 64), at=8 * FAR))
    refused(mb.ERR_INVALID_ARG, call, ko=tensor((6, 2, 64), mb.FLOAT16, at=8 * FAR))
    for r in (mb.Rope(BASE, BASE, 0), mb.Rope(BASE, BASE, 63), mb.Rope(BASE, BASE, 66), mb.Rope(None, BASE, 64), mb.Rope(BASE, None, 64), mb.Rope(BASE, BASE, 64, factor=float("nan"))):
        refused(mb.ERR_INVALID_ARG, call, rope=r)
    refused(mb.ERR_SHAPE, call, q_weight=tensor((32,), at=16 * FAR))
    refused(mb.ERR_INVALID_ARG, call, q_weight=tensor((64,), mb.FLOAT32, at=16 * FAR))
    refused(mb.ERR_INVALID_ARG, call, k_weight=tensor((64,), strides=(2,), at=16 * FAR))
    for eps in (-1.0, 2.0, float("nan")):
        refused(mb.ERR_INVALID_ARG, call, q_weight=tensor((64,), at=16 * FAR), eps=eps)
    refused(mb.ERR_INVALID_ARG, call, qo=k.as_strided((6, 4, 64), (128, 32, 1)))                                # rows of the result overlap
    refused(mb.ERR_INVALID_ARG, call, qo=tensor(Q, offset=64))                                                  # shifted onto its own input
    refused(mb.ERR_INVALID_ARG, call, qo=tensor(Q, at=FAR))                                                     # onto k
    refused(mb.ERR_INVALID_ARG, call, ko=tensor((6, 2, 64), at=4 * FAR))                                        # both results in one place
    rc = mb.lib().magb200_qk_norm_rope(0, C.byref(q.view_struct()), C.byref(k.view_struct()), None, None, 0.0, None, C.byref(q.view_struct()), None)
    assert rc == mb.ERR_INVALID_ARG


def test_slices_of_one_fused_buffer_are_not_an_overlap():
    """q, k and their results as column slices of one buffer, whose address ranges interleave: refused only by the missing device."""
    if mb.device_count() > 0:
        pytest.skip("a device is present")
    w = 8 * 64
    q, k = tensor((6, 4, 64), strides=(w, 64, 1)), tensor((6, 2, 64), strides=(w, 64, 1), offset=4 * 64)
    refused(mb.ERR_NO_DEVICE, mb.qk_norm_rope, q, k, mb.Rope(BASE, BASE, 64), q, k)
    refused(mb.ERR_INVALID_ARG, mb.qk_norm_rope, q, k, mb.Rope(BASE, BASE, 64), q, tensor((6, 2, 64), strides=(w, 64, 1), offset=3 * 64))


def test_refused_overlaps_with_the_cache():
    rows, out = tensor((6, 2, 64)), tensor(Q, at=FAR)
    half = 10 * 2 * 16 * 64                                                   # bytes of a 16-bit pool / 2, of an 8-bit pool
    for i, c in ((0, cache()), (1, cache()), (2, cache(bits=8)), (3, cache(bits=8))):
        inside = tensor((6, 2, 64), at=POOL[i] + 128)
        assert "in the cache" in refused(mb.ERR_INVALID_ARG, mb.kv_cache_write, c, batch(), inside, rows)
        assert "in the cache" in refused(mb.ERR_INVALID_ARG, mb.kv_cache_write, c, batch(), rows, inside)
        assert "in the cache" in refused(mb.ERR_INVALID_ARG, mb.kv_cache_read, c, batch(), BASE, inside, rows)
        assert "in the cache" in refused(mb.ERR_INVALID_ARG, mb.kv_cache_read, c, batch(), BASE, rows, inside)
        assert "in the cache" in refused(mb.ERR_INVALID_ARG, mb.paged_attention, tensor(Q), c, batch(), tensor(Q, at=POOL[i] + 128))
        assert "in the cache" in refused(mb.ERR_INVALID_ARG, mb.paged_attention, tensor(Q), c, batch(), out, lse=tensor((6, 4), mb.FLOAT32, at=POOL[i] + 4))
    for c in (cache(v=POOL[0]), cache(v=POOL[0] + 2 * half - 16), cache(bits=8, v=POOL[0] + half - 16), cache(bits=8, k_exp=POOL[1]), cache(bits=8, v_exp=POOL[2])):
        assert "pools overlap" in refused(mb.ERR_INVALID_ARG, mb.kv_cache_write, c, batch(), rows, rows)
    w = tensor((64,), at=FAR + 64)
    assert "weight" in refused(mb.ERR_INVALID_ARG, mb.qk_norm_rope, tensor(Q), None, None, out, q_weight=w)


def test_refused_caches_beyond_64_bits():
    rows = tensor((6, 65535, 256))
    refused(mb.ERR_TOO_LARGE, mb.kv_cache_write, cache(pages=2 ** 31 - 1, kv_heads=65535, page_size=2 ** 20, head_dim=256), batch(), rows, rows)


def array(data, dtype=np.int32, device=0):
    """A DeviceArray as the checks see it, without a device."""
    a = mb.attention.DeviceArray.__new__(mb.attention.DeviceArray)
    data = np.asarray(data, dtype)
    a.device, a.ptr, a.dtype, a.size = device, None, data.dtype, data.size
    return a


def test_arrays_of_the_wrong_type_or_size_are_refused():
    good = dict(cu_q=array([0, 1, 2]), kv_len=array([1, 1]), pages=array(np.zeros((2, 4))))
    mb.KVBatch(2, 4, **good)
    for change in (dict(cu_q=array([0, 1])), dict(cu_q=array([0, 1, 2], np.int64)), dict(kv_len=array([1])), dict(kv_len=array([1, 1], np.float32)),
                   dict(pages=array(np.zeros((2, 3)))), dict(pages=array(np.zeros((2, 4)), np.int64))):
        with pytest.raises(ValueError):
            mb.KVBatch(2, 4, **(good | change))
    for positions, freq in ((array([0, 1], np.int64), array(np.ones(32), np.float32)), (array([0, 1]), array(np.ones(32), np.float64)),
                            (array([0, 1]), array(np.ones(31), np.float32))):
        with pytest.raises(ValueError):
            mb.Rope(positions, freq, 64)
    short = mb.Rope(array(np.arange(5)), array(np.ones(32), np.float32), 64)
    with pytest.raises(ValueError):
        mb.qk_norm_rope(tensor(Q), None, short, tensor(Q))
    with pytest.raises(ValueError):
        mb.kv_cache_read(cache(), batch(), array([0, 1]), tensor((6, 2, 64)), tensor((6, 2, 64), at=FAR))
    for more in (np.zeros(4, np.int32), np.zeros(2, np.int64)):
        with pytest.raises(ValueError):
            array([0, 1, 2]).update(more)
    for lists in (([], [], []), ([1], [1, 2], [[0], [1]]), ([1, 1], [1, 2], [[0]]), ([-1], [1], [[0]])):
        with pytest.raises(ValueError):
            mb.KVBatch.from_lists(0, *lists)


def test_tensors_of_two_devices_are_refused():
    other = mb.Tensor(1, mb.BFLOAT16, (6, 2, 64), base_ptr=FAR)
    rows = tensor((6, 2, 64))
    for call in (lambda: mb.kv_cache_write(cache(), batch(), rows, other), lambda: mb.kv_cache_read(cache(), batch(), BASE, other, rows),
                 lambda: mb.qk_norm_rope(tensor(Q), other, None, tensor(Q), rows),
                 lambda: mb.paged_attention(tensor(Q), cache(), batch(), mb.Tensor(1, mb.BFLOAT16, Q, base_ptr=FAR))):
        with pytest.raises(ValueError):
            call()


def test_the_oracles_codes():
    v = A.e4m3_values()
    assert v[0x7E] == 448 and v[0x08] == 2.0 ** -6 and v[0x01] == 2.0 ** -9 and np.isnan(v[0x7F])
    finite = np.array([c for c in range(256) if (c & 0x7F) != 0x7F])
    assert np.array_equal(A.e4m3_codes(v[finite]), finite)
    # ties go to the even code
    assert A.e4m3_codes(np.array([17.0, 19.0, 2.0 ** -10, 3 * 2.0 ** -10])).tolist() == [0x58, 0x5A, 0x00, 0x02]
    codes, exps = A.quantise(np.array([[448.0, 1.0], [449.0, 1.0], [0.0, 0.0], [np.inf, 1.0]]), O.BFLOAT16)
    assert exps.tolist() == [0, 1, -126, -128] and codes[0].tolist() == [0x7E, 0x38]


def test_addresses_between_two_elements_are_refused():
    """A load of an element that is not on a multiple of its size ends a device's context, so no such address gets there."""
    rows, out, w = (6, 2, 64), tensor(Q, at=FAR), tensor((64,), at=16 * FAR)
    odd, by_two = BASE + 1, BASE + 2

    def refused_address(fn, *a, **kw):
        assert "multiple of the element size" in refused(mb.ERR_INVALID_ARG, fn, *a, **kw)

    for b in (dict(cu_q=by_two), dict(kv_len=odd), dict(pages=by_two)):
        refused_address(mb.kv_cache_write, cache(), batch(**b), tensor(rows), tensor(rows))
        refused_address(mb.paged_attention, tensor(Q), cache(), batch(**b), out)
    refused_address(mb.kv_cache_write, cache(), batch(), tensor(rows, at=odd), tensor(rows))
    refused_address(mb.kv_cache_write, cache(), batch(), tensor(rows), tensor(rows, at=odd))
    refused_address(mb.kv_cache_read, cache(), batch(), by_two, tensor(rows), tensor(rows, at=FAR))
    refused_address(mb.kv_cache_read, cache(), batch(), BASE, tensor(rows), tensor(rows, at=FAR + 1))
    refused_address(mb.paged_attention, tensor(Q), cache(), batch(), out, lse=tensor((6, 4), mb.FLOAT32, at=2 * FAR + 2))
    for at, dtype in ((odd, mb.BFLOAT16), (by_two, mb.FLOAT32)):
        refused_address(mb.qk_norm_rope, tensor(Q, dtype, at=at), None, None, tensor(Q, dtype, at=FAR))
        refused_address(mb.qk_norm_rope, tensor(Q, dtype), None, None, tensor(Q, dtype, at=FAR + at - BASE))
        refused_address(mb.qk_norm_rope, tensor(Q, dtype), None, None, tensor(Q, dtype, at=FAR), q_weight=tensor((64,), dtype, at=16 * FAR + at - BASE))
    for rope in (mb.Rope(by_two, BASE, 64), mb.Rope(BASE, by_two, 64)):
        refused_address(mb.qk_norm_rope, tensor(Q), None, rope, out, q_weight=w)


def test_arrays_of_another_device_are_refused():
    """What a kernel would read of another device's memory: offsets, lengths, tables, positions and frequencies."""
    rows, far = tensor((6, 2, 64)), tensor((6, 2, 64), at=FAR)

    def there(**kw):
        return mb.KVBatch(2, 4, **(dict(cu_q=array([0, 1, 2]), kv_len=array([1, 1]), pages=array(np.zeros((2, 4)))) | kw))

    one = dict(cu_q=array([0, 1, 2], device=1), kv_len=array([1, 1], device=1), pages=array(np.zeros((2, 4)), device=1))
    for name in one:
        with pytest.raises(ValueError):
            there(**{name: one[name]})                                       # arrays of two devices in one batch
    with pytest.raises(ValueError):
        mb.Rope(array(np.arange(6)), array(np.ones(32), np.float32, device=1), 64)
    elsewhere, plain = there(**one), mb.KVBatch(2, 4, cu_q=BASE, kv_len=one["kv_len"], pages=BASE)
    rope = mb.Rope(array(np.arange(6), device=1), array(np.ones(32), np.float32, device=1), 64)
    for b in (elsewhere, plain):
        for call in (lambda: mb.kv_cache_write(cache(), b, rows, rows), lambda: mb.kv_cache_read(cache(), b, BASE, rows, far),
                     lambda: mb.paged_attention(tensor(Q), cache(), b, tensor(Q, at=FAR))):
            with pytest.raises(ValueError, match="one device"):
                call()
    with pytest.raises(ValueError, match="one device"):
        mb.kv_cache_read(cache(), there(), array([0, 1, 2], device=1), rows, far)
    with pytest.raises(ValueError, match="one device"):
        mb.qk_norm_rope(tensor(Q), None, rope, tensor(Q, at=FAR))
    if mb.device_count() == 0:
        refused(mb.ERR_NO_DEVICE, mb.kv_cache_write, cache(), batch(), rows, rows)    # plain pointers: nothing is known of them


@pytest.mark.parametrize("scale", [1e300, -1e39, 3e38])
def test_scales_past_fp32_are_refused(scale):
    """3e38 * log2(e), the factor of the scores, is past the largest number too."""
    assert "32 bits" in refused(mb.ERR_INVALID_ARG, mb.paged_attention, tensor(Q), cache(), batch(), tensor(Q, at=FAR), scale=scale)
