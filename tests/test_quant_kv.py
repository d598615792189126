"""The 8-bit paged cache: what it holds, and the attention over it, against the 64-bit oracle."""
import numpy as np
import pytest
import torch

from oracle import quant_oracle as qo
from unifiedkv_amd import compaction, decode_step, offload, prefill, quant_kv, staging
from unifiedkv_amd.quant_kv import QuantizedKVPool, QuantLayer

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
FMTS = ["int8", "fp8"]


# ------------------------------------------------------------------------------------ the oracle itself
@pytest.mark.parametrize("fmt", FMTS)
def test_oracle_holds_its_own_grid_and_bounds_its_error(fmt):
    rng = np.random.default_rng(1)
    x = rng.standard_normal((40, 64)) * 2.0 ** rng.integers(-12, 7, (40, 1))
    y, e = qo.quantise(x, fmt)
    again, e2 = qo.quantise(y, fmt)
    np.testing.assert_array_equal(y, again)  # writing what was read gives the same values
    step = 2.0 ** (np.repeat(e.astype(float), 32, -1) - 127)
    if fmt == "int8":
        assert np.all(np.abs(x - y) <= step / 2)
    else:  # three fraction bits: half a step is 2^-4 of the value; the smallest step is 2^-9
        assert np.all(np.abs(x - y) <= np.maximum(np.abs(x) * 2.0 ** -4, step * 2.0 ** -10))


def test_oracle_e4m3_matches_torchs_rounding():
    x = torch.cat([torch.linspace(-448, 448, 4001), torch.randn(4000) * 0.01])
    want = x.to(torch.float8_e4m3fn).double().numpy()
    rows = x.double().numpy()[:, None] * np.ones((1, 2))
    rows[:, 1] = 448.0  # exponent zero
    got, e = qo.quantise(rows, "fp8")
    assert np.all(e == 127)
    np.testing.assert_array_equal(got[:, 0], want)


# ------------------------------------------------------------------------------------ refusals (no GPU)
META = torch.device("meta")


def _meta_layer(N=8, H=2, D=64, fmt=torch.int8, dev=META, **over):
    t = dict(k=torch.empty((N, 16, H, D), dtype=fmt, device=dev), v=torch.empty((N, 16, H, D), dtype=fmt, device=dev),
             k_scale=torch.empty((N, H, -(-D // 32), 16), dtype=torch.uint8, device=dev),
             v_scale=torch.empty((N, H, -(-D // 32), 16), dtype=torch.uint8, device=dev))
    t.update(over)
    return t


def _m(*shape, dtype=torch.float16):
    return torch.empty(shape, dtype=dtype, device=META)


@pytest.mark.parametrize("over, what", [
    (dict(k=_m(8, 16, 2, 64)), "cache_dtype"),
    (dict(k=_m(8, 32, 2, 64, dtype=torch.int8)), "cache"),
    (dict(k=_m(16, 2, 64, dtype=torch.int8)), "cache"),
    (dict(v=_m(8, 16, 2, 64, dtype=torch.float8_e4m3fn)), "cache_dtype"),
    (dict(v=_m(9, 16, 2, 64, dtype=torch.int8)), "v_cache"),
    (dict(k_scale=_m(8, 2, 3, 16, dtype=torch.uint8)), "scale"),
    (dict(v_scale=_m(8, 16, 2, 2, dtype=torch.uint8)), "scale"),
    (dict(v_scale=_m(8, 2, 2, 16, dtype=torch.int8)), "scale_dtype"),
    (dict(k=_m(8, 16, 64, 2, dtype=torch.int8).transpose(2, 3)), "cache_stride"),
    (dict(k_scale=_m(8, 2, 16, 2, dtype=torch.uint8).transpose(2, 3)), "cache_stride"),
])
def test_layer_refusals(over, what):
    with pytest.raises(RuntimeError, match=f"^quant_kv_shape_unsupported:{what}$"):
        QuantLayer(**_meta_layer(**over))


def test_layer_of_two_devices_is_refused():
    t = _meta_layer()
    t["v_scale"] = torch.zeros((8, 2, 2, 16), dtype=torch.uint8)
    with pytest.raises(RuntimeError, match="quant_kv_unavailable:device"):
        QuantLayer(**t)


I32 = dict(dtype=torch.int32, device=META)


@pytest.mark.parametrize("call, what", [
    (lambda c: quant_kv.decode_attention(_m(3, 8), c, torch.empty((3, 4), **I32), torch.empty(3, **I32),
                                         softmax_scale=.1, n_rep=4), "shape_unsupported:q_dim_2"),
    (lambda c: quant_kv.decode_attention(_m(3, 8, 64, dtype=torch.float32), c, torch.empty((3, 4), **I32),
                                         torch.empty(3, **I32), softmax_scale=.1, n_rep=4), "shape_unsupported:dtype"),
    (lambda c: quant_kv.decode_attention(_m(3, 8, 128), c, torch.empty((3, 4), **I32), torch.empty(3, **I32),
                                         softmax_scale=.1, n_rep=4), "shape_unsupported:cache"),
    (lambda c: quant_kv.decode_attention(_m(3, 8, 64), c, torch.empty((3, 4), **I32), torch.empty(3, **I32),
                                         softmax_scale=.1, n_rep=3), "shape_unsupported:gqa"),
    (lambda c: quant_kv.decode_attention(_m(3, 8, 64), c, torch.empty((3, 4), **I32), torch.empty(3, **I32),
                                         softmax_scale=.1, n_rep=4), "unavailable:device"),
    (lambda c: quant_kv.prefill_attention(_m(9, 8, 64), c, torch.empty((3, 4), **I32), [0, 3, 6, 9], [3, 3, 3],
                                          softmax_scale=.1, n_rep=0), "shape_unsupported:gqa"),
    (lambda c: quant_kv.prefill_attention(_m(9, 64, 8).transpose(1, 2), c, torch.empty((3, 4), **I32), [0, 3, 6, 9],
                                          [3, 3, 3], softmax_scale=.1, n_rep=4), "shape_unsupported:stride"),
    (lambda c: quant_kv.append_kv(c, _m(3, 2, 64), _m(3, 1, 64), torch.empty((3, 4), **I32), torch.empty(3, **I32)),
     "shape_unsupported:rows"),
    (lambda c: quant_kv.append_kv(c, _m(3, 2, 2, 64), _m(3, 2, 2, 64), torch.empty((3, 4), **I32),
                                  torch.empty(3, **I32)), "shape_unsupported:rows"),
    (lambda c: quant_kv.append_kv(c, _m(3, 2, 64), _m(3, 2, 64, dtype=torch.bfloat16), torch.empty((3, 4), **I32),
                                  torch.empty(3, **I32)), "shape_unsupported:dtype"),
    (lambda c: quant_kv.write_chunk_kv(c, _m(9, 2, 32), _m(9, 2, 32), torch.empty((3, 4), **I32), [0, 3, 6, 9],
                                       [3, 3, 3]), "shape_unsupported:rows"),
    (lambda c: quant_kv.write_chunk_kv(c, _m(9, 64, 2).transpose(1, 2), _m(9, 64, 2).transpose(1, 2),
                                       torch.empty((3, 4), **I32), [0, 3, 6, 9], [3, 3, 3]), "shape_unsupported:stride"),
    (lambda c: quant_kv.write_chunk_kv(c, _m(9, 2, 64), _m(9, 2, 64), torch.empty((3, 4), **I32), [0, 3, 6, 9],
                                       [3, 3, 3]), "unavailable:device"),
    (lambda c: quant_kv.read_kv(c, torch.empty((3, 4), **I32), [0, 3, 6, 9], [3, 3, 3], dtype=torch.float32),
     "shape_unsupported:dtype"),
    (lambda c: quant_kv.read_kv(c, torch.empty((3, 4), **I32), [0, 3, 6, 9], [3, 3, 3], dtype=torch.float16),
     "unavailable:device"),
])
def test_calls_refuse_before_a_launch(call, what):
    with pytest.raises(RuntimeError, match=f"^quant_kv_{what}$"):
        call(QuantLayer(**_meta_layer()))


def test_c_entry_points_refuse_bad_arguments():
    from unifiedkv_amd import _ext

    lib, s, q2, r4 = _ext.load(), _ext.i64_array([1] * 12), _ext.i64_array([1, 1]), _ext.i64_array([1] * 4)

    def decode(batch=1, Hq=4, Hkv=1, D=64, n_rep=4, blocks=1, fmt=0, dtype=0, q=16):
        return lib.ukv_quant_decode(q, 16, 16, 16, 16, s, 1, 16, 16, 16, batch, Hq, Hkv, D, n_rep, blocks, q2, 0.1, fmt,
                                    dtype, None, 0, None)

    assert decode(batch=0) == _ext.UKV_ERR_EMPTY
    assert decode(D=257) == _ext.UKV_ERR_HEAD_DIM
    assert decode(fmt=2) == _ext.UKV_ERR_DTYPE and decode(dtype=2) == _ext.UKV_ERR_DTYPE
    assert decode(n_rep=3) == _ext.UKV_ERR_GQA and decode(n_rep=0) == _ext.UKV_ERR_GQA
    assert decode(q=None) == _ext.UKV_ERR_INVALID_ARGUMENT
    assert decode(blocks=-1) == _ext.UKV_ERR_INVALID_ARGUMENT
    assert decode(blocks=1 << 28) == _ext.UKV_ERR_INVALID_ARGUMENT
    s16 = _ext.i64_array([1024] * 12)
    assert lib.ukv_quant_decode(16, 16, 16, 16, 16, s16, 1, 16, 16, 16, 65536, 4, 1, 64, 4, 1, _ext.i64_array([256, 64]),
                                0.1, 0, 0, None, 0, None) == _ext.UKV_ERR_INVALID_ARGUMENT

    def write(fmt=0, dtype=0, heads=1, table=16, rows=16, batch=1, chunk=1):
        return lib.ukv_quant_kv_write(16, 16, 16, 16, s, 1, rows, rows, r4, table, 1, None, None, 0, batch, chunk, heads,
                                      64, fmt, dtype, None)

    assert write(fmt=7) == _ext.UKV_ERR_DTYPE and write(dtype=3) == _ext.UKV_ERR_DTYPE
    for bad in (dict(heads=0), dict(table=None), dict(rows=None), dict(batch=65536), dict(batch=1 << 15, chunk=1 << 16)):
        assert write(**bad) == _ext.UKV_ERR_INVALID_ARGUMENT
    assert lib.ukv_quant_prefill(16, 16, 16, 16, 16, s, 1, 16, None, 16, 16, 1, 4, 4, 4, 1, 64, 4, 1, q2, 0.1, 0, 0, None,
                                 0, None) == _ext.UKV_ERR_INVALID_ARGUMENT
    for i in range(8):  # nothing to attend: no scratch
        assert lib.ukv_quant_prefill_workspace_bytes(*[0 if j == i else 4 for j in range(8)]) == 0 or i == 5
    assert lib.ukv_quant_prefill_workspace_bytes(4, 8, 2, 8, 2, 64, 4, 4) > 0


def test_pool_refusals():
    with pytest.raises(ValueError, match="cache_format"):
        QuantizedKVPool(16, 1, 2, 64, cache_format="int4", num_blocks=4, device="cpu")
    with pytest.raises(RuntimeError, match="block_size_32"):
        QuantizedKVPool(32, 1, 2, 64, num_blocks=4, device="cpu")
    with pytest.raises(RuntimeError, match="dtype"):
        QuantizedKVPool(16, 1, 2, 64, torch.float32, num_blocks=4, device="cpu")
    pool = QuantizedKVPool(16, 2, 2, 64, num_blocks=8, device="cpu")
    free = pool.free_blocks
    for call in (lambda: pool.k_cache, lambda: pool.v_cache,
                 lambda: compaction.selected_writeback(pool, [], {}, 16, "x", sink_len=0, obs_len=0),
                 lambda: compaction.write_block_indexed_layer(pool, 0, [0], _m(2, 16, 64), _m(2, 16, 64), [0]),
                 lambda: compaction.compact_selected(pool, [[0]], [16], [None], sink_len=0, obs_len=0),
                 lambda: compaction.prune_window(pool, [0, 1], 32, [0]),
                 lambda: staging.PageStager(pool), lambda: offload.SequenceOffloader(pool, arena_pages=4),
                 lambda: offload.PinnedArena(pool, 4)):
        with pytest.raises(RuntimeError, match="quant_kv_shape_unsupported"):
            call()
    assert pool.free_blocks == free  # nothing was taken
    with pytest.raises(IndexError):
        pool.layer(2)
    assert pool.layer(1).k.shape == (8, 16, 2, 64) and pool.layer(1).k_scale.shape == (8, 2, 2, 16)
    assert pool._bytes_per_block() == 2 * 2 * 16 * 2 * (64 + 2)


# ------------------------------------------------------------------------------------ on the GPU
def _rows(rng, n, H, D, dtype, special=True):
    """Rows over many magnitudes; with the values at which a quantiser goes wrong."""
    x = rng.standard_normal((n, H, D)) * 2.0 ** rng.integers(-20, 10, (n, H, 1))
    x[..., ::3] *= 8
    t = torch.from_numpy(x).to(dtype)
    if special and n >= 12:
        t[0] = 0
        t[1, 0, 0], t[1, -1, D - 1] = float("nan"), float("inf")
        t[2, :, :] = 1.0 / 127 * torch.arange(D) * 64  # ties of int8
        t[3] = torch.finfo(dtype).tiny
        t[4] = torch.finfo(dtype).max
        t[5] = -torch.finfo(dtype).max
        t[6] = torch.finfo(dtype).smallest_normal / 4
        t[7, :, ::2], t[7, :, 1::2] = 448.0, 449.0
        t[8, :, ::2], t[8, :, 1::2] = 127.0, -127.5
        t[9] = (17.0 + torch.arange(D) % 16) / 16 * 448 / 2  # ties of e4m3
        t[10] = -0.0
        t[11, :, 0] = float("-inf")
    return t


def _layer(cuda, fmt, N, H, D, layout="plain", fill=0x35):
    """A cache full of codes that must not matter, in several layouts."""
    nb, of = -(-D // 32), quant_kv.FORMATS[fmt]

    def codes():
        return torch.full((N, 16, H, D), fill, dtype=torch.uint8, device=cuda)

    def scales():
        return torch.full((N, H, nb, 16), 255, dtype=torch.uint8, device=cuda)

    k, v, ks, vs = codes(), codes(), scales(), scales()
    if layout == "interleaved":  # K and V halves of one page, padded heads
        both = torch.full((N, 2, 16, H, D + 16), fill, dtype=torch.uint8, device=cuda)
        k, v = both[:, 0, :, :, :D], both[:, 1, :, :, :D]
        exps = torch.full((N, 2, nb, H, 16), 255, dtype=torch.uint8, device=cuda)
        ks, vs = exps[:, 0].transpose(1, 2), exps[:, 1].transpose(1, 2)
    elif layout == "odd":  # rows that no wide access takes
        k = torch.full((N * 16 * H * D + 1,), fill, dtype=torch.uint8, device=cuda)[1:].view(N, 16, H, D)
        ks = torch.full((N, H, nb, 17), 255, dtype=torch.uint8, device=cuda)[..., 1:]
    elif layout == "heads_first":  # [N, H, 16, D]
        k, v = (torch.full((N, H, 16, D), fill, dtype=torch.uint8, device=cuda).transpose(1, 2) for _ in range(2))
    return QuantLayer(k.view(of), v.view(of), ks, vs)


def _bits(layer):
    return [x.view(torch.uint8).cpu().numpy().copy() for x in (layer.k, layer.v)] + \
        [x.cpu().numpy().copy() for x in (layer.k_scale, layer.v_scale)]


def _values(layer, fmt):
    k, v, ks, vs = _bits(layer)
    return qo.held(k, ks.transpose(0, 3, 1, 2), fmt), qo.held(v, vs.transpose(0, 3, 1, 2), fmt)


def _tables(rng, N, lens, extra=1):
    counts = [-(-n // 16) for n in lens]
    perm = rng.permutation(N)[:sum(counts)]
    table = np.zeros((len(lens), max(counts) + extra), dtype=np.int32)
    at = 0
    for row, n in zip(table, counts):
        row[:n] = perm[at:at + n]
        at += n
    return table


def _dev(x, cuda, dtype=torch.int32):
    return torch.as_tensor(np.asarray(x), dtype=dtype).to(cuda)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H, D, layout", [(8, 128, "plain"), (4, 64, "plain"), (3, 96, "interleaved"), (2, 256, "plain"),
                                          (2, 80, "plain"), (5, 33, "plain"), (1, 128, "odd"), (2, 64, "heads_first"),
                                          (1, 1, "plain")])
def test_write_holds_what_the_format_says_and_reads_back(cuda, fmt, dtype, H, D, layout):
    rng = np.random.default_rng(D + H)
    dt = DTYPES[dtype]
    pre, chunk = [0, 5, 31, 16, 100], [40, 1, 17, 0, 29]
    lens = [p + c for p, c in zip(pre, chunk)]
    table = _tables(rng, 40, lens)
    layer = _layer(cuda, fmt, 40, H, D, layout)
    before = _bits(layer)
    k, v = _rows(rng, sum(chunk), H, D, dt), _rows(rng, sum(chunk), H, D, dt)
    cu = np.concatenate([[0], np.cumsum(chunk)])
    quant_kv.write_chunk_kv(layer, k.to(cuda), v.to(cuda), _dev(table, cuda), _dev(cu, cuda), _dev(lens, cuda),
                            max_chunk=max(chunk))
    got = _values(layer, fmt)
    after = _bits(layer)
    touched = np.zeros((40, 16), dtype=bool)
    for x, y, e_got in ((k, got[0], after[2]), (v, got[1], after[3])):
        want, exps = qo.quantise(x.double().numpy(), fmt)
        for b, (p, c) in enumerate(zip(pre, chunk)):
            for i in range(c):
                page, slot = table[b, (p + i) // 16], (p + i) % 16
                touched[page, slot] = True
                np.testing.assert_array_equal(y[page, slot], want[cu[b] + i])
                np.testing.assert_array_equal(e_got[page, :, :, slot], exps[cu[b] + i])
    for x, y in zip(before[:2], after[:2]):  # every other slot as it was
        np.testing.assert_array_equal(x[~touched], y[~touched])
    for x, y in zip(before[2:], after[2:]):
        np.testing.assert_array_equal(x.transpose(0, 3, 1, 2)[~touched], y.transpose(0, 3, 1, 2)[~touched])
    # reading: exact in either type, whole sequences and windows, from host and device lengths
    for out in DTYPES.values():
        rk, rv = quant_kv.read_kv(layer, _dev(table, cuda), _dev(cu, cuda), _dev(lens, cuda), dtype=out,
                                  max_chunk=max(chunk), total=sum(chunk))
        hk, hv = quant_kv.read_kv(layer, _dev(table, cuda), list(cu), lens, dtype=out)
        for x, r, again in ((k, rk, hk), (v, rv, hv)):
            np.testing.assert_array_equal(r.double().cpu().numpy(), qo.quantise(x.double().numpy(), fmt)[0])
            assert r.dtype == out and torch.equal(r.view(torch.int16), again.view(torch.int16))


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FMTS)
def test_append_equals_a_chunk_of_one_and_skips_bad_pages(cuda, fmt):
    rng = np.random.default_rng(7)
    old = [0, 15, 16, 47, 64, 30]
    table = _tables(rng, 30, [n + 1 for n in old], extra=0)
    table[5, 1] = 30  # outside the pool: not written
    k, v = (_rows(rng, 6, 4, 128, torch.bfloat16, special=False).to(cuda) for _ in range(2))
    a, b = _layer(cuda, fmt, 30, 4, 128), _layer(cuda, fmt, 30, 4, 128)
    wide = torch.stack([k, v], 2)  # rows that are not contiguous
    quant_kv.append_kv(a, wide[:, :, 0], wide[:, :, 1], _dev(table, cuda, torch.int64), _dev(old, cuda, torch.int64))
    quant_kv.write_chunk_kv(b, k, v, _dev(table, cuda), list(range(7)), [n + 1 for n in old])
    for x, y in zip(_bits(a), _bits(b)):
        np.testing.assert_array_equal(x, y)
    rk, rv = quant_kv.read_kv(a, _dev(table, cuda), list(range(7)), [n + 1 for n in old], dtype=torch.bfloat16)
    assert not rk[5].any() and not rv[5].any() and rk[:5].abs().amax(-1).min() > 0
    # lengths outside the table write nothing
    before = _bits(a)
    quant_kv.append_kv(a, k, v, _dev(table, cuda), _dev([16 * table.shape[1]] * 3 + [-1, -5, 1 << 30], cuda))
    for x, y in zip(before, _bits(a)):
        np.testing.assert_array_equal(x, y)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("H, D", [(1, 32), (1, 64), (3, 32), (1, 128), (8, 128)])
def test_whole_pages_outside_the_pool_are_left_alone(cuda, fmt, H, D):
    """Pages whose sixteen tokens are all written, with ids below and above the pool's, between good ones."""
    rng = np.random.default_rng(H * D)
    N, n = 12, 16 * 7 + 3
    table = np.array([[3, -1, 5, N, 11, 1 << 30, 0, 7]], dtype=np.int32)
    layer = _layer(cuda, fmt, N, H, D)
    before = _bits(layer)
    rows = [torch.from_numpy(rng.standard_normal((n, H, D))).half() for _ in range(2)]
    quant_kv.write_chunk_kv(layer, rows[0].to(cuda), rows[1].to(cuda), _dev(table, cuda), [0, n], [n])
    good = [(i, p) for i, p in enumerate(table[0]) if 0 <= p < N]
    rest = [p for p in range(N) if p not in table[0]]
    for x, y, e in zip(rows, _values(layer, fmt), _bits(layer)[2:]):
        want, exps = qo.quantise(x.double().numpy(), fmt)
        for i, p in good:
            m = min(16, n - 16 * i)
            np.testing.assert_array_equal(y[p, :m], want[16 * i:16 * i + m])
            np.testing.assert_array_equal(e[p].transpose(2, 0, 1)[:m], exps[16 * i:16 * i + m])
    for x, y in zip(before, _bits(layer)):
        np.testing.assert_array_equal(x[rest], y[rest])
    back = quant_kv.read_kv(layer, _dev(table, cuda), [0, n], [n], dtype=torch.float16)
    for r in back:
        for i in (1, 3, 5):
            assert not r[16 * i:16 * i + 16].any()


def _bound(out, spread, v, q, k, scale, dtype, weight):
    """How far a result may be off: half a step of its type, then what the weights may be off by, in units of
    sum(p |v|) and once more for their sum. A weight is off by its own rounding (``weight``, relative), by the
    error of its score (a dot product in fp32 of at most D terms, its scaling and the running maximum's
    subtraction, relative to sum |q k|, and two exponentials' 2^-21) and by the fp32 sums over T keys; weights under
    2^-14 of the largest are held in steps of fp16's smallest number, 2^-25 off at most."""
    T, D = k.shape
    half = torch.finfo(dtype).eps / 2
    score = (D + 8) * 2.0 ** -24 * (np.abs(k) @ np.abs(q)).max() * abs(scale) * 1.5
    rel = 2 * (weight + score + 2.0 ** -20 + (T + 64) * 2.0 ** -24)
    tiny = 2.0 ** -24 if dtype == torch.float16 else 0.0
    return half * np.abs(out) * 1.01 + rel * spread * 1.05 + 2.0 ** -24 * np.abs(v).sum(0) + tiny


def _check_rows(got, layer, fmt, q, table, spans, scale, n_rep, weight, num_pages):
    """Each (row, b, keys) of spans against the oracle over the values that the cache holds."""
    kv, vv = _values(layer, fmt)
    got, q64 = got.double().cpu().numpy(), q.double().cpu().numpy()
    for row, b, n in spans:
        ids = table[b, :-(-n // 16)].astype(np.int64)
        ok = np.repeat((ids >= 0) & (ids < num_pages), 16)[:n]
        ids = np.where((ids >= 0) & (ids < num_pages), ids, 0)
        for h in range(q64.shape[1]):
            k, v = (x[ids, :, h // n_rep].reshape(-1, x.shape[-1])[:n][ok] for x in (kv, vv))
            with np.errstate(invalid="ignore"):
                want, spread = qo.attend(q64[row, h], k, v, scale)
            bad = np.isnan(want)
            np.testing.assert_array_equal(np.isnan(got[row, h]), bad, err_msg=f"row {row} head {h}")
            if bad.all():
                continue
            off = np.abs(got[row, h] - want)[~bad]
            tol = _bound(want, spread, v, q64[row, h], k, scale, q.dtype, weight)[~bad]
            assert np.all(off <= tol), (row, h, n, float((off / tol).max()))


# Weights enter P.V in two 16-bit parts (decode) or as one fp16 number (chunks): 2^-16 and 2^-11 relative.
DECODE_WEIGHT, CHUNK_WEIGHT = 2.0 ** -16, 2.0 ** -11

HEADS = [(8, 4, 128), (4, 7, 128), (1, 8, 128), (2, 1, 64), (8, 4, 64), (3, 16, 128), (2, 2, 256), (2, 3, 96), (1, 17, 64),
         (12, 1, 128), (2, 4, 40)]


def _filled(cuda, fmt, dt, rng, N, H, D, layout="plain"):
    """A cache whose every page holds rows of one magnitude (and some channels of a larger one)."""
    layer = _layer(cuda, fmt, N, H, D, layout)
    gen = torch.Generator().manual_seed(int(rng.integers(1 << 30)))
    k, v = (torch.randn((N * 16, H, D), generator=gen) for _ in range(2))
    k *= torch.exp(torch.randn((H, D), generator=gen) * 0.5)
    quant_kv.write_chunk_kv(layer, k.to(dt).to(cuda), v.to(dt).to(cuda), torch.arange(N, device=cuda)[None],
                            [0, 16 * N], [16 * N])
    return layer


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H, n_rep, D", HEADS)
def test_decode_matches_the_oracle(cuda, fmt, dtype, H, n_rep, D):
    rng = np.random.default_rng(100 * H + n_rep + D)
    dt = DTYPES[dtype]
    lens = [1, 15, 16, 17, 333, 0, 64, 129]
    layer = _filled(cuda, fmt, dt, rng, 64, H, D)
    table = _tables(rng, 64, lens)
    q = torch.from_numpy(rng.standard_normal((len(lens), H * n_rep, D))).to(dt).to(cuda)
    scale = D ** -0.5
    got = quant_kv.decode_attention(q, layer, _dev(table, cuda), _dev(lens, cuda), softmax_scale=scale, n_rep=n_rep)
    assert got.dtype == dt and got.shape == q.shape
    _check_rows(got, layer, fmt, q, table, [(b, b, n) for b, n in enumerate(lens)], scale, n_rep, DECODE_WEIGHT, 64)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("batch, lo, hi, H, n_rep", [(1, 20000, 20000, 8, 4), (3, 5000, 9000, 1, 4), (70, 1, 700, 2, 4),
                                                     (5, 1, 6000, 4, 7), (2, 3000, 3000, 16, 2)])
def test_decode_long_and_ragged_batches(cuda, fmt, batch, lo, hi, H, n_rep):
    rng = np.random.default_rng(batch)
    lens = [int(x) for x in rng.integers(lo, hi, size=batch, endpoint=True)]
    N = sum(-(-n // 16) for n in lens) + 3
    layer = _filled(cuda, fmt, torch.bfloat16, rng, N, H, 128)
    table = _tables(rng, N, lens, extra=5)
    q = torch.from_numpy(rng.standard_normal((batch, H * n_rep, 128))).bfloat16().to(cuda)
    got = quant_kv.decode_attention(q, layer, _dev(table, cuda), _dev(lens, cuda), softmax_scale=0.1, n_rep=n_rep)
    some = sorted(set([0, batch - 1] + [int(x) for x in rng.integers(0, batch, 4)]))
    _check_rows(got, layer, fmt, q, table, [(b, b, lens[b]) for b in some], 0.1, n_rep, DECODE_WEIGHT, N)
    # the same call again gives the same bits
    again = quant_kv.decode_attention(q, layer, _dev(table, cuda), _dev(lens, cuda), softmax_scale=0.1, n_rep=n_rep)
    assert torch.equal(got.view(torch.int16), again.view(torch.int16))


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("layout", ["interleaved", "odd", "heads_first"])
def test_attention_takes_other_layouts(cuda, fmt, layout):
    rng = np.random.default_rng(3)
    lens, H, R, D = [77, 16, 130], 2, 4, 128
    layer = _filled(cuda, fmt, torch.float16, rng, 30, H, D, layout)
    table = _tables(rng, 30, lens)
    wide = torch.from_numpy(rng.standard_normal((3, 2 * H * R, D + 8))).half().to(cuda)
    q = wide[:, ::2, :D]  # strided heads and rows
    got = quant_kv.decode_attention(q, layer, _dev(table, cuda), _dev(lens, cuda), softmax_scale=0.1, n_rep=R)
    spans = [(b, b, n) for b, n in enumerate(lens)]
    _check_rows(got, layer, fmt, q, table, spans, 0.1, R, DECODE_WEIGHT, 30)
    got = quant_kv.prefill_attention(q, layer, _dev(table, cuda), [0, 1, 2, 3], lens, softmax_scale=0.1, n_rep=R)
    _check_rows(got, layer, fmt, q, table, spans, 0.1, R, CHUNK_WEIGHT, 30)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H, n_rep, D", HEADS)
def test_chunks_match_the_oracle(cuda, fmt, dtype, H, n_rep, D):
    rng = np.random.default_rng(10 * H + n_rep + D)
    dt = DTYPES[dtype]
    pre, chunk = [0, 40, 7, 100, 0, 300], [33, 5, 0, 1, 1, 16]
    lens = [p + c for p, c in zip(pre, chunk)]
    layer = _filled(cuda, fmt, dt, rng, 64, H, D)
    table = _tables(rng, 64, lens)
    cu = np.concatenate([[0], np.cumsum(chunk)])
    q = torch.from_numpy(rng.standard_normal((sum(chunk), H * n_rep, D))).to(dt).to(cuda)
    scale = D ** -0.5
    got = quant_kv.prefill_attention(q, layer, _dev(table, cuda), _dev(cu, cuda), _dev(lens, cuda), softmax_scale=scale,
                                     n_rep=n_rep, max_chunk=max(chunk))
    spans = [(cu[b] + i, b, pre[b] + i + 1) for b in range(len(pre)) for i in range(chunk[b])]
    _check_rows(got, layer, fmt, q, table, spans, scale, n_rep, CHUNK_WEIGHT, 64)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("pre, chunk, H, n_rep, D", [
    ([6000], [389], 2, 4, 128), ([9000, 3], [4, 700], 1, 4, 128), ([2000, 0, 500], [130, 400, 1], 4, 7, 128),
    ([0] * 5, [1, 350, 64, 65, 200], 2, 2, 64), ([4000] * 8, [3, 8, 1, 5, 2, 7, 4, 6], 2, 4, 128)])
def test_long_chunks_match_the_oracle(cuda, fmt, pre, chunk, H, n_rep, D):
    rng = np.random.default_rng(sum(chunk))
    lens = [p + c for p, c in zip(pre, chunk)]
    N = sum(-(-n // 16) for n in lens) + 2
    layer = _filled(cuda, fmt, torch.float16, rng, N, H, D)
    table = _tables(rng, N, lens, extra=0)
    cu = np.concatenate([[0], np.cumsum(chunk)])
    for dt in DTYPES.values():
        q = torch.from_numpy(rng.standard_normal((sum(chunk), H * n_rep, D))).to(dt).to(cuda)
        got = quant_kv.prefill_attention(q, layer, _dev(table, cuda), list(cu), lens, softmax_scale=0.1, n_rep=n_rep)
        spans = [(cu[b] + i, b, pre[b] + i + 1) for b in range(len(pre))
                 for i in sorted({0, chunk[b] - 1, chunk[b] // 2, chunk[b] // 3})]
        _check_rows(got, layer, fmt, q, table, spans, 0.1, n_rep, CHUNK_WEIGHT, N)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("batch, most, lo, hi, H, n_rep, D", [
    (70, 4, 1, 700, 2, 4, 128), (70, 8, 1, 700, 6, 4, 128), (66, 3, 1, 300, 3, 5, 64), (3, 2, 100, 900, 12, 8, 64),
    (40, 5, 300, 600, 9, 6, 64), (2, 1, 1, 5000, 2, 16, 128), (5, 3, 60000, 65000, 5, 4, 64),
    (4, 7, 66000, 70000, 6, 4, 128)])
def test_few_queries_a_sequence_over_ragged_lengths(cuda, fmt, batch, most, lo, hi, H, n_rep, D):
    """Drafted tokens: chunks of none to ``most`` queries, more sequences than a wave has lanes, more KV heads than a
    workgroup has waves, more pages a wave than its lanes hold ids of. Sequences share pages."""
    rng = np.random.default_rng(batch + H)
    N = 300
    layer = _filled(cuda, fmt, torch.bfloat16, rng, N, H, D)
    lens = [int(x) for x in rng.integers(lo, hi, size=batch, endpoint=True)]
    chunk = [min(n, int(c)) for n, c in zip(lens, rng.integers(0, most, size=batch, endpoint=True))]
    chunk[-1] = min(lens[-1], most)
    table = rng.integers(0, N, size=(batch, -(-max(lens) // 16) + 2)).astype(np.int32)
    table[batch // 2, 0] = N  # sixteen keys without a page
    cu = np.concatenate([[0], np.cumsum(chunk)])
    some = sorted({0, 1, batch // 2, batch - 1} | {int(x) for x in rng.integers(0, batch, 3)})
    spans = [(cu[b] + i, b, lens[b] - chunk[b] + i + 1) for b in some for i in sorted({0, chunk[b] - 1}) if 0 <= i < chunk[b]]
    for dt in DTYPES.values():
        q = torch.from_numpy(rng.standard_normal((sum(chunk), H * n_rep, D))).to(dt).to(cuda)
        got = quant_kv.prefill_attention(q, layer, _dev(table, cuda), _dev(cu, cuda), _dev(lens, cuda), softmax_scale=0.1,
                                         n_rep=n_rep, max_chunk=most)
        _check_rows(got, layer, fmt, q, table, spans, 0.1, n_rep, CHUNK_WEIGHT, N)
    dq = torch.from_numpy(rng.standard_normal((batch, H * n_rep, D))).half().to(cuda)
    got = quant_kv.decode_attention(dq, layer, _dev(table, cuda), _dev(lens, cuda), softmax_scale=0.1, n_rep=n_rep)
    _check_rows(got, layer, fmt, dq, table, [(b, b, lens[b]) for b in some], 0.1, n_rep, DECODE_WEIGHT, N)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("most, H, n_rep, D", [(3, 2, 4, 128), (8, 2, 4, 128), (4, 8, 4, 64), (6, 5, 4, 64)])
def test_nan_blocks_among_few_queries(cuda, fmt, most, H, n_rep, D):
    """A NaN block at every place of the chunk and right before it: only the queries that see it turn NaN, in the
    value's block's dims alone, and every one where a key holds it."""
    rng = np.random.default_rng(most)
    batch = 16
    layer = _filled(cuda, fmt, torch.float16, rng, 40 * batch, H, D)
    lens, chunk = [500 + 3 * b for b in range(batch)], [most] * batch
    table = _tables(rng, 40 * batch, lens, extra=64 - 35)  # (a table wide enough for two column blocks)
    bad = torch.ones((1, H, D), dtype=torch.float16, device=cuda)
    bad[:, :, 32:64] = float("inf")
    for b in range(batch):
        pos = lens[b] - most + b // 2 - 1
        if pos < lens[b]:
            rows = (bad, torch.ones_like(bad)) if b % 2 else (torch.ones_like(bad), bad)
            quant_kv.write_chunk_kv(layer, *rows, _dev(table[b:b + 1], cuda), [0, 1], [pos + 1])
    cu = np.arange(batch + 1) * most
    q = torch.from_numpy(rng.standard_normal((batch * most, H * n_rep, D))).half().to(cuda)
    got = quant_kv.prefill_attention(q, layer, _dev(table, cuda), _dev(cu, cuda), _dev(lens, cuda), softmax_scale=0.1,
                                     n_rep=n_rep, max_chunk=most)
    spans = [(cu[b] + i, b, lens[b] - most + i + 1) for b in range(batch) for i in range(most)]
    _check_rows(got, layer, fmt, q, table, spans, 0.1, n_rep, CHUNK_WEIGHT, 40 * batch)


def _in_shares(batch, total, most, H, n_rep, D, width):
    """Whether a call's keys are cut by its lengths on the device (its partials are of that size, whatever the call's)."""
    from unifiedkv_amd import _ext

    need = _ext.load().ukv_quant_prefill_workspace_bytes(batch, total, most, H * n_rep, H, D, n_rep, width)
    slots = 256 * (2 if D == 64 else 1)
    return any(2 * slots * 128 * cb * (4 * D + 8) <= need < 2 * slots * 128 * cb * (4 * D + 8) + 8192 for cb in (1, 2, 3))


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("pre, chunk, H, n_rep, D, width", [
    ([9000, 300, 0, 4000, 17], [200, 150, 33, 1, 0], 2, 4, 128, 2600),
    ([700, 12000, 0, 40], [1, 120, 120, 77], 2, 7, 128, 3500),
    ([30000, 5, 0, 2000, 900], [256, 200, 256, 31, 0], 2, 4, 64, 3400),
    ([60, 0, 14000, 1000, 333, 1], [90, 90, 17, 64, 2, 90], 3, 5, 64, 3800),
    ([3000 + 400 * (i % 9) for i in range(40)], [1 + i % 10 for i in range(40)], 1, 16, 128, 2100),
    ([150 * i for i in range(30)], [(7 * i) % 25 for i in range(30)], 4, 8, 64, 1200),
    ([0, 3], [1, 2], 1, 4, 128, 3200),
    ([0, 0, 0], [0, 0, 3], 1, 4, 128, 2200)])
def test_chunks_in_shares(cuda, fmt, pre, chunk, H, n_rep, D, width):
    """Tables wide enough that the lengths on the device cut the work: blocks in one piece and in many, sequences
    without queries, queries without keys, fewer tiles than workgroups. Sequences share pages."""
    rng = np.random.default_rng(sum(pre) + D)
    N, batch = 250, len(pre)
    most = max(chunk) if max(chunk) > 3 else 2000  # (declared longer than they are)
    lens = [p + c for p, c in zip(pre, chunk)]
    layer = _filled(cuda, fmt, torch.bfloat16, rng, N, H, D)
    table = rng.integers(0, N, size=(batch, width)).astype(np.int32)
    table[batch // 2, 1] = -5  # keys without a page
    table[0, 3] = N
    cu = np.concatenate([[0], np.cumsum(chunk)])
    assert _in_shares(batch, sum(chunk), most, H, n_rep, D, width)
    some = sorted({0, 1, min(2, batch - 1), batch - 1} | {int(x) for x in rng.integers(0, batch, 3)})
    spans = [(cu[b] + i, b, lens[b] - chunk[b] + i + 1) for b in some
             for i in sorted({0, chunk[b] // 3, chunk[b] // 2, chunk[b] - 1}) if 0 <= i < chunk[b]]
    short = [max(0, n - c // 2 - 1) for n, c in zip(lens, chunk)]  # kv_lens below the chunk's: queries before key 0
    for dt in DTYPES.values():
        q = torch.from_numpy(rng.standard_normal((sum(chunk), H * n_rep, D))).to(dt).to(cuda)
        got = quant_kv.prefill_attention(q, layer, _dev(table, cuda), _dev(cu, cuda), _dev(lens, cuda), softmax_scale=0.1,
                                         n_rep=n_rep, max_chunk=most)
        _check_rows(got, layer, fmt, q, table, spans, 0.1, n_rep, CHUNK_WEIGHT, N)
        again = quant_kv.prefill_attention(q, layer, _dev(table, cuda), _dev(cu, cuda), _dev(lens, cuda),
                                           softmax_scale=0.1, n_rep=n_rep, max_chunk=most)
        assert torch.equal(got.view(torch.int16), again.view(torch.int16))
        if min(pre) == 0:
            got = quant_kv.prefill_attention(q, layer, _dev(table, cuda), _dev(cu, cuda), _dev(short, cuda),
                                             softmax_scale=0.1, n_rep=n_rep, max_chunk=most)
            rows = [(r, b, max(0, n + short[b] - lens[b])) for r, b, n in spans]
            _check_rows(got, layer, fmt, q, table, rows, 0.1, n_rep, CHUNK_WEIGHT, N)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("n_rep, D, width", [(4, 128, 4200), (7, 128, 2200), (4, 64, 5600)])
def test_shares_with_nan_blocks_and_a_chunk_longer_than_declared(cuda, fmt, n_rep, D, width):
    rng = np.random.default_rng(D)
    H, N, pre, chunk, most = 2, 300, [1500, 700, 4000, 90], [180, 200, 150, 160], 180
    lens = [p + c for p, c in zip(pre, chunk)]
    layer = _filled(cuda, fmt, torch.float16, rng, N, H, D)
    table = np.zeros((4, width), dtype=np.int32)
    table[:, :300] = rng.integers(0, 290, size=(4, 300))
    table[0, lens[0] // 16], table[2, 60], table[3, 14] = 291, 292, 293  # pages of their own
    bad = torch.ones((1, H, D), dtype=torch.float16, device=cuda)
    bad[:, :, 32:] = float("nan")
    one = torch.ones_like(bad)
    for b, pos, rows in ((0, lens[0], (bad, bad)), (2, 960, (one, bad)), (3, 230, (bad, one))):
        quant_kv.write_chunk_kv(layer, *rows, _dev(table[b:b + 1], cuda), [0, 1], [pos + 1])
    cu = np.concatenate([[0], np.cumsum(chunk)])
    q = torch.from_numpy(rng.standard_normal((sum(chunk) + 5, H * n_rep, D))).half().to(cuda)
    assert _in_shares(4, sum(chunk) + 5, most, H, n_rep, D, width)
    args = (layer, _dev(table, cuda), _dev(cu, cuda), _dev(lens, cuda))

    def call():
        return quant_kv.prefill_attention(q, *args, softmax_scale=0.1, n_rep=n_rep, max_chunk=most)

    got = call()
    assert torch.isnan(got[cu[1]:cu[2]]).all()  # longer than declared
    spans = [(cu[b] + i, b, pre[b] + i + 1) for b in (0, 2, 3)
             for i in sorted({0, 1, chunk[b] // 2, chunk[b] - 20, chunk[b] - 19, chunk[b] - 1})]
    _check_rows(got, layer, fmt, q, table, spans, 0.1, n_rep, CHUNK_WEIGHT, N)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = call()
        graphs.append((g, out))
    for _ in range(3):
        q.mul_(-1)
        for g, _ in graphs:
            g.replay()
        eager = call()
        torch.cuda.synchronize()
        for _, out in graphs:
            assert torch.equal(out[:cu[4]].view(torch.int16), eager[:cu[4]].view(torch.int16))


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FMTS)
def test_chunks_without_scratch(cuda, fmt, monkeypatch):
    """No workspace: one kernel over whole keys, for few queries and for many."""
    from unifiedkv_amd import _ext

    rng = np.random.default_rng(12)
    H, R, D, N, lens = 2, 4, 128, 300, [2000, 900, 40]
    layer = _filled(cuda, fmt, torch.float16, rng, N, H, D)
    table = _tables(rng, N, lens)
    monkeypatch.setattr(_ext.load(), "ukv_quant_prefill_workspace_bytes", lambda *a: 0)
    for chunk in ([3, 1, 4], [200, 90, 40]):
        cu = np.concatenate([[0], np.cumsum(chunk)])
        q = torch.from_numpy(rng.standard_normal((sum(chunk), H * R, D))).half().to(cuda)
        got = quant_kv.prefill_attention(q, layer, _dev(table, cuda), list(cu), lens, softmax_scale=0.1, n_rep=R)
        spans = [(cu[b] + i, b, lens[b] - c + i + 1) for b, c in enumerate(chunk) for i in sorted({0, c // 2, c - 1})]
        _check_rows(got, layer, fmt, q, table, spans, 0.1, R, CHUNK_WEIGHT, N)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("H, n_rep, D", [(2, 4, 128), (2, 7, 128), (2, 4, 64), (2, 4, 96), (8, 4, 128)])
def test_nan_blocks_and_bad_pages_reach_only_what_sees_them(cuda, fmt, H, n_rep, D):
    """NaN blocks past the length, behind the diagonal and on pages outside the table leave every other row alone."""
    rng = np.random.default_rng(D + n_rep)
    pre, chunk = [40, 64, 20], [30, 17, 45]
    lens = [p + c for p, c in zip(pre, chunk)]
    N = 24
    layer = _filled(cuda, fmt, torch.bfloat16, rng, N, H, D)
    table = _tables(rng, N, lens, extra=0)
    table[1, 2] = N + 5  # sixteen keys without a page
    table[2, 0] = -1
    nan = torch.full((1, H, D), float("nan"), dtype=torch.bfloat16, device=cuda)
    for b in range(3):
        for pos in range(lens[b], 16 * -(-lens[b] // 16)):  # slots behind the end
            quant_kv.write_chunk_kv(layer, nan, nan, _dev(table[b:b + 1], cuda), [0, 1], [pos + 1])
    poison = nan.clone()
    poison[:, :, 32:] = 1.0  # one block of NaN: dims 0 .. 31
    one = torch.ones_like(nan)
    quant_kv.write_chunk_kv(layer, one, poison, _dev(table[:1], cuda), [0, 1], [60])  # V of position 59
    quant_kv.write_chunk_kv(layer, poison, one, _dev(table[2:], cuda), [0, 1], [50])  # K of position 49
    cu = np.concatenate([[0], np.cumsum(chunk)])
    q = torch.from_numpy(rng.standard_normal((sum(chunk), H * n_rep, D))).bfloat16().to(cuda)
    got = quant_kv.prefill_attention(q, layer, _dev(table, cuda), _dev(cu, cuda), _dev(lens, cuda), softmax_scale=0.1,
                                     n_rep=n_rep, max_chunk=max(chunk))
    spans = [(cu[b] + i, b, pre[b] + i + 1) for b in range(3) for i in range(chunk[b])]
    _check_rows(got, layer, fmt, q, table, spans, 0.1, n_rep, CHUNK_WEIGHT, N)
    dq = q[torch.as_tensor(cu[:3], device=cuda)]
    for cut in (lens, [59, lens[1], 49], [60, 33, 50]):
        got = quant_kv.decode_attention(dq, layer, _dev(table, cuda), _dev(cut, cuda), softmax_scale=0.1, n_rep=n_rep)
        _check_rows(got, layer, fmt, dq, table, [(b, b, n) for b, n in enumerate(cut)], 0.1, n_rep, DECODE_WEIGHT, N)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("q_size", [2.0 ** -100, 2.0 ** -20, 2.0 ** 40])
def test_queries_of_any_bf16_magnitude(cuda, fmt, q_size):
    """fp16 cannot hold these queries; the scale brings the scores back to ordinary ones."""
    rng = np.random.default_rng(2)
    lens, H, R, D = [50, 200], 2, 4, 128
    layer = _filled(cuda, fmt, torch.bfloat16, rng, 20, H, D)
    table = _tables(rng, 20, lens)
    q = (torch.from_numpy(rng.standard_normal((2, H * R, D))) * q_size).bfloat16().to(cuda)
    scale = float(np.float32(0.1 / q_size))
    spans = [(b, b, n) for b, n in enumerate(lens)]
    got = quant_kv.decode_attention(q, layer, _dev(table, cuda), _dev(lens, cuda), softmax_scale=scale, n_rep=R)
    _check_rows(got, layer, fmt, q, table, spans, scale, R, DECODE_WEIGHT, 20)
    got = quant_kv.prefill_attention(q, layer, _dev(table, cuda), [0, 1, 2], lens, softmax_scale=scale, n_rep=R)
    _check_rows(got, layer, fmt, q, table, spans, scale, R, CHUNK_WEIGHT, 20)


@pytest.mark.gpu
def test_extreme_held_values(cuda):
    """Keys and values at both ends of what the cache holds."""
    rng = np.random.default_rng(5)
    H, R, D, n = 2, 4, 128, 48
    for fmt, top in (("int8", 65024.0), ("fp8", 57344.0)):
        layer = _layer(cuda, fmt, 4, H, D)
        table = _dev([[2, 0, 3]], cuda)
        k = torch.from_numpy(rng.choice([-top, top, 2.0 ** -24, 0.0], size=(n, H, D))).bfloat16()
        v = torch.from_numpy(rng.choice([-top, top, 1.0], size=(n, H, D))).bfloat16()
        quant_kv.write_chunk_kv(layer, k.to(cuda), v.to(cuda), table, [0, n], [n])
        q = torch.from_numpy(rng.standard_normal((1, H * R, D))).bfloat16().to(cuda)
        scale = 2.0 ** -18
        got = quant_kv.decode_attention(q, layer, table, _dev([n], cuda), softmax_scale=scale, n_rep=R)
        _check_rows(got, layer, fmt, q, table.cpu().numpy(), [(0, 0, n)], scale, R, DECODE_WEIGHT, 4)
        got = quant_kv.prefill_attention(q, layer, table, [0, 1], [n], softmax_scale=scale, n_rep=R)
        _check_rows(got, layer, fmt, q, table.cpu().numpy(), [(0, 0, n)], scale, R, CHUNK_WEIGHT, 4)


@pytest.mark.gpu
def test_chunk_longer_than_declared_is_nan_and_written(cuda):
    rng = np.random.default_rng(4)
    layer = _filled(cuda, "int8", torch.float16, rng, 20, 2, 128)
    table = _dev(_tables(rng, 20, [60, 40]), cuda)
    q = torch.from_numpy(rng.standard_normal((70, 8, 128))).half().to(cuda)
    k = torch.from_numpy(rng.standard_normal((70, 2, 128))).half().to(cuda)
    cu, lens = _dev([0, 40, 70], cuda), _dev([60, 40], cuda)
    quant_kv.write_chunk_kv(layer, k, k, table, cu, lens, max_chunk=36)
    rk, _ = quant_kv.read_kv(layer, table, cu, lens, dtype=torch.float16, max_chunk=36, total=70)
    np.testing.assert_array_equal(rk.double().cpu().numpy(), qo.quantise(k.double().cpu().numpy(), "int8")[0])
    quant_kv.write_chunk_kv(layer, -k, k, table, cu, lens, max_chunk=0)
    assert torch.equal(quant_kv.read_kv(layer, table, cu, lens, dtype=torch.float16, max_chunk=36, total=70)[0], -rk)
    got = quant_kv.prefill_attention(q, layer, table, cu, lens, softmax_scale=0.1, n_rep=4, max_chunk=36)
    assert torch.isnan(got[:40]).all() and torch.isfinite(got[40:]).all()
    with pytest.raises(RuntimeError, match="max_chunk"):
        quant_kv.prefill_attention(q, layer, table, [0, 40, 70], lens, softmax_scale=0.1, n_rep=4, max_chunk=36)
    with pytest.raises(RuntimeError, match="max_chunk"):
        quant_kv.read_kv(layer, table, cu, lens, dtype=torch.float16, max_chunk=20, total=70)


@pytest.mark.gpu
def test_offsets_past_32_bits(cuda):
    """A cache of more than 2^31 bytes a layer, its last pages in use."""
    rng = np.random.default_rng(6)
    N, H, R, D, lens = 140000, 8, 4, 128, [50, 33]
    layer = _layer(cuda, "fp8", N, H, D)
    table = np.zeros((2, 4), dtype=np.int32)
    table[0], table[1, :3] = [N - 1, N - 2, 1, N - 7], [N - 3, 0, N - 4]
    rows = [torch.from_numpy(rng.standard_normal((83, H, D))).bfloat16().to(cuda) for _ in range(2)]
    quant_kv.write_chunk_kv(layer, *rows, _dev(table, cuda), [0, 50, 83], lens)
    back = quant_kv.read_kv(layer, _dev(table, cuda), [0, 50, 83], lens, dtype=torch.bfloat16)
    for x, y in zip(rows, back):
        np.testing.assert_array_equal(y.double().cpu().numpy(), qo.quantise(x.double().cpu().numpy(), "fp8")[0])
    small = QuantLayer(*(x[table.reshape(-1)] if x.dtype == torch.uint8 else
                         x.view(torch.uint8)[table.reshape(-1)].view(x.dtype)
                         for x in (layer.k, layer.v, layer.k_scale, layer.v_scale)))
    same = np.arange(8, dtype=np.int32).reshape(2, 4)
    q = torch.from_numpy(rng.standard_normal((83, H * R, D))).bfloat16().to(cuda)
    for t, c in ((table, layer), (same, small)):
        dec = quant_kv.decode_attention(q[:2], c, _dev(t, cuda), _dev(lens, cuda), softmax_scale=0.1, n_rep=R)
        chk = quant_kv.prefill_attention(q, c, _dev(t, cuda), [0, 50, 83], lens, softmax_scale=0.1, n_rep=R)
        if c is layer:
            first = dec, chk
    assert torch.equal(first[0], dec) and torch.equal(first[1], chk)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FMTS)
def test_streams_and_captured_calls(cuda, fmt):
    """A step's calls captured on one stream, replayed beside eager calls on another."""
    rng = np.random.default_rng(8)
    H, R, D, lens = 4, 4, 128, [700, 90, 2000]
    N = 200
    layer = _filled(cuda, fmt, torch.bfloat16, rng, N, H, D)
    table = _dev(_tables(rng, N, [n + 4 for n in lens]), cuda)
    old, cu = _dev(lens, cuda), _dev([0, 2, 3, 5], cuda)
    attn, kv = old + 1, _dev([n + c for n, c in zip(lens, (2, 1, 2))], cuda)
    x = {n: torch.from_numpy(rng.standard_normal(s)).bfloat16().to(cuda)
         for n, s in (("q", (3, H * R, D)), ("k", (3, H, D)), ("v", (3, H, D)), ("cq", (5, H * R, D)),
                      ("ck", (5, H, D)), ("cv", (5, H, D)))}

    def step():
        quant_kv.append_kv(layer, x["k"], x["v"], table, old)
        a = quant_kv.decode_attention(x["q"], layer, table, attn, softmax_scale=0.1, n_rep=R)
        quant_kv.write_chunk_kv(layer, x["ck"], x["cv"], table, cu, kv, max_chunk=2)
        b = quant_kv.prefill_attention(x["cq"], layer, table, cu, kv, softmax_scale=0.1, n_rep=R, max_chunk=2)
        return [a, b] + list(quant_kv.read_kv(layer, table, cu, kv, dtype=torch.bfloat16, max_chunk=2, total=5))

    want = [t.clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        there = step()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(want, there):
        assert torch.equal(a, b)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        graphs.append((g, out))
    for i in range(3):
        x["q"].mul_(-1)
        x["cq"].mul_(-1)
        for g, _ in graphs:
            g.replay()
        eager = step()
        torch.cuda.synchronize()
        for _, out in graphs:
            for a, b in zip(eager, out):
                assert torch.equal(a, b), i


@pytest.mark.gpu
def test_another_current_device(cuda, monkeypatch):
    """A launch goes to the current device: the layer's is made that one for the call."""
    layer = _filled(cuda, "int8", torch.float16, np.random.default_rng(1), 8, 2, 64)
    q, table, lens = torch.ones((1, 4, 64), dtype=torch.float16, device=cuda), _dev([[1, 2]], cuda), _dev([20], cuda)
    calls = [lambda: quant_kv.decode_attention(q, layer, table, lens, softmax_scale=0.1, n_rep=2),
             lambda: quant_kv.prefill_attention(q, layer, table, [0, 1], lens, softmax_scale=0.1, n_rep=2),
             lambda: quant_kv.read_kv(layer, table, [0, 1], lens, dtype=torch.float16)[0]]
    want = [c() for c in calls]
    entered = []

    class Guard(torch.cuda.device):
        def __init__(self, device):
            entered.append(torch.device(device))
            super().__init__(device)

    monkeypatch.setattr(torch.cuda, "device", Guard)
    monkeypatch.setattr(quant_kv, "_device_now", lambda: 1 + (cuda.index or 0))
    for call, w in zip(calls, want):
        entered.clear()
        assert torch.equal(call(), w) and entered[-1] == layer.device
    quant_kv.append_kv(layer, q[:, :2], q[:, :2], table, lens)
    assert len(entered) == 2


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_pool_prefill_decode_and_compaction_together(cuda, fmt, dtype):
    """Chunked prefill, decode steps and page copies over one pool, as an engine runs them, against the oracle over
    the rows that went in."""
    rng = np.random.default_rng(9)
    dt, L, H, R, D = DTYPES[dtype], 2, 2, 4, 128
    pool = QuantizedKVPool(16, L, H, D, dt, cache_format=fmt, num_blocks=64, device=cuda)
    rows = [[[np.empty((0, H, D))] * 2 for _ in range(3)] for _ in range(L)]  # [layer][seq] -> K, V in fp64
    pp = prefill.PrefillPages(pool, 3)

    def new(n, heads):
        return torch.from_numpy(rng.standard_normal((n, heads, D))).to(dt).to(cuda)

    def check(layer, out, q, at, b, weight):
        k, v = rows[layer][b]
        for h in range(H * R):
            qh = q[h].double().cpu().numpy()
            kk, vv = k[:at + 1, h // R], v[:at + 1, h // R]
            want, spread = qo.attend(qh, kk, vv, 0.1)
            tol = _bound(want, spread, vv, qh, kk, 0.1, dt, weight)
            assert np.all(np.abs(out[h].double().cpu().numpy() - want) <= tol)

    for chunk in ([20, 33, 1], [7, 0, 40]):
        pp.begin_chunk(chunk)
        before = pp.seq_lens
        for layer in range(L):
            q, k, v = new(sum(chunk), H * R), new(sum(chunk), H), new(sum(chunk), H)
            out = pp.attention(layer, q, k, v, softmax_scale=0.1, n_rep=R)
            at = 0
            for b, c in enumerate(chunk):
                rows[layer][b] = [np.concatenate([o, qo.quantise(x[at:at + c].double().cpu().numpy(), fmt)[0]])
                                  for o, x in zip(rows[layer][b], (k, v))]
                for i in sorted({0, c - 1} & set(range(c))):
                    check(layer, out[at + i], q[at + i], before[b] + i, b, CHUNK_WEIGHT)
                at += c
        with pytest.raises(RuntimeError, match="obs_stats"):
            pp.attention(0, q, k, v, softmax_scale=0.1, n_rep=R, obs_stats=object())
        pp.end_chunk()
    batch = decode_step.DecodeBatch(pool, pp.page_lists, pp.seq_lens, fused_append=True)
    for _ in range(18):
        batch.begin_step()
        for layer in range(L):
            q, k, v = new(3, H * R), new(3, H), new(3, H)
            out = batch.attention(layer, q, k, v, softmax_scale=0.1, n_rep=R)
            for b in range(3):
                rows[layer][b] = [np.concatenate([o, qo.quantise(x[b:b + 1].double().cpu().numpy(), fmt)[0]])
                                  for o, x in zip(rows[layer][b], (k, v))]
                check(layer, out[b], q[b], batch.seq_lens[b], b, DECODE_WEIGHT)
        batch.end_step()
    # the longest sequence (59 tokens, four pages): a read, and a copy of its pages, the same rows
    ids, n = batch.page_lists[2], batch.seq_lens[2]
    new_ids = pool.allocate_blocks(len(ids))
    pool.copy_pages(torch.tensor(ids, dtype=torch.int32, device=cuda),
                    torch.tensor(new_ids, dtype=torch.int32, device=cuda))
    for layer in range(L):
        for pages in (ids, new_ids):
            K, V = pool.read_kv_from_blocks(layer, pages, n)
            assert K.shape == (H, n, D) and K.is_contiguous()
            for got, want in zip((K, V), rows[layer][2]):
                np.testing.assert_array_equal(got.transpose(0, 1).double().cpu().numpy(), want)
    # block-aligned compaction: pages 0, 2 and 3 of each layer
    keep = torch.tensor([[0, 2, 3]] * L, dtype=torch.int32, device=cuda)
    res = compaction.compact(pool, [new_ids], [keep], [43])
    K, _ = pool.read_kv_from_blocks(1, res.page_lists[0], 43)
    want = rows[1][2][0]
    np.testing.assert_array_equal(K.transpose(0, 1).double().cpu().numpy(), np.concatenate([want[:16], want[32:]]))


@pytest.mark.gpu
def test_pool_token_io(cuda):
    rng = np.random.default_rng(11)
    pool = QuantizedKVPool(16, 1, 2, 64, torch.bfloat16, cache_format="int8", num_blocks=8, device=cuda)
    K, V = (torch.from_numpy(rng.standard_normal((2, 21, 64))).float() for _ in range(2))  # cast and moved, as ever
    pool.write_kv_to_blocks(0, [5, 2], K, V)
    rk, rv = pool.read_kv_from_blocks(0, [5, 2], 100)
    assert rk.shape == (2, 32, 64)
    for x, y in ((K, rk), (V, rv)):
        want = qo.quantise(x.bfloat16().double().numpy(), "int8")[0]
        np.testing.assert_array_equal(y[:, :21].double().cpu().numpy(), want)
    tok = torch.from_numpy(rng.standard_normal((2, 1, 64))).bfloat16().to(cuda)
    pool.write_one_token(0, 2, 5, tok, tok)
    lens = pool.append_decode_tokens(0, _dev([[5, 2]], cuda), _dev([22], cuda), tok.transpose(0, 1), tok.transpose(0, 1))
    assert lens.tolist() == [23]
    rk, _ = pool.read_kv_from_blocks(0, [5, 2], 23)
    want = qo.quantise(tok[:, 0].double().cpu().numpy(), "int8")[0]
    for at in (21, 22):
        np.testing.assert_array_equal(rk[:, at].double().cpu().numpy(), want)
    assert pool.read_kv_from_blocks(0, [], 5)[0].shape == (2, 0, 64)
    with pytest.raises(IndexError):
        pool.write_one_token(0, 8, 0, tok, tok)
    assert pool.release_if_empty() and not pool.is_allocated
    with pytest.raises(IndexError):
        pool.layer(-1)
