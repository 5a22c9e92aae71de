"""CPU checks of the refusals of the rotated appends, the 4-bit pool and the
verification of drafts: every C entry point, and the facade over host
tensors, before anything is launched."""

import importlib

import pytest
import torch

FAKE = 1 << 20  # never dereferenced: validation fails first
FAR = 1 << 40
NAN, INF = float("nan"), float("inf")


@pytest.fixture(scope="module")
def L(pkg):
    return pkg._lib


def _refused(L, name, args, code, text, **changes):
    args = dict(args)
    for key, value in changes.items():
        assert key in args
        args[key] = value
    assert getattr(L.lib(), name)(*args.values()) == getattr(L, code), changes
    assert text in L.last_error(), L.last_error()


ROTARY = dict(q=FAKE, k=FAKE, v=FAKE, out=FAR, kr=FAKE, vr=FAKE, rows=64, slots=FAKE,
              positions=FAKE, dtype=1, tokens=3, q_heads=8, kv_heads=2, head_dim=128,
              value_dim=64, rotary=128, style=0, base=1e4, scale=1.0, stream=None)
APPEND = dict(q=FAKE, k=FAKE, v=FAKE, out=FAR, kc=FAKE, ks=FAKE, vc=FAKE, vs=FAKE, page_size=32,
              num_pages=5, slots=FAKE, positions=FAKE, dtype=1, tokens=3, q_heads=8, kv_heads=2,
              head_dim=128, rotary=128, style=1, base=1e4, scale=1.0, stream=None)


@pytest.mark.parametrize("name,args", [("alpx_rotary_append_rows", ROTARY),
                                       ("alpx_q4_append_rows", APPEND)])
def test_append_refusals(L, name, args):
    for key, value in args.items():
        if value in (FAKE, FAR):
            _refused(L, name, args, "EINVAL", "null buffer", **{key: None})
    for key in ("tokens", "kv_heads", "head_dim", "value_dim", "rows", "num_pages"):
        if key in args:
            for value in (0, -1):
                _refused(L, name, dict(args, rotary=0), "EINVAL", "positive", **{key: value})
    _refused(L, name, args, "EINVAL", "positive", q_heads=-1)
    for value in (-2, 1, 127, 130):
        _refused(L, name, args, "EINVAL", "rotary_dim", rotary=value)
    for value in (-1, 2):
        _refused(L, name, args, "EINVAL", "style", style=value)
    for value in (-1, 3):
        _refused(L, name, args, "EINVAL", "dtype", dtype=value)
    for value in (0.0, -1.0, NAN, INF):
        _refused(L, name, args, "EINVAL", "positive and finite", base=value)
        _refused(L, name, args, "EINVAL", "positive and finite", scale=value)
    _refused(L, name, args, "EUNSUPPORTED", "too many heads", q_heads=1 << 28)
    q = 3 * 8 * 128 * 2  # bytes of the query
    for at in (FAKE, FAKE + q - 2, FAKE - q + 2):
        _refused(L, name, args, "EINVAL", "overlap", out=at)
    _refused(L, name, args, "EINVAL", "overlap", q=FAR * 2, v=FAR * 2, out=FAKE + 2)
    _refused(L, name, args, "EINVAL", "overlap", q=FAR * 2, k=FAR * 2, out=FAKE + 2)


def test_rotary_append_refuses_wide_heads(L):
    for key in ("head_dim", "value_dim"):
        _refused(L, "alpx_rotary_append_rows", ROTARY, "EUNSUPPORTED", "above 512", **{key: 513})


ROWS = dict(kc=FAKE, ks=FAKE, vc=FAKE, vs=FAKE, page_size=32, num_pages=5, slots=FAKE, rows=3,
            kv_heads=2, head_dim=128, k=FAKE, v=FAKE, dtype=0, stream=None)
ATTEND = dict(q=FAKE, kc=FAKE, ks=FAKE, vc=FAKE, vs=FAKE, table=FAKE, max_pages=4, page_size=32,
              num_pages=5, prefix=FAKE, counts=None, length=100, gate=None, out=FAR, ws=FAKE,
              ws_bytes=1 << 40, batch=2, nodes=3, q_heads=8, kv_heads=2, head_dim=128, scale=0.1,
              dtype=1, out_dtype=1, stream=None)


@pytest.mark.parametrize("name,args", [("alpx_q4_append_rows", APPEND), ("alpx_q4_rows", ROWS),
                                       ("alpx_q4_attention", ATTEND)])
def test_pool_refusals(L, name, args):
    for size in (0, -32, 16, 48):
        _refused(L, name, args, "EINVAL", "power of two", page_size=size)
    for width in (32, 80, 160, 512):
        _refused(L, name, dict(args, **({"rotary": 0} if "rotary" in args else {})),
                 "EUNSUPPORTED", "64, 96, 128 or 256", head_dim=width)
    _refused(L, name, args, "EUNSUPPORTED", "2^31", num_pages=1 << 26)
    for key in ("kc", "ks", "vc", "vs"):
        _refused(L, name, args, "EINVAL", "aligned", **{key: FAKE + 8})


def test_rows_refusals(L):
    name = "alpx_q4_rows"
    for key, value in ROWS.items():
        if value == FAKE:
            _refused(L, name, ROWS, "EINVAL", "null buffer", **{key: None})
    for key in ("rows", "kv_heads", "num_pages"):
        _refused(L, name, ROWS, "EINVAL", "positive", **{key: 0})
    _refused(L, name, ROWS, "EINVAL", "dtype", dtype=3)
    for key in ("k", "v"):
        _refused(L, name, ROWS, "EINVAL", "aligned", **{key: FAKE + 4})


def test_attention_refusals(L):
    name = "alpx_q4_attention"
    for key in ("q", "kc", "ks", "vc", "vs", "table", "prefix", "out"):
        _refused(L, name, ATTEND, "EINVAL", "null buffer", **{key: None})
    for key in ("batch", "nodes", "q_heads", "kv_heads", "length", "max_pages", "num_pages"):
        for value in (0, -1):
            _refused(L, name, ATTEND, "EINVAL", "positive", **{key: value})
    _refused(L, name, ATTEND, "EINVAL", "multiple of KV heads", q_heads=7)
    _refused(L, name, ATTEND, "ERANGE", "block table", length=129)
    _refused(L, name, ATTEND, "EUNSUPPORTED", "2^31", max_pages=1 << 26)
    _refused(L, name, ATTEND, "EUNSUPPORTED", "2^24", page_size=1 << 25)
    for key in ("dtype", "out_dtype"):
        for value in (-1, 3):
            _refused(L, name, ATTEND, "EINVAL", "dtype", **{key: value})
    for value in (0.0, -1.0, NAN, INF):
        _refused(L, name, ATTEND, "EINVAL", "scale", scale=value)
    q = 2 * 3 * 8 * 128 * 2
    for at in (FAKE, FAKE + q - 2, FAKE - q + 2):
        _refused(L, name, ATTEND, "EINVAL", "overlap", out=at)
        _refused(L, name, ATTEND, "EINVAL", "overlap", q=FAR * 2, gate=FAKE, out=at)


def test_attention_workspace(L):
    name, size = "alpx_q4_attention", L.lib().alpx_q4_workspace_bytes
    # sizes whose counts pass 31 bits, and no workspace that they would take
    good = dict(batch=2, nodes=3, q_heads=8, kv_heads=2, head_dim=128, length=4000, dtype=1)
    long = dict(ATTEND, length=4000, max_pages=1 << 20, out=1 << 60)
    assert size(*good.values()) > 0
    need = size(*good.values())
    _refused(L, name, long, "EINVAL", "workspace", ws=None)
    _refused(L, name, long, "EINVAL", "workspace", ws_bytes=need - 1)
    _refused(L, name, long, "EINVAL", "workspace", ws=FAKE + 8)
    for bad in (dict(batch=(1 << 24) + 1), dict(nodes=1 << 24), dict(length=2 ** 31 - 40),
                dict(q_heads=1 << 20, nodes=60000), dict(batch=60000, length=1 << 24),
                dict(batch=1 << 20, nodes=1 << 10, q_heads=1 << 10, kv_heads=1 << 10)):
        _refused(L, name, dict(long, max_pages=(2 ** 31 - 32) // 32), "EUNSUPPORTED", "too many",
                 **bad)
        assert size(*dict(good, **bad).values()) == 0
    for bad in (dict(batch=0), dict(nodes=-1), dict(q_heads=7), dict(kv_heads=0),
                dict(head_dim=80), dict(length=0), dict(dtype=9)):
        assert size(*dict(good, **bad).values()) == 0


def test_verify_refusals(L):
    name, size = "alpx_verify_drafts", L.lib().alpx_verify_workspace_bytes
    args = dict(tokens=FAKE, target=FAKE, draft=None, parents=None, counts=None, uniforms=FAKE,
                paths=FAKE, accepted=FAKE, new=FAKE, ws=FAKE, ws_bytes=1 << 30, batch=2, nodes=5,
                vocab=1000, dtype=0, stream=None)
    for key in ("tokens", "target", "uniforms", "paths", "accepted", "new"):
        _refused(L, name, args, "EINVAL", "null buffer", **{key: None})
    for key in ("batch", "nodes", "vocab"):
        for value in (0, -1):
            _refused(L, name, args, "EINVAL", "positive", **{key: value})
    for changes in (dict(batch=65536), dict(nodes=1025), dict(vocab=2 ** 31)):
        _refused(L, name, args, "EUNSUPPORTED", "at most", **changes)
        assert size(*{**dict(batch=2, nodes=5, vocab=1000), **changes}.values()) == 0
    _refused(L, name, args, "EINVAL", "dtype", dtype=3)
    need = size(2, 5, 1000)
    assert need > 0
    for changes in (dict(ws=None), dict(ws_bytes=need - 1), dict(ws=FAKE + 8)):
        _refused(L, name, args, "EINVAL", "workspace", **changes)


# ------------------------------------------------------------------ facade


@pytest.fixture
def ops(pkg, monkeypatch):
    """The facade over host tensors (their device index is -1), with nothing
    behind its checks."""
    m = importlib.import_module(pkg.__name__ + ".qwen35_rocm_ops")
    o = m.Qwen35RocmOps(_capability=m.RocmCapability(True, "injected", 0, "gfx950"))
    o.device_index = -1

    def reached(*args, **kw):
        raise AssertionError("passed every check")
    for name in ("rotary_append_rows", "q4_append_rows", "q4_rows", "q4_attention",
                 "verify_drafts"):
        monkeypatch.setattr(m._ops, name, reached)
    return o


f = torch.zeros


def _i32(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def _pool(pages=5, heads=2, page=32, width=64):
    codes = torch.zeros((pages, heads, page, width // 2), dtype=torch.uint8)
    scales = torch.zeros((pages, heads, 2, width // 32, page), dtype=torch.float16)
    return dict(key_codes=codes, key_scales=scales, value_codes=codes.clone(),
                value_scales=scales.clone())


def _check(call, base, table):
    with pytest.raises(AssertionError, match="passed"):
        call(**base)
    for error, text, changes in table:
        with pytest.raises(error, match=text):
            call(**dict(base, **changes))


POOL_TABLE = [
    (TypeError, "uint8", dict(key_codes=f(5, 2, 32, 32))),
    (TypeError, "uint8", dict(key_codes=[1])),
    (TypeError, "float16", dict(value_scales=f(5, 2, 2, 2, 32))),
    (ValueError, "codes .num_pages", dict(value_codes=torch.zeros(4, 2, 32, 32, dtype=torch.uint8))),
    (ValueError, "codes .num_pages", dict(key_scales=f(5, 2, 2, 1, 32).half())),
    (ValueError, "codes .num_pages", _pool(page=16)),
    (ValueError, "codes .num_pages", _pool(page=48)),
    (ValueError, "codes .num_pages", _pool(width=32)),
    (ValueError, "codes .num_pages", _pool(pages=0)),
    (ValueError, "contiguous", dict(value_codes=torch.zeros(5, 2, 32, 64,
                                                            dtype=torch.uint8)[..., ::2])),
]


def test_facade_append_refusals(ops):
    rows = dict(query=f(3, 4, 64), key=f(3, 2, 64), value=f(3, 2, 64), slots=_i32(3),
                positions=_i32(3), rotary_dimension=64)
    table = [
        (ValueError, "at least one token", dict(key=f(0, 2, 64), value=f(0, 2, 64))),
        (ValueError, "tokens or heads differ", dict(value=f(2, 2, 64))),
        (TypeError, "share one dtype", dict(value=f(3, 2, 64).half())),
        (TypeError, "share one dtype", dict(query=f(3, 4, 64).half())),
        (ValueError, "tokens or head width", dict(query=f(2, 4, 64))),
        (ValueError, "tokens or head width", dict(query=f(3, 4, 32))),
        (ValueError, "multiple of KV heads", dict(query=f(3, 3, 64))),
        (ValueError, "multiple of KV heads", dict(query=f(3, 0, 64))),
        (ValueError, "token shape", dict(key=f(3, 1, 64), value=f(3, 1, 64))),
        (ValueError, "one entry", dict(slots=[0, 1])),
        (ValueError, "one entry", dict(slots=[0, 1, 160])),
        (ValueError, "integers", dict(slots=[0, 1.5, 2])),
        (ValueError, "one entry", dict(positions=[0, -1, 2])),
        (ValueError, "needs positions", dict(positions=None)),
        (ValueError, "rotary_dimension", dict(rotary_dimension=63)),
        (ValueError, "rotary_dimension", dict(rotary_dimension=66)),
        (ValueError, "rotary_dimension", dict(rotary_dimension=-2)),
        (ValueError, "style", dict(style="gptj")),
        (ValueError, "frequency_base", dict(frequency_base=0.0)),
        (ValueError, "frequency_scale", dict(frequency_scale=NAN)),
    ]
    pages = dict(key_pages=f(5, 32, 2, 64), value_pages=f(5, 32, 2, 64))
    _check(ops.paged_rotary_append_rows_, dict(rows, **pages), table + [
        (ValueError, "count, size or heads", dict(value_pages=f(5, 16, 2, 64))),
        (ValueError, "token shape", dict(value_pages=f(5, 32, 2, 48))),
        (TypeError, "share one dtype", dict(key_pages=f(5, 32, 2, 64).half()))])
    _check(ops.paged_q4_append_rows_, dict(rows, **_pool()), table + POOL_TABLE + [
        (ValueError, "token shape", dict(value=f(3, 2, 32)))])
    for call, pool in ((ops.paged_rotary_append_rows_, pages), (ops.paged_q4_append_rows_, _pool())):
        with pytest.raises(AssertionError, match="passed"):
            call(**dict(rows, **pool, query=None, positions=None, rotary_dimension=0))


def test_facade_pool_and_rows_refusals(ops):
    ops.device = "cpu"
    pool = ops.initialize_paged_q4_workspace(num_pages=5, page_size=32, kv_heads=2,
                                             head_dimension=96)
    assert pool.key_codes.shape == (5, 2, 32, 48) and pool.value_scales.shape == (5, 2, 2, 3, 32)
    assert pool.descriptor()["page_size"] == 32
    with pytest.raises(AssertionError, match="passed"):
        ops.paged_q4_rows(*pool.arrays, _i32(3))
    for key, bad in (("num_pages", 0), ("page_size", 48), ("page_size", 16), ("kv_heads", 0),
                     ("head_dimension", 80), ("num_pages", 1 << 26)):
        with pytest.raises(ValueError):
            ops.initialize_paged_q4_workspace(**dict(dict(num_pages=5, page_size=32, kv_heads=2,
                                                          head_dimension=96), **{key: bad}))
    _check(ops.paged_q4_rows, dict(_pool(), slots=_i32(3)), POOL_TABLE + [
        (ValueError, "at least one row", dict(slots=_i32(0))),
        (ValueError, "at least one row", dict(slots=_i32(1, 3))),
        (ValueError, "one entry", dict(slots=[0, 160])),
        (TypeError, "float32, float16", dict(dtype=torch.int32))])


def test_facade_attention_refusals(ops):
    base = dict(_pool(), query=f(2, 3, 4, 64), block_table=_i32(2, 2), length=60,
                prefix_lens=_i32(2))
    _check(ops.paged_q4_attention, base, POOL_TABLE + [
        (ValueError, "exceeds capacity", dict(length=65)),
        (ValueError, "positive integer", dict(length=0)),
        (ValueError, "head width", dict(query=f(2, 3, 4, 128))),
        (ValueError, "at least one token", dict(query=f(2, 0, 4, 64))),
        (ValueError, "multiple of KV heads", dict(query=f(2, 3, 5, 64))),
        (ValueError, "table batch", dict(block_table=_i32(3, 2))),
        (TypeError, "block table", dict(block_table=[[0, 1]])),
        (TypeError, "block table", dict(block_table=f(2, 2))),
        (ValueError, "match the attention output", dict(gate=f(2, 3, 4, 32))),
        (TypeError, "share one dtype", dict(gate=f(2, 3, 4, 64).half())),
        (ValueError, "one entry", dict(prefix_lens=[0])),
        (ValueError, "one entry", dict(prefix_lens=[0, 61])),
        (ValueError, "one entry", dict(counts=[1, 4])),
        (ValueError, "integers", dict(counts=[1, True])),
        (ValueError, "positive and finite", dict(scale=0.0)),
        (TypeError, "float32, float16", dict(out_dtype=torch.int8)),
        (ValueError, "expected", dict(out=f(2, 3, 4, 32))),
        (TypeError, "bfloat16", dict(out=f(2, 3, 4, 64), out_dtype=torch.bfloat16))])


def test_facade_verify_refusals(ops):
    base = dict(drafts=_i32(2, 4), target=f(2, 4, 10), uniforms=f(2, 4))
    _check(ops.verify_drafts, base, [
        (ValueError, "1 to 1024", dict(target=f(2, 0, 10))),
        (ValueError, "1 to 1024", dict(target=f(1, 1025, 1))),
        (ValueError, "1 to 1024", dict(target=f(2, 4, 0))),
        (ValueError, "at most 65535", dict(target=f(65536, 1, 1))),
        (TypeError, "int32", dict(drafts=[[0] * 4] * 2)),
        (TypeError, "int32|remain", dict(drafts=f(2, 4))),
        (TypeError, "float32", dict(uniforms=f(2, 4).half())),
        (ValueError, "uniform numbers have", dict(uniforms=f(2, 3))),
        (ValueError, "shapes differ", dict(draft=f(2, 4, 9))),
        (TypeError, "share one dtype", dict(draft=f(2, 4, 10).half())),
        (TypeError, "int32", dict(parents=[[0] * 4] * 2)),
        (TypeError, "int32|remain", dict(parents=_i32(2, 3))),
        (ValueError, "one entry", dict(counts=[1, 5]))])
    for extra in (dict(draft=f(2, 4, 10)), dict(parents=_i32(2, 4)), dict(counts=_i32(2))):
        with pytest.raises(AssertionError, match="passed"):
            ops.verify_drafts(**dict(base, **extra))


def test_facade_refuses_host_tensors(pkg):
    m = importlib.import_module(pkg.__name__ + ".qwen35_rocm_ops")
    o = m.Qwen35RocmOps(_capability=m.RocmCapability(True, "injected", 0, "gfx950"))
    pool = tuple(_pool().values())
    for call in (lambda: o.paged_rotary_append_rows_(f(1, 2, 8), f(1, 2, 8), f(1, 2, 8),
                                                     f(1, 4, 2, 8), f(1, 4, 2, 8), [0], [0],
                                                     rotary_dimension=8),
                 lambda: o.verify_drafts(_i32(1, 2), f(1, 2, 8), f(1, 2))):
        with pytest.raises(TypeError, match="must remain on the ROCm device"):
            call()
    with pytest.raises(ValueError, match="must be on device 0"):
        o.paged_q4_rows(*pool, _i32(2))


@pytest.mark.parametrize("which", range(4))
def test_facade_pool_arrays_that_are_no_tensors(ops, which):
    ops.device = "cpu"
    arrays = list(ops.initialize_paged_q4_workspace(num_pages=2, page_size=32, kv_heads=1,
                                                    head_dimension=64).arrays)
    arrays[which] = None
    with pytest.raises(TypeError, match="must be a"):
        ops.paged_q4_rows(*arrays, _i32(3))


@pytest.mark.parametrize("name,args", [("alpx_rotary_append_rows", ROTARY),
                                       ("alpx_q4_append_rows", APPEND)])
def test_append_refuses_frequencies_past_what_angles_hold(L, name, args):
    """Angles stay below 2^33: frequencies up to 4, positions below 2^31.  A
    base below 1 makes frequencies rise, up to base^(-126 / 128) here."""
    for value in (4.0000001, 1e6, 1e300):
        _refused(L, name, args, "EUNSUPPORTED", "frequencies above 4", scale=value)
    for value in (0.24, 1e-3, 1e-300, 5e-324):
        _refused(L, name, args, "EUNSUPPORTED", "frequencies above 4", base=value)
    for value in (0.06, 1e-3, 1e-300, 5e-324):  # two pairs: up to base^(-1 / 2)
        _refused(L, name, args, "EUNSUPPORTED", "frequencies above 4", base=value, rotary=4)
    # one pair has the scale for its frequency, whatever the base
    _refused(L, name, args, "EUNSUPPORTED", "frequencies above 4", rotary=2, scale=5.0)


@pytest.mark.parametrize("name,args", [("alpx_rotary_append_rows", ROTARY),
                                       ("alpx_q4_append_rows", APPEND)])
def test_append_refuses_more_tokens_than_a_launch_has_blocks(L, name, args):
    for value in (1 << 24, 0x7fffffff):
        _refused(L, name, args, "EUNSUPPORTED", "too many tokens", tokens=value)
