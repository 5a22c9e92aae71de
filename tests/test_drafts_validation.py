"""CPU checks of the draft-tree operators' refusals: every C entry point, and
the facade over host tensors, before anything is launched."""

import ctypes
import importlib

import pytest
import torch

FAKE = 4096  # never dereferenced: validation fails first
FAR = 1 << 40


@pytest.fixture(scope="module")
def L(pkg):
    return pkg._lib


def _call(L, name, args, changes):
    args = dict(args)
    for key, value in changes.items():
        assert key in args
        args[key] = value
    return getattr(L.lib(), name)(*args.values())


def _refused(L, name, args, code, text, **changes):
    assert _call(L, name, args, changes) == getattr(L, code), changes
    assert text in L.last_error(), L.last_error()


TREE = dict(q=FAKE, k=FAKE, v=FAKE, masks=FAKE, mask_stride=8, words=1, prefix=FAKE, counts=None,
            length=100, gate=None, out=FAR, ws=FAKE, ws_bytes=1 << 40, batch=2, nodes=8, q_heads=8,
            kv_heads=2, key_dim=64, value_dim=64, k_pos=256, k_batch=128, k_head=64, v_pos=256,
            v_batch=128, v_head=64, scale=0.125, dtype=1, out_dtype=1, stream=None)
PAGED = dict(q=FAKE, k=FAKE, v=FAKE, table=FAKE, max_pages=4, page_size=32, num_pages=9, masks=FAKE,
             mask_stride=8, words=1, prefix=FAKE, counts=None, length=100, gate=None, out=FAR,
             ws=FAKE, ws_bytes=1 << 40, batch=2, nodes=8, q_heads=8, kv_heads=2, key_dim=64,
             value_dim=64, scale=0.125, dtype=1, out_dtype=1, stream=None)


@pytest.mark.parametrize("name,args", [("alpx_tree_attention", TREE),
                                       ("alpx_tree_attention_paged", PAGED)])
def test_tree_attention_refusals(L, name, args):
    for key in ("q", "k", "v", "masks", "prefix", "out"):
        _refused(L, name, args, "EINVAL", "null buffer", **{key: None})
    for key in ("batch", "nodes", "q_heads", "kv_heads", "key_dim", "value_dim", "length"):
        for value in (0, -1):
            _refused(L, name, args, "EINVAL", "positive", **{key: value})
    _refused(L, name, args, "EINVAL", "multiple of KV heads", q_heads=7)
    _refused(L, name, args, "EINVAL", "mask_words", nodes=65)
    _refused(L, name, args, "EINVAL", "mask_words", words=-1)
    _refused(L, name, args, "EINVAL", "mask_words", mask_stride=-8)
    for key in ("key_dim", "value_dim"):
        _refused(L, name, args, "EUNSUPPORTED", "above 256", **{key: 257})
    for key in ("dtype", "out_dtype"):
        for value in (-1, 3):
            _refused(L, name, args, "EINVAL", "dtype", **{key: value})
    for value in (0.0, -1.0, float("nan"), float("inf")):
        _refused(L, name, args, "EINVAL", "scale", scale=value)
    _refused(L, name, args, "EINVAL", "16-byte aligned", ws=FAKE + 8)
    # many rows: two launches, which need the workspace
    many = dict(args, length=2000, **({"max_pages": 64} if "max_pages" in args else {}))
    need = L.lib().alpx_tree_workspace_bytes(2, 8, 8, 2, 64, 64, 2000, 1)
    assert need > 0
    _refused(L, name, many, "EINVAL", "workspace", ws_bytes=100)
    _refused(L, name, many, "EINVAL", "workspace", ws=None)
    # out over the queries or the gate, wholly or in part
    for at in (FAKE, FAKE + 2 * 8 * 8 * 64 * 2 - 2, FAKE - 2):
        _refused(L, name, args, "EINVAL", "overlap", out=at)
        _refused(L, name, args, "EINVAL", "overlap", q=FAR * 2, gate=FAKE, out=at)


def test_tree_attention_refuses_rows_past_its_range(L):
    name = "alpx_tree_attention"
    _refused(L, name, TREE, "EUNSUPPORTED", "too far apart", k_pos=1 << 26)
    _refused(L, name, TREE, "EUNSUPPORTED", "too far apart", v_pos=1 << 26)
    _refused(L, name, TREE, "EUNSUPPORTED", "too many rows", length=(1 << 30) + 1)
    _refused(L, name, TREE, "EUNSUPPORTED", "too many rows", length=1 << 30, batch=64)
    _refused(L, name, TREE, "EUNSUPPORTED", "too many drafts", nodes=1 << 24, words=1 << 18)
    for key in ("k_pos", "k_batch", "k_head", "v_pos", "v_batch", "v_head"):
        _refused(L, name, TREE, "EINVAL", "negative", **{key: -64})


def test_paged_tree_attention_refuses_bad_pages(L):
    name = "alpx_tree_attention_paged"
    _refused(L, name, PAGED, "EINVAL", "null buffer", table=None)
    for size in (0, -32, 16, 48):
        _refused(L, name, PAGED, "EINVAL", "power of two", page_size=size)
    for key in ("max_pages", "num_pages"):
        _refused(L, name, PAGED, "EINVAL", "positive", **{key: 0})
    _refused(L, name, PAGED, "ERANGE", "capacity", length=129)


def test_tree_workspace_is_zero_for_sizes_that_are_refused(L):
    good = dict(batch=2, nodes=8, q_heads=8, kv_heads=2, key_dim=64, value_dim=64, length=4000,
                dtype=1)
    size = L.lib().alpx_tree_workspace_bytes
    assert size(*good.values()) > 0
    for key, bad in (("batch", 0), ("nodes", -1), ("q_heads", 7), ("kv_heads", 0),
                     ("key_dim", 300), ("value_dim", 0), ("length", 0), ("dtype", 9)):
        assert size(*dict(good, **{key: bad}).values()) == 0


def test_tree_workspace_is_zero_for_rows_and_sequences_past_the_range(L):
    good = dict(batch=2, nodes=8, q_heads=8, kv_heads=2, key_dim=64, value_dim=64, length=4000,
                dtype=1)
    size = L.lib().alpx_tree_workspace_bytes
    for bad in (dict(length=(1 << 30) + 1), dict(length=2 ** 31 - 1), dict(length=1 << 30, batch=64),
                dict(batch=2 ** 31 - 1, length=32), dict(nodes=1 << 24),
                dict(batch=1 << 20, nodes=1 << 10, q_heads=1 << 10, kv_heads=1 << 10)):
        args = dict(good, **bad)
        assert size(*args.values()) == 0
        # as the call: no workspace that it would take
        names = ("batch", "nodes", "q_heads", "kv_heads", "key_dim", "value_dim", "length", "dtype")
        call = dict(dict(TREE, words=1 << 20, out=1 << 60), **{k: args[k] for k in names})
        _refused(L, "alpx_tree_attention", call, "EUNSUPPORTED", "too many")


def test_tree_attention_refuses_counts_past_31_bits(L):
    # a slot's first tile is slot x tiles per slot, rounded up: with up to 2048
    # slots the tiles have to end that far below 2^31; mask words count twice
    # (2048 sequences of 2^20 - 1 tiles are 2^31 - 2048)
    size = L.lib().alpx_tree_workspace_bytes
    rows = 32 * (2 ** 20 - 2)
    assert size(2048, 8, 8, 2, 64, 64, rows, 1) == 0 < size(2000, 8, 8, 2, 64, 64, rows, 1)
    _refused(L, "alpx_tree_attention", dict(TREE, out=1 << 60), "EUNSUPPORTED", "too many rows",
             batch=2048, length=rows)
    for name, args in (("alpx_tree_attention", TREE), ("alpx_tree_attention_paged", PAGED)):
        _refused(L, name, args, "EINVAL", "mask_words", words=1 << 30)


def test_tree_masks_refusals(L):
    name = "alpx_tree_masks"
    args = dict(parents=FAKE, counts=None, lengths=FAKE, masks=FAKE, depths=FAKE, lanes=FAKE,
                batch=2, nodes=65, words=2, stream=None)
    for key in ("parents", "masks", "depths", "lengths"):
        _refused(L, name, args, "EINVAL", "null buffer", **{key: None})
    for key in ("batch", "nodes"):
        _refused(L, name, args, "EINVAL", "positive", **{key: 0})
    for words in (1, 3, -1):
        _refused(L, name, args, "EINVAL", "mask_words", words=words)
    _refused(L, name, args, "EUNSUPPORTED", "1024", nodes=1025, words=17)
    _refused(L, name, args, "EINVAL", "aligned", lanes=FAKE + 8)


def test_tree_commit_refusals(L):
    args = dict(k=FAKE, v=FAKE, paths=FAKE, accepted=FAKE, prefix=FAKE, dtype=1, capacity=100,
                batch=2, kv_heads=2, key_dim=64, value_dim=64, path_max=5, stream=None)
    paged = dict(k=FAKE, v=FAKE, table=FAKE, max_pages=4, page_size=32, num_pages=9, paths=FAKE,
                 accepted=FAKE, prefix=FAKE, dtype=1, batch=2, kv_heads=2, key_dim=64,
                 value_dim=64, path_max=5, stream=None)
    for name, base in (("alpx_tree_commit", args), ("alpx_tree_commit_paged", paged)):
        for key, value in base.items():
            if value == FAKE:
                _refused(L, name, base, "EINVAL", "null buffer", **{key: None})
        for key in ("capacity", "max_pages", "num_pages", "batch", "kv_heads", "key_dim",
                    "value_dim", "path_max"):
            if key in base:
                _refused(L, name, base, "EINVAL", "positive", **{key: 0})
        _refused(L, name, base, "EINVAL", "dtype", dtype=7)
    for size in (0, 3, 48):
        _refused(L, "alpx_tree_commit_paged", paged, "EINVAL", "power of two", page_size=size)


def test_paged_resize_refusals(L):
    name = "alpx_paged_resize"
    args = dict(table=FAKE, lengths=FAKE, free=FAKE, count=FAKE, targets=FAKE, batch=2, max_pages=4,
                page_size=32, num_pages=9, tokens=64, starts=FAKE, slots=FAKE, positions=FAKE,
                sequences=FAKE, granted=FAKE, scratch=FAKE, stream=None)
    for key, value in args.items():
        if value == FAKE:
            _refused(L, name, args, "EINVAL", "null buffer", **{key: None})
    for key in ("batch", "max_pages", "num_pages"):
        _refused(L, name, args, "EINVAL", "positive", **{key: 0})
    _refused(L, name, args, "EINVAL", "positive", tokens=-1)
    for size in (0, 3, 48, -32):
        _refused(L, name, args, "EINVAL", "power of two", page_size=size)
    _refused(L, name, args, "EUNSUPPORTED", "2^31", num_pages=1 << 26)
    _refused(L, name, args, "EUNSUPPORTED", "2^31", max_pages=1 << 26)
    _refused(L, name, args, "EUNSUPPORTED", "2^20", max_pages=(1 << 20) + 1, page_size=1)


def test_paged_resize_refuses_tokens_past_its_grid(L):
    # blocks of 256 rows are counted in 31 bits
    args = dict(table=FAKE, lengths=FAKE, free=FAKE, count=FAKE, targets=FAKE, batch=2, max_pages=4,
                page_size=32, num_pages=9, tokens=2 ** 31 - 255, starts=FAKE, slots=FAKE,
                positions=FAKE, sequences=FAKE, granted=FAKE, scratch=FAKE, stream=None)
    for tokens in (2 ** 31 - 255, 2 ** 31 - 1):
        _refused(L, "alpx_paged_resize", args, "EUNSUPPORTED", "tokens", tokens=tokens)


def test_prologue_rows_refusals(L):
    name = "alpx_attention_prologue_rows"
    sections = (ctypes.c_int * 4)(11, 11, 10, 0)
    args = dict(qg=FAKE, k=FAKE, v=FAKE, qw=FAKE, kw=FAKE, q=FAKE, g=FAKE, kr=FAKE, vr=FAKE,
                rows=64, slots=FAKE, lanes=FAKE, dtype=1, tokens=3, q_heads=8, kv_heads=2,
                head_dim=128, value_dim=128, sections=sections, base=1e7, eps=1e-6, stream=None)
    for key, value in args.items():
        if isinstance(value, int) and value == FAKE:
            _refused(L, name, args, "EINVAL", "null buffer", **{key: None})
    _refused(L, name, args, "EINVAL", "null buffer", sections=None)
    for key in ("rows", "tokens", "q_heads", "kv_heads", "head_dim", "value_dim"):
        _refused(L, name, args, "EINVAL", "positive", **{key: 0})
    _refused(L, name, args, "EINVAL", "multiple of KV heads", q_heads=9)
    _refused(L, name, args, "EINVAL", "dtype", dtype=3)
    for key in ("head_dim", "value_dim"):
        _refused(L, name, args, "EUNSUPPORTED", "above 512", **{key: 513})
    _refused(L, name, args, "EINVAL", "rotary pair", sections=(ctypes.c_int * 4)(0, 0, 0, 0))
    _refused(L, name, args, "EINVAL", "shorter", head_dim=62)
    for value in (0.0, float("nan"), float("inf")):
        _refused(L, name, args, "EINVAL", "frequency_base", base=value)
        _refused(L, name, args, "EINVAL", "epsilon", eps=value)


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
    for name in ("tree_attention", "tree_masks", "tree_commit", "paged_resize",
                 "attention_prologue_rows"):
        monkeypatch.setattr(m._ops, name, reached)
    return o


def _i32(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def test_facade_refuses_host_tensors(pkg):
    m = importlib.import_module(pkg.__name__ + ".qwen35_rocm_ops")
    o = m.Qwen35RocmOps(_capability=m.RocmCapability(True, "injected", 0, "gfx950"))
    f = torch.zeros(2, 2, 2, 2)
    with pytest.raises(TypeError, match="must remain on the ROCm device"):
        o.tree_attention(f, f, f, f, length=2, prefix_lens=[0, 0])
    with pytest.raises(TypeError, match="must remain on the ROCm device"):
        o.paged_tree_attention(f, f, f, _i32(2, 2), f, length=2, prefix_lens=[0, 0])
    with pytest.raises(TypeError, match="must remain on the ROCm device"):
        o.tree_commit_(f, f, _i32(2, 2), prefix_lens=[0, 0], accepted=[0, 0])
    with pytest.raises(TypeError, match="must remain on the ROCm device"):
        o.paged_resize_(_i32(2, 2), _i32(2), _i32(4), _i32(1), [1, 1], page_size=32, tokens=2)
    with pytest.raises(TypeError, match="must remain on the ROCm device"):
        o.tree_masks(_i32(2, 2))


def _attend(ops, paged=False, **changes):
    a = dict(query=torch.zeros(2, 8, 4, 64), masks=torch.zeros(2, 8, 1, dtype=torch.int64),
             length=60, prefix_lens=_i32(2))
    if paged:
        a.update(key_pages=torch.zeros(5, 32, 2, 64), value_pages=torch.zeros(5, 32, 2, 48),
                 block_table=_i32(2, 2))
    else:
        a.update(key_cache=torch.zeros(64, 2, 2, 64), value_cache=torch.zeros(64, 2, 2, 48))
    a.update(changes)
    return (ops.paged_tree_attention if paged else ops.tree_attention)(**a)


@pytest.mark.parametrize("paged", [False, True])
def test_facade_tree_attention_refusals(ops, paged):
    with pytest.raises(AssertionError, match="passed"):
        _attend(ops, paged)
    f, i64 = torch.zeros, torch.int64
    for error, text, changes in [
            (ValueError, "exceeds capacity", dict(length=65)),
            (ValueError, "positive integer", dict(length=0)),
            (ValueError, "batch/head width", dict(query=f(3, 8, 4, 64))),
            (ValueError, "batch/head width", dict(query=f(2, 8, 4, 32))),
            (ValueError, "at least one draft", dict(query=f(2, 0, 4, 64))),
            (ValueError, "multiple of KV heads", dict(query=f(2, 8, 5, 64))),
            (TypeError, "share one dtype", dict(query=f(2, 8, 4, 64, dtype=torch.bfloat16))),
            (TypeError, "int64", dict(masks=_i32(2, 8, 1))),
            (ValueError, "64 drafts a word", dict(masks=f(2, 8, dtype=i64))),
            (ValueError, "64 drafts a word", dict(masks=f(3, 8, 1, dtype=i64))),
            (ValueError, "64 drafts a word", dict(masks=f(2, 7, 1, dtype=i64))),
            (ValueError, "64 drafts a word", dict(masks=f(2, 8, 0, dtype=i64))),
            (ValueError, "contiguous", dict(masks=f(2, 1, 8, dtype=i64).transpose(1, 2)[:, ::2])),
            (ValueError, "match the attention output", dict(gate=f(2, 8, 4, 64))),
            (ValueError, "one entry", dict(prefix_lens=[0])),
            (ValueError, "one entry", dict(prefix_lens=[0, 61])),
            (ValueError, "one entry", dict(prefix_lens=[0, -1])),
            (ValueError, "one entry", dict(counts=[1, 9])),
            (ValueError, "positive and finite", dict(scale=0.0)),
            (ValueError, "expected", dict(out=f(2, 8, 4, 64))),
            (TypeError, "bfloat16", dict(out=f(2, 8, 4, 48), out_dtype=torch.bfloat16))]:
        with pytest.raises(error, match=text):
            _attend(ops, paged, **changes)


def test_facade_refuses_numbers_past_32_bits(ops, monkeypatch):
    # a C int would take the low 32 bits of them
    wide = torch.zeros(1, dtype=torch.int32).expand(2, 2 ** 28)
    monkeypatch.setattr(ops, "_paged", lambda keys, values, table: (keys, values))
    with pytest.raises(ValueError, match="2\\^31"):
        _attend(ops, True, length=2 ** 32 + 5, block_table=wide)
    # (only the checks of host tensors stand between the call and its sizes)
    monkeypatch.setattr(ops, "_device_ints", lambda value, *a, **k: value)

    class OnDevice(torch.Tensor):
        is_cuda = True

    def ints(*shape):
        return _i32(*shape).as_subclass(OnDevice)
    for kw in (dict(page_size=2 ** 32, tokens=2), dict(page_size=2 ** 30, tokens=2),
               dict(page_size=32, tokens=2 ** 32 + 2)):
        with pytest.raises(ValueError, match="2\\^31"):
            ops.paged_resize_(ints(2, 2), ints(2), ints(4), ints(1), ints(2), **kw)
    with pytest.raises(AssertionError, match="passed"):
        ops.paged_resize_(ints(2, 2), ints(2), ints(4), ints(1), ints(2), page_size=32, tokens=2)


def test_facade_takes_whole_host_numbers_only(ops):
    import numpy as np
    for bad in ([3.7, 1], [3.0, 1], [True, 1], np.array([1.5, 2.0]), torch.tensor([1.5, 2.0]),
                ["1", 2], [None, 1]):
        for key in ("prefix_lens", "counts"):
            with pytest.raises(ValueError, match="integers"):
                _attend(ops, **{key: bad})
    ops.device = "cpu"  # where the accepted ones go
    for good in ([3, 1], (0, 8), iter([3, 1]), np.array([1, 2], dtype=np.int64), np.array([1, 2], dtype=np.int8),
                 torch.tensor([1, 2])):
        with pytest.raises(AssertionError, match="passed"):
            _attend(ops, counts=good)


def test_facade_refuses_tokens_past_the_grid(ops, monkeypatch):
    monkeypatch.setattr(ops, "_device_ints", lambda value, *a, **k: value)

    class OnDevice(torch.Tensor):
        is_cuda = True

    def ints(*shape):
        return _i32(*shape).as_subclass(OnDevice)
    for tokens, error, text in ((2 ** 31 - 256, AssertionError, "passed"),
                                (2 ** 31 - 255, ValueError, "2\\^31")):
        with pytest.raises(error, match=text):
            ops.paged_resize_(ints(2, 2), ints(2), ints(4), ints(1), ints(2), page_size=32,
                              tokens=tokens)


def test_facade_masks_commit_and_resize_refusals(ops):
    with pytest.raises(ValueError, match=r"\[batch, nodes\]"):
        ops.tree_masks([[-1, 0]])
    with pytest.raises(ValueError, match="1 to 1024"):
        ops.tree_masks(_i32(1, 1025))
    with pytest.raises(ValueError, match="1 to 1024"):
        ops.tree_masks(_i32(2, 0))
    with pytest.raises(ValueError, match="one entry"):
        ops.tree_masks(_i32(2, 4), counts=[4, 5])
    with pytest.raises(ValueError, match="one entry"):
        ops.tree_masks(_i32(2, 4), lengths=[0, -1])

    k, v, paths = torch.zeros(64, 2, 2, 64), torch.zeros(64, 2, 2, 48), _i32(2, 5)
    with pytest.raises(ValueError, match="capacity, batch, or heads"):
        ops.tree_commit_(k, v[:, :1].contiguous(), paths, prefix_lens=[0, 0], accepted=[0, 0])
    with pytest.raises(TypeError, match="share one dtype"):
        ops.tree_commit_(k, v.half(), paths, prefix_lens=[0, 0], accepted=[0, 0])
    with pytest.raises(ValueError, match="one entry"):
        ops.tree_commit_(k, v, paths, prefix_lens=_i32(2), accepted=[0, 6])
    with pytest.raises(ValueError, match=r"\[batch, steps\]"):
        ops.tree_commit_(k, v, _i32(2, 0), prefix_lens=_i32(2), accepted=_i32(2))
    pages = torch.zeros(5, 32, 2, 64)
    with pytest.raises(TypeError, match="block table"):
        ops.paged_tree_commit_(pages, pages, torch.zeros(2, 2), paths, prefix_lens=_i32(2),
                               accepted=_i32(2))

    with pytest.raises(TypeError, match="block table"):
        ops.paged_resize_([[0]], _i32(1), _i32(4), _i32(1), [1], page_size=32, tokens=2)
    with pytest.raises(ValueError, match="cannot be empty"):
        ops.paged_resize_(_i32(0, 2), _i32(0), _i32(4), _i32(1), [], page_size=32, tokens=2)
    with pytest.raises(TypeError, match="one-dimensional device tensor"):
        ops.paged_resize_(_i32(2, 2), [0, 0], _i32(4), _i32(1), [1, 1], page_size=32, tokens=2)


def test_facade_prologue_refusals(ops):
    a = dict(query_gate=torch.zeros(3, 4 * 128), key=torch.zeros(3, 2 * 64),
             value=torch.zeros(3, 2 * 48), query_norm=torch.ones(64), key_norm=torch.ones(64),
             key_pages=torch.zeros(5, 32, 2, 64), value_pages=torch.zeros(5, 32, 2, 48),
             slots=_i32(3), position_lanes=torch.zeros(3, 4, dtype=torch.int64),
             sections=(11, 11, 10, 0), frequency_base=1e7, epsilon=1e-6)
    with pytest.raises(AssertionError, match="passed"):
        ops.paged_attention_prologue_rows_(**a)
    f = torch.zeros
    for error, text, changes in [
            (ValueError, "count, size or heads", dict(value_pages=f(5, 16, 2, 48))),
            (ValueError, "at least one token", dict(query_gate=f(0, 512))),
            (ValueError, "page head width", dict(query_gate=f(3, 500))),
            (ValueError, "multiple of KV heads", dict(query_gate=f(3, 3 * 128))),
            (ValueError, "page token shape", dict(key=f(3, 64))),
            (ValueError, "page token shape", dict(value=f(2, 96))),
            (ValueError, "head dimension", dict(key_norm=f(32))),
            (TypeError, "float32", dict(query_norm=torch.ones(64).half())),
            (TypeError, "share one dtype", dict(key=f(3, 128).half())),
            (ValueError, "one entry", dict(slots=[0, 1])),
            (ValueError, "one entry", dict(slots=[0, 1, 160])),
            (ValueError, "int64", dict(position_lanes=_i32(3, 4))),
            (ValueError, "int64", dict(position_lanes=f(3, 3, dtype=torch.int64))),
            (ValueError, "four sections", dict(sections=(16, 16))),
            (ValueError, "nonnegative|non-negative", dict(sections=(16, 16, -1, 0))),
            (ValueError, "frequency_base", dict(frequency_base=0.0)),
            (ValueError, "epsilon", dict(epsilon=float("nan")))]:
        with pytest.raises(error, match=text):
            ops.paged_attention_prologue_rows_(**dict(a, **changes))
