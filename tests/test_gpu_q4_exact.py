"""What the attention over 4-bit pools gives before its output's rounding
(float32 output whatever the queries' type), against the float64 oracle.

Tolerances.  A weight p is off by what its score is, and by 2^-22 for its two
float16 parts; p times a step by 2^-22 more.  Scores of deviation 1 stay below 8
in size, so that float32 forms them, and the exponential, within 2^-20 or so
(queries of 16 bits against codes as they stand: 2^-18).  A row's share of a
channel is thus off by less than 2^-17 of its gross p (|least| + step code),
and a channel by less than 2^-17 of the weighted gross.  The rows' errors are
independent and values have mean zero, so the 2-norm of all channels' errors
is below 2^-17 of the result's, on any number of rows."""

import importlib

import numpy as np
import pytest

from oracle import inputs as I
from oracle import q4 as Q
from tests.test_gpu_q4 import PKG, Case, _host, _td, _up

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(gpu):
    return importlib.import_module(PKG + ".qwen35_rocm_ops").Qwen35RocmOps()


def _close(case, ops, bound, extra=0.0, **kw):
    got = _host(case.call(ops, out_dtype=_td("f32"), **kw))
    want, weight = case.oracle(kw.get("scale"), True)
    assert np.isfinite(got).all()
    off = np.abs(got - want)
    assert (off <= bound * weight + extra).all(), np.max(off / (weight + 1e-30))
    return got, want


def _coarse(case, step):
    """What large steps cost: weights are formed 2^lift smaller, for a step below
    2^lift, so that their products with it stay in float16.  The largest one is
    then 2^(11 - lift) at least, and a row's, and its product with any step, are
    off by 2^-25 and twice 2^-25 at most where float16 is subnormal: times |least
    + 8 step| <= gross and |code - 8| <= 8, 2^-25 (16 + gross) a row."""
    lift = np.frexp(step)[1]
    lost = np.zeros(case.q.shape)
    for b, slots in enumerate(case.slots):
        k, gross = Q.get(case.pool[:2], slots), Q.gross(case.pool[2:], slots)
        for i in range(case.counts[b]):
            n = case.prefix[b] + i + 1
            for h in range(case.q.shape[2]):
                kv = h // (case.q.shape[2] // k.shape[1])
                s = (k[:n, kv].astype(np.float64) @ case.q[b, i, h]) * case.d ** -0.5
                lost[b, i, h] = (16 + gross[:n, kv]).sum(0) / np.exp(s - s.max()).sum()
    return 2.0 ** (lift - 36) * lost


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_least_and_step_are_cut_where_float16_ends(gpu, ops, dtype):
    """The numbers of the definition, by hand, stored and read back."""
    import torch
    x = torch.zeros(3, 1, 64, device=gpu)
    x[0], x[1, :, :16], x[1, :, 16:] = 3e38, 20480.0, 122880.0
    x[2, :, ::2], x[2, :, 1::2] = -3e38, 3e38
    pool = ops.initialize_paged_q4_workspace(num_pages=1, page_size=32, kv_heads=1,
                                             head_dimension=64).arrays
    x = x.to(_td(dtype))
    ops.paged_q4_append_rows_(None, x, x, *pool, [0, 1, 2], None, rotary_dimension=0)
    for got in ops.paged_q4_rows(*pool, [0, 1, 2]):
        assert (got[0] == 16 * 65504).all()
        # (102400 / 15 = 6826.7, of steps 4 apart 6828)
        assert (got[1, :, :16] == 20480).all() and (got[1, :, 16:32] == 20480 + 15 * 6828).all()
        # (57376 / 15 = 3825.07 above least, of steps 2 apart 3826)
        assert (got[1, :, 32:] == 65504 + 15 * 3826).all()
        assert (got[2, :, ::2] == -65504).all() and (got[2, :, 1::2] == 14 * 65504).all()


# Groups whose middle, least + 8 steps, float16 does not hold.
FAR_GROUPS = [(60000.0, 80000.0), (20000.0, 120000.0), (-1000.0, 900000.0)]
FAR_SHAPES = [(64, 4, 1), (96, 6, 2), (128, 4, 1), (128, 8, 3), (128, 32, 1), (128, 8, 10),
              (256, 4, 1), (256, 4, 6), (256, 8, 9), (64, 8, 9), (96, 8, 9)]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("d,hq,nodes", FAR_SHAPES)
@pytest.mark.parametrize("span", FAR_GROUPS)
def test_values_past_what_float16_holds(gpu, ops, dtype, d, hq, nodes, span):
    """Some of V's groups lie about a middle past 65504."""
    case = Case(gpu, 60, dtype=dtype, d=d, hq=hq, hkv=2, nodes=nodes, prefix=[700, 33])
    rng = np.random.default_rng(61)
    for row in (0, 5, 32, 33):
        case.v[:, row, :, 32:64] = rng.uniform(*span, case.v[:, row, :, 32:64].shape)
    case.v[0, 690:700, 1, :32] = rng.uniform(*span, (10, 32))
    case.store()
    _close(case, ops, 2.0 ** -17, _coarse(case, (span[1] - span[0]) / 15))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("d,hq", [(64, 4), (128, 8), (256, 8)])
@pytest.mark.parametrize("which", ["k", "v"])
def test_values_past_what_float16_holds_stay_with_the_tokens_that_see_them(gpu, ops, dtype, d, hq,
                                                                          which):
    """They lie in the last tokens' rows; those before see none of them."""
    for nodes in (2, 7, 20):
        case = Case(gpu, 62, dtype=dtype, d=d, hq=hq, hkv=2, nodes=nodes, prefix=[600, 30])
        rng = np.random.default_rng(63)
        x = case.k if which == "k" else case.v
        if which == "k":  # (scores that a softmax is still one of)
            case.q[:] = I.round_to(case.q * 2.0 ** -20, dtype)
        for b in range(2):
            at = case.prefix[b] + nodes - 1
            x[b, at, :, :32] = rng.uniform(20000.0, 120000.0, x[b, at, :, :32].shape)
        case.store()
        _close(case, ops, 2.0 ** -17, _coarse(case, 1e5 / 15) if which == "v" else 0.0)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("d,hq,nodes", FAR_SHAPES)
def test_keys_past_what_float16_holds(gpu, ops, dtype, d, hq, nodes):
    """Terms of a score sum to less than 2^5 in size, of which a float32 sum
    loses 2^-20 at most: 2^-15 of a weight."""
    case = Case(gpu, 64, dtype=dtype, d=d, hq=hq, hkv=2, nodes=nodes, prefix=[700, 33])
    rng = np.random.default_rng(65)
    case.q[:] = I.round_to(case.q * 2.0 ** -16, dtype)
    for row in (0, 5, 32, 33):
        case.k[:, row, :, 32:64] = rng.uniform(60000.0, 80000.0, case.k[:, row, :, 32:64].shape)
    case.store()
    _close(case, ops, 2.0 ** -15)


@pytest.mark.parametrize("dtype,d,hq,hkv,nodes,rows,batch", [
    ("f16", 128, 8, 2, 1, 500, 2), ("f16", 128, 8, 2, 1, 20000, 1), ("bf16", 128, 8, 2, 1, 131072, 1),
    ("f16", 64, 8, 2, 1, 131072, 1), ("f32", 128, 8, 2, 1, 131072, 1), ("f16", 128, 8, 2, 1, 8192, 64),
    ("f16", 96, 6, 2, 4, 8192, 2), ("bf16", 256, 8, 1, 1, 32768, 2), ("f32", 256, 8, 1, 2, 8192, 1),
    ("f16", 128, 8, 2, 64, 32768, 1), ("bf16", 128, 8, 2, 64, 4133, 2), ("f32", 128, 8, 2, 64, 32768, 1),
    ("bf16", 256, 8, 1, 33, 8192, 1)])
def test_no_more_is_lost_on_more_rows(gpu, ops, dtype, d, hq, hkv, nodes, rows, batch):
    """Values of mean zero: what is left of their sum shrinks beside its terms
    as rows grow.  Against float64 products here on the device."""
    import torch
    g = torch.Generator(device=gpu).manual_seed(rows)
    page = 64
    per = -(-rows // page)
    pool = ops.initialize_paged_q4_workspace(num_pages=batch * per, page_size=page, kv_heads=hkv,
                                             head_dimension=d).arrays
    slots = torch.arange(batch * per * page, dtype=torch.int32, device=gpu)
    for part in slots.split(32768):
        k, v = (torch.randn(part.numel(), hkv, d, generator=g, device=gpu) for _ in range(2))
        ops.paged_q4_append_rows_(None, k, v, *pool, part, None, rotary_dimension=0)
    q = torch.randn(batch, nodes, hq, d, generator=g, device=gpu).to(_td(dtype))
    got = ops.paged_q4_attention(
        q, *pool, torch.arange(batch * per, dtype=torch.int32, device=gpu).view(batch, per),
        length=rows, prefix_lens=[rows - nodes] * batch, out_dtype=torch.float32).double()
    want = torch.empty_like(got)
    seen = torch.arange(rows, device=gpu) <= \
        rows - nodes + torch.arange(nodes, device=gpu).unsqueeze(1)
    for b in range(batch):
        k, v = ops.paged_q4_rows(*pool, slots[b * per * page:][:rows])
        for h in range(hq):
            kv = h // (hq // hkv)
            kt = k[:, kv].double().t().contiguous()
            s = (q[b, :, h].double() @ kt) * d ** -0.5
            p = torch.softmax(s.masked_fill(~seen, float("-inf")), -1)
            want[b, :, h] = p @ v[:, kv].double().contiguous()
    assert (got - want).norm() <= 2.0 ** -17 * want.norm()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("d,hq,nodes", [(64, 4, 1), (128, 8, 2), (128, 8, 9), (256, 8, 3)])
@pytest.mark.parametrize("size,scale", [(2.0 ** -24, 1e-38), (1.0, 1e-44), (2.0 ** -20, 1e-30)])
def test_scores_too_small_for_float32(gpu, ops, dtype, d, hq, nodes, size, scale):
    """All scores are as good as 0: the mean of the rows that a token sees."""
    case = Case(gpu, 67, dtype=dtype, d=d, hq=hq, hkv=2, nodes=nodes, prefix=[600, 30])
    case.q[:] = I.round_to(case.q * size, dtype)
    _close(case, ops, 2.0 ** -17, scale=scale)


# Column classes of a kv head: up to 4, up to 8, up to 16, and more (one column
# tile of 32, and several with an end inside).
COLUMNS = {"4": (4, 1), "3": (3, 1), "8": (4, 2), "6": (6, 1), "16": (8, 2), "10": (5, 2),
           "27": (3, 9), "40": (8, 5)}


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("d", [64, 96, 128, 256])
@pytest.mark.parametrize("columns", list(COLUMNS))
def test_every_kernel_matches_the_oracle(gpu, ops, dtype, d, columns):
    """Every type, width and class of columns, on whole sequences (one launch)
    and on shares of them (two), with a tile and a page that end inside."""
    group, nodes = COLUMNS[columns]
    for prefix in ([100, 0, 33], [1301, 70]):
        case = Case(gpu, 66, dtype=dtype, d=d, hq=2 * group, hkv=2, nodes=nodes, prefix=prefix)
        got, want = _close(case, ops, 2.0 ** -17)
        assert np.linalg.norm(got - want) <= 2.0 ** -17 * np.linalg.norm(want)


@pytest.mark.parametrize("dtype,d", [("bf16", 256), ("f16", 128), ("f32", 64)])
def test_normed_heads_reach_codes_over_a_float_pool(gpu, ops, dtype, d):
    """Heads with a norm and a gate of their own: their prologue writes a float
    pool of the call's rows, which are stored as they are."""
    import torch
    rng = np.random.default_rng(70)
    tokens, hq, hkv, page = 21, 4, 2, 32
    qg = _up(gpu, rng.standard_normal((tokens, hq * 2 * d)), dtype)
    k, v = (_up(gpu, rng.standard_normal((tokens, hkv * d)), dtype) for _ in range(2))
    weights = [_up(gpu, rng.uniform(0.5, 1.5, d).astype(np.float32)) for _ in range(2)]
    rows = torch.zeros(2, 1, page, hkv, d, dtype=_td(dtype), device=gpu)
    at = torch.arange(tokens, dtype=torch.int32, device=gpu)
    lanes = torch.from_numpy(rng.integers(0, 5000, (tokens, 4))).to(gpu)
    ops.paged_attention_prologue_rows_(qg, k, v, *weights, rows[0], rows[1], at, lanes,
                                       sections=(8, 8, 8, 8), frequency_base=1e7, epsilon=1e-6)
    pages = 3
    pool = ops.initialize_paged_q4_workspace(num_pages=pages, page_size=page, kv_heads=hkv,
                                             head_dimension=d).arrays
    slots = rng.permutation(pages * page)[:tokens].astype(np.int32)
    ops.paged_q4_append_rows_(None, rows[0, 0, :tokens], rows[1, 0, :tokens], *pool,
                              _up(gpu, slots), None, rotary_dimension=0)
    for i in range(2):
        want = Q.empty_pool(pages, hkv, page, d)
        Q.put(want, slots, _host(rows[i, 0, :tokens]))
        assert np.abs(_host(rows[i, 0, :tokens])).max() > 1.0
        assert np.array_equal(pool[2 * i].cpu().numpy(), want[0])
        assert np.array_equal(pool[2 * i + 1].cpu().numpy(), want[1])
