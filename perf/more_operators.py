"""What decoding over a page pool of 4 bits a value is timed on.

Such a server turns the new tokens' queries and keys by their positions and
writes keys and values to their pool rows, in the pool's own type (``rotary``)
or as 4-bit codes with a step and a least value per 32 channels (``store``),
reads rows of codes back as numbers (``rows``: a prompt's chunk attends to a
stored prefix, a snapshot), lets a token, or a run of drafted ones, attend to
the codes (``attend``), and decides from given random numbers which drafted
tokens stand and what comes behind them (``verify``).

``run`` computes them in elementary torch operations, or, where ``own`` is
true, through ``Qwen35RocmOps``.
"""

import importlib
import math

import torch

own = False

PACKAGE = "alpacca-open-sourced-by-jt_amd"
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
ROPE_BASE = 5.0e5
GROUP = 32  # channels that share a step and a least value

_facade = []


def _ops():
    if not _facade:
        module = importlib.import_module(PACKAGE + ".qwen35_rocm_ops")
        _facade.append(module.Qwen35RocmOps(device_index=0))
    return _facade[0]


# ------------------------------------------------------------------ cases


def listed():
    return [
        # one chat user on a small llama in the engine's float32: the smallest
        # append, all latency
        dict(name="rotary_f32_1", kind="rotary", tokens=1, q_heads=32, kv_heads=8, dim=64,
             rotary=64, style="norm", dtype="f32", page=64),
        # prompts of mixed lengths, packed
        dict(name="rotary_bf16_4133", kind="rotary", tokens=4133, q_heads=32, kv_heads=8, dim=128,
             rotary=128, style="norm", dtype="bf16", page=32),
        # one token of each sequence of a serving batch
        dict(name="store_f16_16", kind="store", tokens=16, q_heads=32, kv_heads=8, dim=128,
             rotary=128, style="norm", dtype="f16", page=64),
        # a prompt, heads of 256 with a quarter of them turned
        dict(name="store_bf16_4133", kind="store", tokens=4133, q_heads=16, kv_heads=2, dim=256,
             rotary=64, style="neox", dtype="bf16", page=64),
        # the stored prefix of a prompt that goes on
        dict(name="rows_bf16_8192", kind="rows", tokens=8192, kv_heads=8, dim=128, dtype="bf16",
             page=64),
        # one chat user on a small llama, a short chat: the smallest attention
        dict(name="attend_f32_1_on_500", kind="attend", batch=1, nodes=1, q_heads=32, kv_heads=8,
             dim=64, length=500, dtype="f32", page=64, gate=False),
        # a serving batch at mixed lengths, the most rows
        dict(name="attend_f16_16x1_ragged_8k", kind="attend", batch=16, nodes=1, q_heads=32,
             kv_heads=8, dim=128, length=8192, dtype="f16", page=64, gate=False),
        # a gated attention layer of head width 256 at a long context
        dict(name="attend_bf16_4x1_on_32k", kind="attend", batch=4, nodes=1, q_heads=16,
             kv_heads=2, dim=256, length=32768, dtype="bf16", page=256, gate=True),
        # the ends of four prompts, or long drafts: the most arithmetic, pages
        # that end inside a tile
        dict(name="attend_bf16_4x64_on_4k", kind="attend", batch=4, nodes=64, q_heads=32,
             kv_heads=8, dim=128, length=4133, dtype="bf16", page=32, gate=False),
        # one user's chain of drafts from a small model
        dict(name="verify_f32_1x8", kind="verify", batch=1, nodes=8, vocab=32768, dtype="f32",
             tree=False, draft=True),
        # a full house with short chains
        dict(name="verify_f32_64x6", kind="verify", batch=64, nodes=6, vocab=131101, dtype="f32",
             tree=False, draft=True),
        # trees of the likeliest continuations, which no distribution drew
        dict(name="verify_bf16_32x24", kind="verify", batch=32, nodes=24, vocab=131101,
             dtype="bf16", tree=True, draft=False),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


LLAMA_HEADS = ((32, 8), (32, 8), (24, 8), (8, 8))
QWEN_HEADS = ((16, 2), (16, 2), (8, 2), (24, 4))
MOST_VALUES = 1 << 27  # of K, in a drawn attention case
MOST_FLOPS = 1.7e10
MOST_ENTRIES = 1 << 25  # of the target's probabilities, in a drawn verification


def draw(rng):
    kind = rng.choice(["rotary", "store", "rows"] + ["attend"] * 4 + ["verify"] * 2)
    q_heads, kv_heads = rng.choice(LLAMA_HEADS + QWEN_HEADS)
    wide = (q_heads, kv_heads) in QWEN_HEADS
    dim = 256 if wide else rng.choice([64, 96, 128, 128])
    dtype = rng.choice(["f16", "bf16", "bf16", "f32"])
    page = rng.choice([32, 64, 256])
    if kind == "attend":
        batch, nodes = _log_int(rng, 1, 32), rng.choice([1, _log_int(rng, 1, 64)])
        rows = min(MOST_VALUES // (kv_heads * dim), int(MOST_FLOPS / (4 * dim * q_heads * nodes)))
        most = max(nodes + 1, min(32768, rows // batch))
        return dict(kind=kind, batch=batch, nodes=nodes, q_heads=q_heads, kv_heads=kv_heads,
                    dim=dim, length=_log_int(rng, min(most, nodes + 64), most), dtype=dtype,
                    page=page, gate=wide)
    if kind == "verify":
        vocab = _log_int(rng, 1000, 200000)
        nodes = _log_int(rng, 1, 32)
        tree, draft = rng.random() < 0.5, rng.random() < 0.6
        if tree and draft:
            nodes = min(nodes, 12)
        most = max(1, min(64, MOST_ENTRIES // (vocab * nodes)))
        return dict(kind=kind, batch=_log_int(rng, 1, most), nodes=nodes, vocab=vocab,
                    dtype=dtype, tree=tree, draft=draft)
    if kind == "rows":
        return dict(kind=kind, tokens=_log_int(rng, 1, 8192), kv_heads=kv_heads, dim=dim,
                    dtype=dtype, page=page)
    return dict(kind=kind, tokens=_log_int(rng, 1, 4096), q_heads=q_heads, kv_heads=kv_heads,
                dim=dim, rotary=64 if wide else dim, style="neox" if wide else "norm",
                dtype=dtype, page=page)


# ------------------------------------------------------------------ inputs


class _Draw:
    """Seeded values on the GPU."""

    def __init__(self, seed):
        self.gen = torch.Generator(device="cuda")
        self.gen.manual_seed(seed)

    def normal(self, *shape, dtype=torch.float32):
        return torch.randn(shape, generator=self.gen, device="cuda").to(dtype)

    def uniform(self, *shape):
        return torch.rand(shape, generator=self.gen, device="cuda")

    def integers(self, lo, hi, *shape):
        """In ``[lo, hi]``."""
        return torch.randint(lo, hi + 1, shape, generator=self.gen, device="cuda",
                             dtype=torch.int32)

    def order(self, n):
        return torch.randperm(n, generator=self.gen, device="cuda").to(torch.int32)

    def keys(self, *shape):
        """Keys as models have them: a few channels much larger than the
        others, and off centre."""
        x = self.normal(*shape)
        large = self.uniform(shape[-2], shape[-1]) < 0.03
        return x * torch.where(large, 6.0, 1.0) + self.normal(shape[-2], shape[-1])

    def parents(self, batch, nodes):
        """Trees below node 0: half of the nodes go on from the one before
        them, the rest from any before them."""
        i = torch.arange(nodes, device="cuda")
        u, chain = self.uniform(batch, nodes), self.uniform(batch, nodes) < 0.5
        any_before = torch.minimum((u * i).to(torch.int64), (i - 1).clamp_min(0))
        return torch.where(i == 0, -1, torch.where(chain, i - 1, any_before)).to(torch.int32)


def _codes(x):
    """Codes 0 .. 15, steps and least values (float16) of x ``[..., D]``, in
    groups of 32 channels; the numbers in float64, since a value next to a
    code's border would go one way in one order of sums and one in another."""
    x = x.double().unflatten(-1, (-1, GROUP))
    least = x.amin(-1).clamp(-65504.0, 65504.0).float().half()
    step = ((x.amax(-1) - least.double()) / 15.0).clamp(0.0, 65504.0).float().half()
    wide = step.double()[..., None]
    code = torch.round((x - least.double()[..., None]) / torch.where(wide == 0.0, 1.0, wide))
    code = torch.where(wide == 0.0, 0.0, code).clamp(0.0, 15.0)
    return code.to(torch.uint8).flatten(-2), step, least


def _packed(x):
    """``(bytes [..., D / 2], steps, least values)``: two channels a byte, the
    even one in the low half."""
    code, step, least = _codes(x)
    return code[..., 0::2] | (code[..., 1::2] << 4), step, least


def _pool(pages, page, heads, dim):
    """An empty pool of codes ``[pages, heads, page, D / 2]`` and scales
    ``[pages, heads, 2, D / 32, page]`` (steps, then least values)."""
    return (torch.zeros((pages, heads, page, dim // 2), dtype=torch.uint8, device="cuda"),
            torch.zeros((pages, heads, 2, dim // GROUP, page), dtype=torch.float16,
                        device="cuda"))


def _filled(x):
    """The pool of rows ``x [pages, page, heads, D]``."""
    data, step, least = _packed(x.transpose(1, 2))
    scales = torch.stack([step, least], 2).transpose(3, 4)
    return data.contiguous(), scales.contiguous()


def _put(pool, slots, x):
    """Rows ``x [T, heads, D]`` into their places of a pool."""
    codes, scales = pool
    page = codes.shape[2]
    at, row = slots.long() // page, slots.long() % page
    data, step, least = _packed(x)
    codes[at, :, row] = data
    scales[at, :, 0, :, row] = step
    scales[at, :, 1, :, row] = least


def _numbers(codes, step, least):
    """float32 numbers ``[..., D]`` of bytes ``[..., D / 2]``."""
    code = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).float()
    wide, low = (x.float().repeat_interleave(GROUP, -1) for x in (step, least))
    return code * wide + low


def _get(pool, slots):
    codes, scales = pool
    page = codes.shape[2]
    at, row = slots.long() // page, slots.long() % page
    return _numbers(codes[at, :, row], scales[at, :, 0, :, row], scales[at, :, 1, :, row])


def prepare(case, seed):
    """What the caller holds before the call."""
    c, d = case, _Draw(seed)
    kind = c["kind"]
    s = {"case": c}
    if kind in ("rotary", "store"):
        dt, tokens, dim = DTYPES[c["dtype"]], c["tokens"], c["dim"]
        s["q"] = d.normal(tokens, c["q_heads"], dim, dtype=dt)
        s["k"] = d.keys(tokens, c["kv_heads"], dim).to(dt)
        s["v"] = d.normal(tokens, c["kv_heads"], dim, dtype=dt)
        pages = (tokens + c["page"] - 1) // c["page"] + 1
        if kind == "store":
            s["kp"], s["vp"] = (_pool(pages, c["page"], c["kv_heads"], dim) for _ in range(2))
        else:
            shape = (pages, c["page"], c["kv_heads"], dim)
            s["kp"], s["vp"] = (torch.zeros(shape, dtype=dt, device="cuda") for _ in range(2))
        # pages in any order, rows of a page side by side
        at = torch.arange(tokens, device="cuda")
        order = d.order(pages)
        s["slots"] = (order[at // c["page"]] * c["page"] + at % c["page"]).to(torch.int32)
        s["positions"] = (d.integers(0, 30000, 1) + at).to(torch.int32)
    elif kind == "rows":
        pages = (c["tokens"] + c["page"] - 1) // c["page"] + 1
        shape = (pages, c["page"], c["kv_heads"], c["dim"])
        s["kp"], s["vp"] = _filled(d.keys(*shape)), _filled(d.normal(*shape))
        at = torch.arange(c["tokens"], device="cuda")
        s["slots"] = (d.order(pages)[at // c["page"]] * c["page"] + at % c["page"]).to(torch.int32)
    elif kind == "attend":
        dt, batch, nodes = DTYPES[c["dtype"]], c["batch"], c["nodes"]
        s["q"] = d.normal(batch, nodes, c["q_heads"], c["dim"], dtype=dt)
        per = (c["length"] + c["page"] - 1) // c["page"]
        s["table"] = d.order(batch * per).reshape(batch, per).contiguous()
        shape = (batch * per, c["page"], c["kv_heads"], c["dim"])
        s["kp"], s["vp"] = _filled(d.keys(*shape)), _filled(d.normal(*shape))
        s["gate"] = d.normal(batch, nodes, c["q_heads"], c["dim"], dtype=dt) if c["gate"] else None
        most = c["length"] - nodes
        s["lens"] = d.integers(most // 8 if batch > 4 else most, most, batch)
        s["counts"] = d.integers((nodes + 1) // 2, nodes, batch)
    elif kind == "verify":
        dt, batch, nodes, vocab = DTYPES[c["dtype"]], c["batch"], c["nodes"], c["vocab"]
        logits = d.normal(batch, nodes, vocab) * 3.0
        s["target"] = torch.softmax(logits, -1).to(dt)
        s["parents"] = d.parents(batch, nodes) if c["tree"] else None
        up = _parents(s)
        if c["draft"]:  # a smaller model, which has the target's view but for some noise
            s["draft"] = torch.softmax(logits + 0.7 * d.normal(batch, nodes, vocab), -1).to(dt)
            rows = s["draft"].float().gather(
                1, up.clamp_min(0)[:, :, None].expand(-1, -1, vocab)).flatten(0, 1)
            s["tokens"] = torch.multinomial(rows, 1, generator=d.gen).reshape(batch, nodes)
        else:  # the likeliest tokens behind a node, one for each of its children
            s["draft"] = None
            best = s["target"].float().topk(min(8, vocab), -1).indices
            before = (up[:, :, None] == up[:, None, :]).tril(-1).sum(-1) % best.shape[-1]
            s["tokens"] = best.gather(1, up.clamp_min(0)[:, :, None].expand(-1, -1, best.shape[-1])
                                      ).gather(2, before[:, :, None])[:, :, 0]
        s["tokens"] = s["tokens"].to(torch.int32).contiguous()
        s["uniforms"] = d.uniform(batch, nodes)
        s["counts"] = d.integers((nodes + 1) // 2, nodes, batch)
    else:
        raise ValueError("unknown kind " + kind)
    return s


# ------------------------------------------------------------------ plain forms


def _turned(x, positions, rotary, style):
    """x ``[T, heads, D]`` with its first ``rotary`` channels turned, in
    float64: neighbours ("norm"), or channels half of them apart ("neox")."""
    x = x.double()
    p = torch.arange(rotary // 2, device=x.device)
    angle = positions.double()[:, None] * ROPE_BASE ** (-2.0 * p.double() / rotary)
    cos, sin = angle.cos()[:, None], angle.sin()[:, None]
    if style == "norm":
        a, b = x[..., 0:rotary:2], x[..., 1:rotary:2]
        turned = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    else:
        a, b = x[..., :rotary // 2], x[..., rotary // 2:rotary]
        turned = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    return torch.cat([turned, x[..., rotary:]], -1)


def _rotary(s, c):
    q, k = (_turned(s[x], s["positions"], c["rotary"], c["style"]) for x in ("q", "k"))
    s["kp"].flatten(0, 1)[s["slots"].long()] = k.to(s["kp"].dtype)
    s["vp"].flatten(0, 1)[s["slots"].long()] = s["v"]
    return q.to(s["q"].dtype), s["kp"], s["vp"]


def _store(s, c):
    q, k = (_turned(s[x], s["positions"], c["rotary"], c["style"]) for x in ("q", "k"))
    _put(s["kp"], s["slots"], k)
    _put(s["vp"], s["slots"], s["v"])
    return q.to(s["q"].dtype), _get(s["kp"], s["slots"]), _get(s["vp"], s["slots"])


def _rows(s, c):
    return tuple(_get(s[x], s["slots"]).to(DTYPES[c["dtype"]]) for x in ("kp", "vp"))


def _stored(pool, table, length):
    """``[B, heads, length, D]`` of the sequences of a block table."""
    codes, scales = (x[table.long()] for x in pool)
    step, least = scales.unbind(3)
    x = _numbers(codes, step.transpose(-1, -2), least.transpose(-1, -2))
    return x.transpose(1, 2).flatten(2, 3)[:, :, :length]


def _attend(s, c):
    q = s["q"].float()
    batch, nodes, q_heads, dim = q.shape
    length, kv_heads = c["length"], c["kv_heads"]
    k = _stored(s["kp"], s["table"], length).transpose(2, 3).contiguous()
    v = _stored(s["vp"], s["table"], length).contiguous()
    q = q.reshape(batch, nodes, kv_heads, -1, dim).permute(0, 2, 1, 3, 4)
    score = torch.matmul(q.reshape(batch, kv_heads, -1, dim), k) / math.sqrt(dim)
    score = score.reshape(batch, kv_heads, nodes, -1, length)
    node = torch.arange(nodes, device=q.device)
    seen = torch.arange(length, device=q.device) <= (s["lens"][:, None] + node)[:, :, None]
    seen = seen & (node < s["counts"][:, None])[:, :, None]
    score = score.masked_fill(~seen[:, None, :, None, :], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.reshape(batch, kv_heads, -1, length), v)
    out = out.reshape(batch, kv_heads, nodes, -1, dim) / torch.where(total == 0.0, 1.0, total)
    out = out.permute(0, 2, 1, 3, 4).reshape(batch, nodes, q_heads, dim)
    if s["gate"] is not None:
        out = out / (1.0 + torch.exp(-s["gate"].float()))
    return out.to(s["q"].dtype)


def _parents(s):
    """Parents in int64; a chain's where none are given."""
    if s["parents"] is not None:
        return s["parents"].long()
    batch, nodes, _ = s["target"].shape
    return (torch.arange(nodes, device="cuda") - 1).expand(batch, nodes)


def _accepted_at_once(s, up):
    """Which nodes stand ``[B, N]``, where each one's own numbers decide:
    single children, and drafts without a distribution."""
    batch, nodes, _ = s["target"].shape
    b = torch.arange(batch, device=up.device)[:, None]
    i = torch.arange(nodes, device=up.device)
    token, row = s["tokens"].long(), up.clamp_min(0)
    p = s["target"][b, row, token].double()
    if s["draft"] is not None:
        fine = s["uniforms"].double() * s["draft"][b, row, token].double() < p
    else:
        brother = (up[:, :, None] == up[:, None, :]) & (i[None, :] < i[:, None])
        same = brother & (token[:, :, None] == token[:, None, :])
        first = ~same.any(-1)  # a token that was refused once weighs nothing
        gone = (brother & first[:, None, :]).double() @ p[:, :, None]
        fine = first & (s["uniforms"].double() * (1.0 - gone[:, :, 0]) < p)
        fine = fine & (i > 0)
        fine = fine & ~(brother & fine[:, None, :]).any(-1)
    good = torch.where(i == 0, True, fine) & (i < s["counts"][:, None])
    # all ancestors too: each doubling looks twice as far up
    for _ in range(max(1, nodes - 1).bit_length()):
        good, up = (good & torch.where(up >= 0, good.gather(1, up.clamp_min(0)), True),
                    torch.where(up >= 0, up.gather(1, up.clamp_min(0)), -1))
    return good


def _weights_behind(s, up, last):
    """What is left of the target's row behind node ``last [B]``, whose
    children were all refused."""
    batch, nodes, vocab = s["target"].shape
    b = torch.arange(batch, device=up.device)
    p = s["target"][b, last].double()
    child = (up == last[:, None]) & (torch.arange(nodes, device=up.device) < s["counts"][:, None])
    if s["draft"] is not None:
        left = (p - s["draft"][b, last].double()).clamp_min(0.0)
        return torch.where(child.any(1)[:, None], left, p), p
    out = torch.zeros_like(p).scatter_add_(1, s["tokens"].long(), child.double())
    return torch.where(out > 0.0, 0.0, p), p


def _accepted_in_turn(s, up):
    """The same two for trees of drawn drafts: every refusal leaves the next
    brother what the target has over the draft."""
    batch, nodes, vocab = s["target"].shape
    b = torch.arange(batch, device=up.device)
    last = torch.zeros(batch, dtype=torch.int64, device=up.device)
    p = s["target"][b, last].double()
    left, total = p, torch.ones(batch, dtype=torch.float64, device=up.device)
    good = [s["counts"] > 0]
    for i in range(1, nodes):
        mine = (up[:, i] == last) & (i < s["counts"])
        token, q = s["tokens"][:, i].long(), s["draft"][b, last].double()
        fine = s["uniforms"][:, i].double() * q[b, token] * total < left[b, token]
        good.append(mine & fine)
        last = torch.where(mine & fine, i, last)
        less = (left - total[:, None] * q).clamp_min(0.0)
        p = s["target"][b, last].double()
        left = torch.where((mine & ~fine)[:, None], less,
                           torch.where((mine & fine)[:, None], p, left))
        total = torch.where(mine & ~fine, less.sum(1), torch.where(mine & fine, 1.0, total))
    return torch.stack(good, 1), left, p


def _verify(s, c):
    batch, nodes, vocab = s["target"].shape
    up = _parents(s)
    i = torch.arange(nodes, device=up.device)
    if c["tree"] and c["draft"]:
        good, left, p = _accepted_in_turn(s, up)
    else:
        good = _accepted_at_once(s, up)
        left, p = _weights_behind(s, up, (good * i).amax(1))
    left = torch.where(left.sum(1, keepdim=True) > 0.0, left, p)
    sums = left.cumsum(1)
    place = (sums <= s["uniforms"][:, :1].double() * sums[:, -1:]).sum(1)
    last_one = ((left > 0.0) * torch.arange(vocab, device=up.device)).amax(1)
    token = torch.minimum(place, last_one)
    accepted = good.sum(1)
    # the nodes of the path in order, then the tokens behind each of them
    paths = torch.where(good, i, nodes).sort(1).values
    inside = i < accepted[:, None]
    behind = torch.nn.functional.pad(paths, (0, 1), value=nodes)[:, 1:].clamp_max(nodes - 1)
    tokens = torch.where(i + 1 < accepted[:, None], s["tokens"].long().gather(1, behind),
                         token[:, None])
    return tuple(x.to(torch.int32) for x in (torch.where(inside, paths, -1), accepted,
                                             torch.where(inside, tokens, -1)))


def run(state):
    """One pass through an operator; a pass of ``store`` reads its rows back."""
    s, c = state, state["case"]
    kind = c["kind"]
    if not own:
        return {"rotary": _rotary, "store": _store, "rows": _rows, "attend": _attend,
                "verify": _verify}[kind](s, c)
    ops = _ops()
    if kind == "rotary":
        q = ops.paged_rotary_append_rows_(
            s["q"], s["k"], s["v"], s["kp"], s["vp"], s["slots"], s["positions"],
            rotary_dimension=c["rotary"], frequency_base=ROPE_BASE, style=c["style"])
        return q, s["kp"], s["vp"]
    if kind == "verify":
        r = ops.verify_drafts(s["tokens"], s["target"], s["uniforms"], parents=s["parents"],
                              draft=s["draft"], counts=s["counts"])
        return r.paths, r.accepted, r.tokens
    pool = (*s["kp"], *s["vp"])
    if kind == "store":
        q = ops.paged_q4_append_rows_(
            s["q"], s["k"], s["v"], *pool, s["slots"], s["positions"],
            rotary_dimension=c["rotary"], frequency_base=ROPE_BASE, style=c["style"])
        return (q, *ops.paged_q4_rows(*pool, s["slots"]))
    if kind == "rows":
        return ops.paged_q4_rows(*pool, s["slots"], dtype=DTYPES[c["dtype"]])
    return ops.paged_q4_attention(s["q"], *pool, s["table"], length=c["length"],
                                  prefix_lens=s["lens"], counts=s["counts"], gate=s["gate"])


# ------------------------------------------------------------------ work


def _row_bytes(dim):
    """Codes and scales of one row of one head."""
    return dim // 2 + 4 * (dim // GROUP)


def work(case):
    c, kind = case, case["kind"]
    if kind in ("rotary", "store"):
        es, tokens, dim = BYTES[c["dtype"]], c["tokens"], c["dim"]
        read = es * tokens * dim * (c["q_heads"] + 2 * c["kv_heads"]) + 8 * tokens
        wrote = es * tokens * dim * c["q_heads"]
        rows = 2 * tokens * c["kv_heads"]
        if kind == "rotary":
            wrote += es * rows * dim
        else:  # written, read back, and given as float32
            wrote += rows * (2 * _row_bytes(dim) + 4 * dim)
        return {"bytes": read + wrote,
                "flops": tokens * (3 * c["rotary"] * (c["q_heads"] + c["kv_heads"])
                                   + (10 * c["kv_heads"] * dim if kind == "store" else 0))}
    if kind == "rows":
        rows = 2 * c["tokens"] * c["kv_heads"]
        return {"bytes": rows * (_row_bytes(c["dim"]) + BYTES[c["dtype"]] * c["dim"])
                + 4 * c["tokens"], "flops": 2 * rows * c["dim"]}
    if kind == "attend":
        nodes, most = c["nodes"], c["length"] - c["nodes"]
        low = most // 8 if c["batch"] > 4 else most
        live = ((nodes + 1) // 2 + nodes) / 2  # mean of the drawn counts
        rows = c["batch"] * ((low + most) / 2 + live)
        heads = c["batch"] * nodes * c["q_heads"] * c["dim"] * BYTES[c["dtype"]]
        return {"bytes": int(2 * rows * c["kv_heads"] * _row_bytes(c["dim"])
                             + heads * (3 if c["gate"] else 2)),
                "flops": int(4 * c["dim"] * c["q_heads"] * live * rows)}
    # the rows that the last token is drawn from, and each draft's own entries
    rows, es = c["batch"] * (2 if c["draft"] else 1), BYTES[c["dtype"]]
    nodes = c["batch"] * c["nodes"]
    return {"bytes": rows * c["vocab"] * es + nodes * (2 * es + 20),
            "flops": 3 * rows * c["vocab"]}


# ------------------------------------------------------------------ exact


def _exact_turn(x, s, c):
    """The definition, pair by pair."""
    x, half = x.double(), c["rotary"] // 2
    out = x.clone()
    for p in range(half):
        angle = (s["positions"].double() * ROPE_BASE ** (-p / half))[:, None]
        first, second = (2 * p, 2 * p + 1) if c["style"] == "norm" else (p, p + half)
        a, b = x[..., first], x[..., second]
        out[..., first] = a * angle.cos() - b * angle.sin()
        out[..., second] = b * angle.cos() + a * angle.sin()
    return out


def _exact_stored(x):
    """What 4-bit rows of x stand for, group by group."""
    out = torch.empty_like(x)
    for g in range(0, x.shape[-1], GROUP):
        part = x[..., g:g + GROUP]
        low = part.min(-1, keepdim=True).values.float().half().double()
        step = ((part.max(-1, keepdim=True).values - low) / 15).clamp_min(0).float().half().double()
        code = torch.nan_to_num((part - low) / step, nan=0.0, posinf=0.0, neginf=0.0)
        out[..., g:g + GROUP] = low + step * code.round().clamp(0, 15)
    return out


def _exact_rows(pool, slots):
    codes, scales = pool
    page = codes.shape[2]
    at, row = slots.long() // page, slots.long() % page
    out = torch.empty((slots.numel(), codes.shape[1], 2 * codes.shape[3]), dtype=torch.float64,
                      device="cuda")
    for odd in (0, 1):
        half = codes[at, :, row].long().div(16 if odd else 1, rounding_mode="floor") % 16
        out[..., odd::2] = half.double()
    for g in range(scales.shape[3]):
        part = out[..., GROUP * g:GROUP * (g + 1)]
        part *= scales[at, :, 0, g, row].double()[..., None]
        part += scales[at, :, 1, g, row].double()[..., None]
    return out


def _exact_attend(s, c):
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    group = c["q_heads"] // c["kv_heads"]
    for b in range(c["batch"]):
        prefix, count = int(s["lens"][b]), int(s["counts"][b])
        at = torch.arange(prefix + count, device="cuda")
        slots = s["table"][b].long()[at // c["page"]] * c["page"] + at % c["page"]
        k, v = _exact_rows(s["kp"], slots), _exact_rows(s["vp"], slots)
        hidden = at[None, :] > prefix + torch.arange(count, device="cuda")[:, None]
        for h in range(c["kv_heads"]):
            q = s["q"][b, :count, h * group:(h + 1) * group].double()
            score = torch.einsum("ngd,jd->ngj", q, k[:, h]) * c["dim"] ** -0.5
            score = score.masked_fill(hidden[:, None, :], -math.inf)
            out[b, :count, h * group:(h + 1) * group] = torch.einsum(
                "ngj,jd->ngd", torch.softmax(score, -1), v[:, h])
    return out if s["gate"] is None else out * torch.sigmoid(s["gate"].double())


def exact(case, seed):
    """``run``'s outputs in float64; a verification gives whole numbers."""
    c = case
    if c["kind"] == "verify":
        return None
    s = prepare(case, seed)
    if c["kind"] == "attend":
        return _exact_attend(s, c)
    if c["kind"] == "rows":
        return _exact_rows(s["kp"], s["slots"]), _exact_rows(s["vp"], s["slots"])
    q, k = _exact_turn(s["q"], s, c), _exact_turn(s["k"], s, c)
    if c["kind"] == "store":
        return q, _exact_stored(k), _exact_stored(s["v"].double())
    kp, vp = s["kp"].double(), s["vp"].double()
    for pages, rows in ((kp, k), (vp, s["v"].double())):
        pages.view(-1, c["kv_heads"], c["dim"]).index_copy_(0, s["slots"].long(), rows)
    return q, kp, vp
