"""What the decode operators over a paged KV cache are measured on: the plan of a pass (block tables, slots, positions, tree masks), rotary
positions, the cache write, and attention of new tokens (one token, a tree of drafts, a piece of a prompt) over the pages.

`run` computes an operator from elementary torch operations in 32 bits, or, with `own`, calls this repository's kernels for it.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "bf16": 2}


# ---------------------------------------------------------------------------------------------------------------- the cases

def listed():
    return [
        # a server's quiet moment: four requests, each with a small tree of drafts, pages of 16
        dict(name="plan, 4 small trees", op="plan", batch=4, cached=2000, new=12, page=16, tree=True),
        # a full batch taking in prompts: 256 requests with up to 4096 new tokens each, slots for over half a million tokens
        dict(name="plan, 256 prompts", op="plan", batch=256, cached=4096, new=4096, page=64, tree=False),
        # one decode step of the 124M model's 12 x 64 heads (q and k together), eight requests
        dict(name="rope, decode step", op="rope", back=False, tokens=8, heads=24, dim=64, rotary=64, layout="half", scaling="none", factor=1.0, far=1024, dtype="bf16"),
        # a long prompt in one piece, neighbouring pairs, half of each head rotated, a context stretched eightfold
        dict(name="rope, long prompt", op="rope", back=False, tokens=32768, heads=40, dim=128, rotary=64, layout="interleaved", scaling="by_turns", factor=8.0, far=131072, dtype="bf16"),
        # the gradient of the training step's batch of 32 x 1024 tokens in the f32 tier
        dict(name="rope, gradient", op="rope", back=True, tokens=32767, heads=24, dim=64, rotary=64, layout="half", scaling="linear", factor=4.0, far=4096, dtype="f32"),
        # one decode step of 61 requests: new keys rotated on the way into bf16 pages
        dict(name="write, decode step", op="write", tokens=61, heads=8, dim=128, page=16, src="bf16", dst="bf16", rotate=True, far=32768),
        # 16384 prompt tokens of the 24-layer configuration's 16 x 128 heads, from the f32 tier's activations into bf16 pages
        dict(name="write, prompt", op="write", tokens=16384, heads=16, dim=128, page=64, src="f32", dst="bf16", rotate=True, far=4096),
        # the smallest call: one token of one request, the 124M model's heads in the f32 tier
        dict(name="attention, one token f32", op="attention", batch=1, cached=776, new=1, heads=12, kv_heads=12, dim=64, page=16, tree=False, window=0, dtype="f32"),
        # a decode step of a ragged batch, four query heads to a KV head
        dict(name="attention, decode batch", op="attention", batch=64, cached=8191, new=1, heads=32, kv_heads=8, dim=128, page=16, tree=False, window=0, dtype="bf16"),
        # five drafts over one long context: the cache of 131 thousand tokens is all the work there is
        dict(name="attention, long context", op="attention", batch=1, cached=131071, new=5, heads=32, kv_heads=8, dim=128, page=64, tree=True, window=0, dtype="bf16"),
        # trees of up to 63 drafts, the 24-layer configuration's 16 x 128 heads
        dict(name="attention, trees of 63", op="attention", batch=8, cached=4095, new=63, heads=16, kv_heads=16, dim=128, page=32, tree=True, window=0, dtype="bf16"),
        # wide trees over many shared heads: the arithmetic counts here
        dict(name="attention, wide trees", op="attention", batch=16, cached=8000, new=128, heads=32, kv_heads=4, dim=128, page=64, tree=True, window=0, dtype="bf16"),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw(rng):
    op = rng.choice(["plan", "rope", "write", "attention", "attention"])
    if op == "plan":
        tree = rng.random() < 0.6
        return dict(op=op, batch=_spread(rng, 1, 512), cached=_spread(rng, 1, 32768), new=_spread(rng, 1, 128 if tree else 4096), page=rng.choice([1, 8, 16, 20, 32, 64, 128]), tree=tree)
    if op == "rope":
        dim = rng.choice([32, 64, 80, 96, 128, 256])
        rotary = rng.choice([dim, dim, dim // 2, dim // 4])
        scaling = rng.choice(["none", "linear", "base", "by_turns"])
        return dict(op=op, back=rng.random() < 0.4, tokens=_spread(rng, 1, 32768), heads=rng.choice([1, 3, 8, 24, 32, 40]), dim=dim, rotary=rotary,
                    layout=rng.choice(["half", "interleaved"]), scaling=scaling, factor=1.0 if scaling == "none" else rng.choice([2.0, 4.0, 8.0, 40.0]), far=_spread(rng, 16, 1 << 20),
                    dtype=rng.choice(["f32", "bf16"]))
    if op == "write":
        src = rng.choice(["f32", "bf16"])
        return dict(op=op, tokens=_spread(rng, 1, 16384), heads=rng.choice([1, 4, 8, 12, 16]), dim=rng.choice([64, 80, 96, 128]), page=rng.choice([1, 8, 16, 20, 32, 64, 128]), src=src,
                    dst=src if src == "bf16" else rng.choice(["f32", "bf16"]), rotate=rng.random() < 0.6, far=_spread(rng, 16, 1 << 20))
    heads, kv_heads = rng.choice([(12, 12), (16, 16), (32, 8), (32, 4), (16, 2), (8, 1), (12, 4)])
    new = rng.choice([1, 1, _spread(rng, 2, 128), _spread(rng, 2, 512)])
    return dict(op=op, batch=_spread(rng, 1, 128), cached=_spread(rng, 1, 131072), new=new, heads=heads, kv_heads=kv_heads, dim=rng.choice([64, 64, 128, 128, 96]),
                page=rng.choice([8, 16, 20, 32, 64, 128]), tree=1 < new <= 128 and rng.random() < 0.7, window=0 if rng.random() < 0.8 else _spread(rng, 16, 8192),
                dtype=rng.choice(["bf16", "bf16", "bf16", "f32"]))


def _load(case):
    """What bounds a case's cost here: its bytes and, at the plain form's rate, its operations; the plain form pads every request to the longest."""
    w = work(case)
    flops = w["flops"] * (6 if case.get("dtype") == "f32" and case["op"] == "attention" else 1)
    padded = 0
    if case["op"] == "attention":
        padded = case["batch"] * (case["cached"] + case["new"]) * (4 * case["kv_heads"] * case["dim"] + 2 * case["heads"] * case["new"])
    return w["bytes"], flops, padded


def draw(rng):
    most = {}
    for c in listed():
        for k, v in enumerate(_load(c)):
            most[c["op"], k] = max(most.get((c["op"], k), 0), v)
    while True:
        case = _draw(rng)
        if all(v <= most[case["op"], k] for k, v in enumerate(_load(case))):
            return case


def _lengths(case):
    """(cached, new) tokens of every request: the same for every seed, so that a case's work is known; the first is the longest."""
    g = np.random.RandomState((case["batch"] * 1009 + case["cached"] * 31 + case["new"]) % (1 << 31))
    cached = g.randint(case["cached"] // 4, case["cached"] + 1, case["batch"])
    new = g.randint(0 if case["op"] == "plan" else (case["new"] + 1) // 2, case["new"] + 1, case["batch"])
    cached[0], new[0] = case["cached"], case["new"]
    return cached.astype(np.int64), new.astype(np.int64)


def _words(case):
    return (case["new"] + 31) // 32


def work(case):
    if case["op"] == "plan":
        cached, new = _lengths(case)
        pages = (cached + new + case["page"] - 1) // case["page"] - (cached + case["page"] - 1) // case["page"]
        tokens = int(new.sum())
        # lengths in, row starts out, fresh pages read and entered, a slot and a position per token; parents in and ancestor bits out for trees
        return {"bytes": 12 * case["batch"] + 8 * int(pages.sum()) + 8 * tokens + (tokens * 4 * (1 + _words(case)) if case["tree"] else 0), "flops": 0}
    if case["op"] == "rope":
        n = case["tokens"] * case["heads"] * case["dim"]
        return {"bytes": 2 * n * SIZE[case["dtype"]] + 4 * case["tokens"], "flops": 3 * case["tokens"] * case["heads"] * case["rotary"]}
    if case["op"] == "write":
        n = case["tokens"] * case["heads"] * case["dim"]
        return {"bytes": 2 * n * (SIZE[case["src"]] + SIZE[case["dst"]]) + 8 * case["tokens"], "flops": 3 * n if case["rotate"] else 0}
    cached, new = _lengths(case)
    size, h, hk, d = SIZE[case["dtype"]], case["heads"], case["kv_heads"], case["dim"]
    # cached positions that some new token of the request sees: all of them, or the window of the first token on
    past = np.minimum(cached, case["window"] - 1) if case["window"] else cached
    reads = int((past + new).sum()) * 2 * hk * d * size
    tokens = int(new.sum())
    # per query head and token: two products of length d with every cached position in sight, and with the new tokens up to itself
    # (for a tree fewer of those count, but few against the cache)
    ahead = new * (new + 1) // 2
    if case["window"]:
        w = case["window"]
        reach = np.minimum(new, w)
        ahead = reach * (reach + 1) // 2 + (new - reach) * w
        t = np.minimum(new, w)  # token i sees min(cached, w - 1 - i) cached positions
        past_seen = np.array([int(np.minimum(c, np.maximum(0, w - 1 - np.arange(n))).sum()) for c, n in zip(cached, t)])
    else:
        past_seen = cached * new
    return {"bytes": reads + tokens * h * (2 * d * size + 4), "flops": 4 * d * h * int((past_seen + ahead).sum())}


# ---------------------------------------------------------------------------------------------------------------- the inputs

_open = {}


def _backend():
    """The program's one backend handle."""
    if "be" not in _open:
        from ojas_b200 import CudaBackend
        _open["be"] = CudaBackend(0, 64 << 30)
    return _open["be"]


def _t(x):
    """The framework's descriptor of a torch tensor's memory."""
    from ojas_b200 import DType, Tensor
    kind = {torch.float32: DType.F32, torch.bfloat16: DType.BF16, torch.int32: DType.U32}[x.dtype]
    return Tensor(_backend(), x.data_ptr(), tuple(x.shape), kind, tuple(x.stride()), owner=x)


def _ints(a):
    return torch.from_numpy(np.ascontiguousarray(a).astype(np.int64).astype(np.uint32).view(np.int32)).cuda()


def _trees(new, seed):
    """Parent of every draft within its request (-1: the last cached token): a few candidates at every depth."""
    g = np.random.RandomState(seed % (1 << 31))
    local = np.concatenate([np.arange(n) for n in new]) if len(new) else np.zeros(0, np.int64)
    return np.maximum(local - 1 - g.randint(0, 4, len(local)), -1), local


def _ancestors(parents, local, starts_of, words):
    """Bit j of row i: draft j is i or one of its ancestors; and every draft's depth."""
    n = len(local)
    bits, at, depth = np.zeros((n, words), np.uint32), local.copy(), np.zeros(n, np.int64)
    rows = np.arange(n)
    while len(rows):
        bits[rows, at[rows] // 32] |= (np.uint32(1) << (at[rows] % 32).astype(np.uint32))
        at[rows] = parents[starts_of[rows] + at[rows]]
        rows = rows[at[rows] >= 0]
        depth[rows] += 1
    return bits, depth


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    state = {"case": case}
    if case["op"] == "rope":
        n, h, d = case["tokens"], case["heads"], case["dim"]
        # q and k are the first heads of a fused projection's rows, v follows them; a gradient comes as a tensor of its own
        wide = h if case["back"] else h + max(1, h // 4)
        rows = torch.randn(n, wide, d, device="cuda", generator=g).to(DTYPES[case["dtype"]])
        state["x"] = rows[:, :h]
        state["positions"] = torch.randint(0, case["far"], (n,), device="cuda", generator=g, dtype=torch.int32)
        state["y"] = torch.empty(n, h, d, device="cuda", dtype=rows.dtype)
        state["turns"] = torch.from_numpy(_frequencies(case["rotary"], case["scaling"], case["factor"], 4096)).cuda()
        if own:
            from ojas_b200 import RopeSpec
            be = _backend()
            state["rope"] = be.rope_plan(RopeSpec(case["rotary"], layout=case["layout"], scaling=case["scaling"], factor=case["factor"], original_length=4096, amplitude=_amplitude(case)))
            state["t"] = {k: _t(state[k]) for k in ("x", "positions", "y")}
    elif case["op"] == "write":
        n, h, d, page = case["tokens"], case["heads"], case["dim"], case["page"]
        rows = torch.randn(n, 2 * h, d, device="cuda", generator=g).to(DTYPES[case["src"]])
        state["k"], state["v"] = rows[:, :h], rows[:, h:]
        pages = (n + page - 1) // page + 9
        order = torch.randperm(pages, device="cuda", generator=g)
        at = torch.arange(n, device="cuda") + seed % page
        state["slots"] = (order[at // page] * page + at % page).to(torch.int32)
        state["positions"] = torch.randint(0, case["far"], (n,), device="cuda", generator=g, dtype=torch.int32)
        state["k_pages"] = torch.randn(pages, page, h, d, device="cuda", generator=g).to(DTYPES[case["dst"]])
        state["v_pages"] = torch.randn(pages, page, h, d, device="cuda", generator=g).to(DTYPES[case["dst"]])
        state["turns"] = torch.from_numpy(_frequencies(d, "none", 1.0, 4096)).cuda()
        if own:
            from ojas_b200 import RopeSpec
            state["rope"] = _backend().rope_plan(RopeSpec(d)) if case["rotate"] else None
            state["t"] = {k: _t(state[k]) for k in ("k_pages", "v_pages", "k", "v", "slots", "positions")}
    else:
        cached, new = _lengths(case)
        order = np.random.RandomState(seed % (1 << 31)).permutation(case["batch"])
        cached, new = cached[order], new[order]
        page, batch, tokens = case["page"], case["batch"], int(new.sum())
        starts = np.concatenate([[0], np.cumsum(new)])
        held, total = (cached + page - 1) // page, (cached + new + page - 1) // page
        width = int(total.max()) + 2
        pool = int(total.sum()) + 7
        free = np.random.RandomState((seed + 1) % (1 << 31)).permutation(pool)
        entered = held if case["op"] == "plan" else total
        tables = np.full((batch, width), -1, np.int64)
        first = np.cumsum(entered) - entered
        col = np.arange(width)[None, :]
        inside = col < entered[:, None]
        tables[inside] = free[(first[:, None] + col)[inside]]
        state["cached"], state["tables"] = _ints(cached), _ints(tables)
        state["longest"], state["tokens"] = int((cached + new).max()), tokens
        parents, local = _trees(new, seed)
        bits, depth = (None, local) if not case["tree"] else _ancestors(parents, local, np.repeat(starts[:-1], new), _words(case))
        if case["op"] == "plan":
            state["new"] = _ints(new)
            state["free"], state["head"] = _ints(np.concatenate([free[:3], free[int(entered.sum()):]])), _ints([3])
            state["parents"] = _ints(parents) if case["tree"] else None
            out = dict(starts=batch + 1, slots=tokens, positions=tokens, taken=1)
            state["out"] = {k: torch.empty(v, device="cuda", dtype=torch.int32) for k, v in out.items()}
            state["out"]["masks"] = torch.empty(tokens, _words(case), device="cuda", dtype=torch.int32) if case["tree"] else None
            if own:
                state["t"] = {k: _t(state[k]) if state[k] is not None else None for k in ("cached", "new", "free", "head", "tables", "parents")}
                state["t"].update({"out_" + k: _t(v) if v is not None else None for k, v in state["out"].items()})
        else:
            kind, h, hk, d = DTYPES[case["dtype"]], case["heads"], case["kv_heads"], case["dim"]
            state["starts"] = _ints(starts)
            state["positions"] = _ints(np.repeat(cached, new) + depth)
            state["masks"] = _ints(bits) if case["tree"] else None
            # keys and queries as a norm over the head leaves them, queries with some weight: rows attend to few keys, as they do in use
            state["q"] = (2 * torch.randn(tokens, h, d, device="cuda", generator=g)).to(kind)
            state["k_pages"] = torch.randn(pool, page, hk, d, device="cuda", generator=g, dtype=torch.float32).to(kind)
            state["v_pages"] = torch.randn(pool, page, hk, d, device="cuda", generator=g, dtype=torch.float32).to(kind)
            state["out"], state["lse"] = torch.empty_like(state["q"]), torch.empty(tokens, h, device="cuda")
            if own:
                names = ("q", "k_pages", "v_pages", "tables", "cached", "starts", "positions", "masks", "out", "lse")
                state["t"] = {k: _t(state[k]) if state[k] is not None else None for k in names}
                state["work"] = _backend().paged_attention_workspace(state["t"]["q"], state["t"]["k_pages"])
    torch.cuda.synchronize()  # the framework's stream is its own
    return state


# ---------------------------------------------------------------------------------------------------------------- rotary frequencies

def _amplitude(case):
    return 1.0 if case["scaling"] != "by_turns" else 0.1 * math.log(case["factor"]) + 1.0


def _frequencies(rotary, scaling, factor, original):
    """Radians per position of each pair, in 64 bits."""
    i = np.arange(0, rotary, 2, dtype=np.float64)
    base = 10000.0 * factor ** (rotary / (rotary - 2)) if scaling == "base" else 10000.0
    f = base ** (-i / rotary)
    if scaling == "linear":
        return f / factor
    if scaling == "by_turns":  # pairs that turn often within the original length stay, slow ones are stretched, a ramp between
        keep = np.clip((original * f / (2 * math.pi) - 1.0) / (32.0 - 1.0), 0.0, 1.0)
        return f * keep + f / factor * (1 - keep)
    return f


def _rotate(x, positions, freqs, layout, amplitude, back):
    """x [tokens, heads, dim] with its leading pairs turned by position x frequency; the angles in 64 bits."""
    r = 2 * freqs.numel()
    angle = positions.double()[:, None] * freqs[None, :]
    cos, sin = (amplitude * angle.cos()).float()[:, None], (amplitude * angle.sin()).float()[:, None]
    sin = -sin if back else sin
    x = x.float()
    a, b = (x[..., : r // 2], x[..., r // 2 : r]) if layout == "half" else (x[..., 0:r:2], x[..., 1:r:2])
    u, v = a * cos - b * sin, b * cos + a * sin
    turned = torch.cat([u, v], -1) if layout == "half" else torch.stack([u, v], -1).flatten(-2)
    return torch.cat([turned, x[..., r:]], -1)


# ---------------------------------------------------------------------------------------------------------------- one pass

def run(state):
    return {"plan": _run_plan, "rope": _run_rope, "write": _run_write, "attention": _run_attention}[state["case"]["op"]](state)


def _run_plan(state):
    case = state["case"]
    if own:
        t = state["t"]
        _backend().paged_plan(t["cached"], t["new"], t["free"], t["head"], t["tables"], case["page"], parents=t["parents"], starts=t["out_starts"], slots=t["out_slots"],
                              positions=t["out_positions"], masks=t["out_masks"], free_head_out=t["out_taken"])
        return dict({k: v for k, v in state["out"].items() if v is not None}, tables=state["tables"])
    page, batch, tokens = case["page"], case["batch"], state["tokens"]
    cached, new = state["cached"].long(), state["new"].long()
    ends = torch.cumsum(new, 0)
    starts = torch.cat([torch.zeros_like(ends[:1]), ends])
    held, total = (cached + page - 1) // page, (cached + new + page - 1) // page
    grown = torch.cumsum(total - held, 0)
    first = state["head"].long() + grown - (total - held)
    col = torch.arange(state["tables"].shape[1], device="cuda")[None, :]
    fresh = (col >= held[:, None]) & (col < total[:, None])
    entry = (first[:, None] + col - held[:, None]).clamp(0, state["free"].numel() - 1)
    tables = torch.where(fresh, state["free"][entry], state["tables"])
    token = torch.arange(tokens, device="cuda")
    request = torch.searchsorted(ends, token, right=True)
    local = token - starts[request]
    at = cached[request] + local
    slots = tables[request, at // page].long() * page + at % page
    out = {"starts": starts.int(), "slots": slots.int(), "taken": (state["head"].long() + grown[-1:]).int(), "tables": tables}
    if not case["tree"]:
        return dict(out, positions=at.int())
    m = case["new"]
    # ancestors: the closure of "is the parent of", by squaring
    reach = torch.zeros(batch, m, m + 1, device="cuda")
    parents = state["parents"].long()
    reach[request, local, torch.where(parents < 0, m, parents)] = 1
    reach = reach[..., :m] + torch.eye(m, device="cuda")
    for _ in range(max(1, math.ceil(math.log2(m + 1)))):
        reach = (reach @ reach > 0).float()
    reach = reach[request, local]
    bits = torch.nn.functional.pad(reach, (0, 32 * _words(case) - m)).view(tokens, -1, 32).long()
    masks = (bits << torch.arange(32, device="cuda")).sum(-1)
    return dict(out, positions=(cached[request] + reach.sum(-1).long() - 1).int(), masks=(masks - ((masks >> 31) << 32)).int())


def _run_rope(state):
    case = state["case"]
    if own:
        t, be = state["t"], _backend()
        (be.rope_backward if case["back"] else be.rope_forward)(t["x"], t["positions"], state["rope"], out=t["y"])
        return state["y"]
    return _rotate(state["x"], state["positions"], state["turns"], case["layout"], _amplitude(case), case["back"]).to(state["y"].dtype)


def _run_write(state):
    case = state["case"]
    if own:
        t = state["t"]
        _backend().paged_kv_write(t["k_pages"], t["v_pages"], t["k"], t["v"], t["slots"], rope=state["rope"], positions=t["positions"] if case["rotate"] else None)
    else:
        k = _rotate(state["k"], state["positions"], state["turns"], "half", 1.0, False) if case["rotate"] else state["k"]
        slots = state["slots"].long()
        state["k_pages"].flatten(0, 1)[slots] = k.to(state["k_pages"].dtype)
        state["v_pages"].flatten(0, 1)[slots] = state["v"].to(state["v_pages"].dtype)
    return state["k_pages"], state["v_pages"]


def _run_attention(state):
    case = state["case"]
    if own:
        t = state["t"]
        _backend().paged_attention_forward(t["q"], t["k_pages"], t["v_pages"], t["tables"], t["cached"], t["starts"], masks=t["masks"], positions=t["positions"],
                                           window=case["window"] or None, out=t["out"], lse=t["lse"], workspace=state["work"])
        return {"out": state["out"], "lse": state["lse"]}
    h, hk, d, page, batch, m, length = case["heads"], case["kv_heads"], case["dim"], case["page"], case["batch"], case["new"], state["longest"]
    cached, starts = state["cached"].long(), state["starts"].long()
    new = starts[1:] - starts[:-1]
    at = torch.arange(length, device="cuda")
    slot = state["tables"].long()[:, at // page].clamp(min=0) * page + at % page
    k = state["k_pages"].flatten(0, 1)[slot].float().permute(0, 2, 3, 1)                     # [batch, kv_heads, dim, length]
    v = state["v_pages"].flatten(0, 1)[slot].float().transpose(1, 2)                         # [batch, kv_heads, length, dim]
    i = torch.arange(m, device="cuda")
    row = (starts[:-1, None] + i).clamp(max=state["tokens"] - 1)                             # [batch, m]
    q = state["q"][row].float().view(batch, m, hk, h // hk, d).permute(0, 2, 1, 3, 4).reshape(batch, hk, m * (h // hk), d)
    draft = at[None, :] - cached[:, None]                                                    # [batch, length]
    inside = (draft >= 0) & (draft < new[:, None])
    if case["tree"]:
        j = draft.clamp(0, m - 1)
        word = state["masks"].long()[row].gather(2, (j // 32)[:, None, :].expand(batch, m, length))
        sees = inside[:, None, :] & ((word >> (j % 32)[:, None, :]) & 1 > 0)
    else:
        sees = inside[:, None, :] & (draft[:, None, :] <= i[None, :, None])
    sees = sees | (draft < 0)[:, None, :]
    if case["window"]:
        positions = state["positions"].long()
        place = torch.where(draft < 0, at[None, :].expand(batch, length), positions[(starts[:-1, None] + draft.clamp(0, m - 1)).clamp(max=state["tokens"] - 1)])
        sees = sees & (place[:, None, :] > positions[row][:, :, None] - case["window"])
    sees = sees[:, None, :, None, :].expand(batch, hk, m, h // hk, length).reshape(batch, hk, -1, length)
    s = torch.where(sees, (q @ k) * d ** -0.5, -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.where(sees, (s - top).exp(), 0.0)
    total = p.sum(-1, keepdim=True)
    o = ((p @ v) / total).view(batch, hk, m, h // hk, d).transpose(1, 2).reshape(batch, m, h, d)
    lse = (top + total.log()).view(batch, hk, m, h // hk).transpose(1, 2).reshape(batch, m, h)
    token = torch.arange(state["tokens"], device="cuda")
    request = torch.searchsorted(starts[1:].contiguous(), token, right=True)
    local = token - starts[request]
    return {"out": o[request, local].to(state["q"].dtype), "lse": lse[request, local]}


# ---------------------------------------------------------------------------------------------------------------- the definitions in 64 bits

def exact(case, seed):
    if case["op"] == "plan":
        return None
    s = prepare(case, seed)
    if case["op"] == "rope":
        return _turned(s["x"], s["positions"], s["turns"], case["layout"], _amplitude(case), -1.0 if case["back"] else 1.0)
    if case["op"] == "write":
        k = _turned(s["k"], s["positions"], s["turns"], "half", 1.0, 1.0) if case["rotate"] else s["k"].double()
        made = []
        for pages, x in ((s["k_pages"], k), (s["v_pages"], s["v"].double())):
            flat = pages.double().flatten(0, 1)
            flat.index_copy_(0, s["slots"].long(), x)
            made.append(flat.view(pages.shape))
        return tuple(made)
    return _attention_exact(case, s)


def _turned(x, positions, freqs, layout, amplitude, sign):
    """Each pair as a complex number times amplitude e^(i angle)."""
    y = x.double().clone()
    r = 2 * freqs.numel()
    first, second = (slice(0, r // 2), slice(r // 2, r)) if layout == "half" else (slice(0, r, 2), slice(1, r, 2))
    turn = torch.polar(torch.full_like(freqs, amplitude).expand(len(positions), -1), sign * positions.double()[:, None] * freqs)
    z = torch.complex(y[..., first], y[..., second]) * turn[:, None]
    y[..., first], y[..., second] = z.real, z.imag
    return y


def _attention_exact(case, s):
    h, hk, d, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    out = torch.zeros(s["tokens"], h, d, device="cuda", dtype=torch.float64)
    lse = torch.zeros(s["tokens"], h, device="cuda", dtype=torch.float64)
    cached, starts = s["cached"].tolist(), s["starts"].tolist()
    k_flat, v_flat = s["k_pages"].flatten(0, 1), s["v_pages"].flatten(0, 1)
    for b in range(case["batch"]):
        c, lo, hi = cached[b], starts[b], starts[b + 1]
        n = hi - lo
        at = torch.arange(c + n, device="cuda")
        slot = s["tables"][b].long()[at // page] * page + at % page
        sees = torch.ones(n, c + n, dtype=torch.bool, device="cuda")
        if case["tree"]:
            bits = (s["masks"][lo:hi].long()[:, :, None] >> torch.arange(32, device="cuda")) & 1
            sees[:, c:] = bits.flatten(1)[:, :n] > 0
        else:
            sees[:, c:] = torch.ones(n, n, dtype=torch.bool, device="cuda").tril()
        if case["window"]:
            mine = s["positions"][lo:hi].long()
            sees &= torch.cat([at[:c], mine])[None, :] > mine[:, None] - case["window"]
        for kv in range(hk):
            heads = slice(kv * (h // hk), (kv + 1) * (h // hk))
            k, v = k_flat[slot, kv].double(), v_flat[slot, kv].double()
            score = torch.einsum("nhd,ld->hnl", s["q"][lo:hi, heads].double(), k) / math.sqrt(d)
            score.masked_fill_(~sees, -math.inf)
            lse[lo:hi, heads] = torch.logsumexp(score, -1).T
            out[lo:hi, heads] = torch.einsum("hnl,ld->nhd", torch.softmax(score, -1), v)
    return {"out": out, "lse": lse}
