"""Performance cases of the text model's serving operators: an 8-bit key/value cache in blocks, the attention that reads
it, and linear layers with 4-bit weights.

Kinds:

- write       keys and values of new tokens go into the cache (`ops.kv_write`), and the blocks that this touched are read
              back as values (`ops.kv_read`)
- attention   queries of each sequence's newest tokens over its cached keys and values (`ops.kv_attention`): one token a
              sequence while it answers, many while a prompt (or the rest of one behind a cached prefix) goes in
- linear4     a linear layer whose weights are 4-bit codes with a scale, and perhaps a minimum, for each group of inputs
              (`ops.Int4Linear`): a few rows while tokens are answered, hundreds for a prompt

The cache of one layer holds blocks of 64 tokens: codes k [blocks, kv heads, 64, width] and v [blocks, kv heads, width,
64] (width: the head size up to the next multiple of 64) and one float32 scale for each block and head. A sequence is a
row of the block table and its tokens so far. Sizes: the text encoder's heads (64 over 8 of 128) and the widths of this
repository's layers; head sizes and groupings beside them are generic.

With `own` false, `run` computes the same in elementary torch operations.
"""
import math

import torch

own = False

HIDDEN, WIDE, FF, VOCAB = 5376, 7168, 14336, 131072
LAYERS = {"square": (HIDDEN, HIDDEN), "out": (WIDE, HIDDEN), "up": (HIDDEN, 2 * FF), "down": (FF, HIDDEN), "head": (HIDDEN, VOCAB)}
BLOCK = 64
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
FLOOR = 1e-30                                                       # the least scale of a block


def listed():
    return [
        # one token of one sequence goes into a layer's cache: the smallest call there is
        {"name": "write_one", "kind": "write", "seqs": 1, "new": 1, "past": 299, "kv": 8, "dim": 128, "dtype": "bf16"},
        # a step of 64 sequences of ragged lengths, one token each
        {"name": "write_step_64", "kind": "write", "seqs": 64, "new": 1, "past": 4000, "kv": 8, "dim": 128, "dtype": "bf16"},
        # four prompts of up to 2048 tokens behind prefixes that end inside a block
        {"name": "write_prompts", "kind": "write", "seqs": 4, "new": 2048, "past": 37, "kv": 8, "dim": 128, "dtype": "bf16"},
        # one answered token over a short prompt: latency
        {"name": "one_300", "kind": "attention", "seqs": 1, "new": 1, "keys": 300, "kv": 8, "group": 8, "dim": 128, "dtype": "bf16"},
        # a step of 64 sequences of up to 8192 tokens: the serving load, bound by the cache's bytes
        {"name": "step_64x8192", "kind": "attention", "seqs": 64, "new": 1, "keys": 8192, "kv": 8, "group": 8, "dim": 128, "dtype": "bf16"},
        # one answered token over the longest context: few rows, one long axis
        {"name": "one_131072", "kind": "attention", "seqs": 1, "new": 1, "keys": 131072, "kv": 8, "group": 8, "dim": 128, "dtype": "f16"},
        # a prompt of 601 tokens in float32 behind a cached prefix, heads of 80 features, with the rows' log sums
        {"name": "prompt_601_f32", "kind": "attention", "seqs": 1, "new": 601, "keys": 901, "kv": 8, "group": 4, "dim": 80, "dtype": "f32", "lse": True},
        # a long prompt's second half: bound by its products
        {"name": "prompt_4096", "kind": "attention", "seqs": 1, "new": 4096, "keys": 8192, "kv": 8, "group": 8, "dim": 128, "dtype": "bf16"},
        # single-token products: a square layer with small groups and minima, and the widest layer (the vocabulary's)
        {"name": "linear4_square_1", "kind": "linear4", "m": 1, "layer": "square", "group": 32, "mins": True, "dtype": "bf16"},
        {"name": "linear4_head_1", "kind": "linear4", "m": 1, "layer": "head", "group": 128, "mins": False, "dtype": "bf16"},
        # a step of 16 sequences through the MLP's widest layer
        {"name": "linear4_up_16", "kind": "linear4", "m": 16, "layer": "up", "group": 64, "mins": False, "dtype": "f16"},
        # a prompt of 300 tokens through the MLP's second layer
        {"name": "linear4_down_300", "kind": "linear4", "m": 300, "layer": "down", "group": 32, "mins": True, "dtype": "bf16"},
    ]


def _between(rng, lo, hi):
    """A whole number of [lo, hi], spread evenly over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["write", "attention", "attention", "linear4"])
    if kind == "linear4":
        layer = rng.choice(["square", "out", "up", "down", "head"])
        return {"kind": kind, "m": _between(rng, 1, 512 if layer != "head" else 32), "layer": layer,
                "group": rng.choice([32, 64, 128]), "mins": rng.random() < 0.5, "dtype": rng.choice(["bf16", "bf16", "f16", "f32"])}
    heads = {"kv": rng.choice([1, 2, 4, 8, 16]), "dim": rng.choice([64, 80, 96, 128, 128, 256]),
             "dtype": rng.choice(["bf16", "bf16", "f16", "f32"])}
    seqs = _between(rng, 1, 64)
    if kind == "write":
        new = 1 if rng.random() < 0.4 else _between(rng, 2, max(2, 8192 // seqs))
        return {"kind": kind, "seqs": seqs, "new": new, "past": _between(rng, 1, 4096) - 1, **heads}
    heads["group"] = rng.choice([1, 2, 4, 7, 8, 16])
    if rng.random() < 0.6:                                          # answered tokens: one, or a few checked at once
        heads["dim"] = min(heads["dim"], 128)
        new, keys = rng.choice([1, 1, 1, 2, 5]), _between(rng, 16, 4 * 131072 * 8 // (heads["kv"] * max(seqs, 4)))
        keys = min(keys, 131072)
    else:                                                           # prompts
        new, before = _between(rng, 2, max(2, 2048 // seqs)), _between(rng, 1, 4096) - 1
        products = 4 * heads["kv"] * heads["group"] * heads["dim"] * seqs * (new + before)
        new = max(2, min(new, int(8e11 / products)))                # at most the longest listed prompt's work
        keys = new + before
    case = {"kind": kind, "seqs": seqs, "new": new, "keys": max(keys, new), **heads}
    case["lse"] = rng.random() < 0.3
    case["window"] = rng.choice([0, 0, 0, _between(rng, 16, 4096)])
    case["mask"] = rng.random() < 0.2
    return case


# ---- inputs -----------------------------------------------------------------------------------------------------------

def _spread(most, count, lowest, turn):
    """`count` whole numbers between lowest * most and most, the first of them `most`, in no order."""
    return [max(1, round(most * (1 - (1 - lowest) * ((i * turn) % count) / max(1, count - 1)))) if most else 0 for i in range(count)]


def _lengths(case):
    """(new tokens, tokens in the cache after them) of each sequence."""
    new = _spread(case["new"], case["seqs"], 0.4, 23)
    if case["kind"] == "write":
        return new, [n + p for n, p in zip(new, _spread(case["past"], case["seqs"], 0.2, 37))]
    return new, [max(n, l) for n, l in zip(new, _spread(case["keys"], case["seqs"], 0.2, 37))]


def _blocks(n):
    return -(-n // BLOCK)


def _width(dim):
    return -(-dim // 64) * 64


class _Make:
    """The inputs of one case, from its seed alone."""

    def __init__(self, seed):
        self.g = torch.Generator(device="cuda")
        self.g.manual_seed(int(seed))

    def normal(self, *shape, sd=1.0, dtype=torch.float32):
        return (torch.randn(shape, generator=self.g, device="cuda") * sd).to(dtype)

    def uniform(self, *shape):
        return torch.rand(shape, generator=self.g, device="cuda")


def _inputs(case, seed):
    """The case's tensors by name: what a user's program has in hand."""
    mk, dt = _Make(seed), TYPES[case["dtype"]]
    if case["kind"] == "linear4":
        k, n = LAYERS[case["layer"]]
        groups = k // case["group"]
        t = {"x": mk.normal(case["m"], k, dtype=dt),
             "codes": torch.randint(0, 256, (n, k // 2), generator=mk.g, device="cuda", dtype=torch.uint8),
             "scale": ((0.5 + mk.uniform(n, groups)) / (4.6 * math.sqrt(k))).half(), "bias": mk.normal(n, sd=0.1)}
        if case["mins"]:
            t["mins"] = (t["scale"].float() * (6 + 3 * mk.uniform(n, groups))).half()
        return t
    new, lengths = _lengths(case)
    kv, dim, seqs = case["kv"], case["dim"], case["seqs"]
    width, rows = _width(dim), sum(new)
    each = [_blocks(l) for l in lengths]
    wide = max(each)
    pages = sum(each) + 3
    # the blocks of the sequences lie anywhere in the pool
    order = torch.randperm(pages, generator=mk.g, device="cuda").to(torch.int32)
    table = torch.full((seqs, wide), -1, dtype=torch.int32, device="cuda")
    used = torch.arange(wide, device="cuda")[None, :] < torch.tensor(each, device="cuda")[:, None]
    table[used] = order[: sum(each)]
    starts = torch.tensor([sum(new[:i]) for i in range(seqs + 1)], dtype=torch.int32, device="cuda")
    t = {"table": table, "starts": starts, "lengths": torch.tensor(lengths, dtype=torch.int32, device="cuda"),
         "past": torch.tensor([l - n for l, n in zip(lengths, new)], dtype=torch.int32, device="cuda")}
    # keys with a few features larger than the rest, as rotated and normalized keys have them
    gain = torch.ones(width, device="cuda")
    gain[::16] = 3
    gain[dim:] = 0
    t["k"] = torch.empty(pages, kv, BLOCK, width, dtype=torch.int8, device="cuda")
    t["v"] = torch.empty(pages, kv, width, BLOCK, dtype=torch.int8, device="cuda")
    t["k_scale"], t["v_scale"] = (torch.empty(pages, kv, device="cuda") for _ in range(2))
    for p in range(0, pages, 256):
        x = mk.normal(min(256, pages - p), kv, BLOCK, width) * gain
        s = (x.abs().amax((2, 3)) / 127).clamp_min(FLOOR)
        t["k"][p:p + 256], t["k_scale"][p:p + 256] = (x / s[:, :, None, None]).round().to(torch.int8), s
        x = mk.normal(min(256, pages - p), kv, width, BLOCK)
        x[:, :, dim:] = 0
        s = (x.abs().amax((2, 3)) / 127).clamp_min(FLOOR)
        t["v"][p:p + 256], t["v_scale"][p:p + 256] = (x / s[:, :, None, None]).round().to(torch.int8), s
    if case["kind"] == "write":
        # the projections' rows: keys beside values, the newest tokens somewhat larger than what the blocks hold
        t["rows"] = mk.normal(rows, 2 * kv * dim, sd=1.2, dtype=dt)
        first = [(l - n) // BLOCK * BLOCK for l, n in zip(lengths, new)]
        seen = [l - f for l, f in zip(lengths, first)]
        t["first"] = torch.tensor(first, dtype=torch.int32, device="cuda")
        t["seen"] = torch.tensor([sum(seen[:i]) for i in range(seqs + 1)], dtype=torch.int32, device="cuda")
        t["k_out"], t["v_out"] = (torch.zeros(sum(seen), kv * dim, device="cuda") for _ in range(2))
        return t
    t["q"] = mk.normal(rows, kv * case["group"] * dim, dtype=dt)
    t["out"] = torch.zeros(rows, kv * case["group"] * dim, dtype=dt, device="cuda")
    if case.get("lse"):
        t["lse"] = torch.zeros(rows, kv * case["group"], device="cuda")
    if case.get("mask"):
        t["mask"] = (mk.uniform(seqs, wide * BLOCK) < 0.8).to(torch.uint8)
    return t


def prepare(case, seed):
    return {"case": dict(case), "t": _inputs(case, seed), "new": max(_lengths(case)[0]) if case["kind"] != "linear4" else 0,
            "keys": max(_lengths(case)[1]) if case["kind"] != "linear4" else 0}


# ---- the framework's calls ----------------------------------------------------------------------------------------------

_devices = {}


def _handles(s):
    """The framework's tensors over the state's, made once as a user's program makes them."""
    from sycl_minimax_h3_amd import Device, Tensor, ops

    stream = torch.cuda.current_stream().cuda_stream
    if stream not in _devices:
        _devices[stream] = Device.from_torch()
    dev, case = _devices[stream], s["case"]
    h = {k: Tensor.from_torch(v, dev=dev) for k, v in s["t"].items()}
    h["ops"] = ops
    if case["kind"] == "linear4":
        k, n = LAYERS[case["layer"]]
        s["t"]["y"] = torch.empty(case["m"], n, dtype=TYPES[case["dtype"]], device="cuda")
        h["y"] = Tensor.from_torch(s["t"]["y"], dev=dev)
        h["layer"] = ops.Int4Linear(h["codes"], h["scale"], h.get("mins"), h["bias"])
    else:
        kv, dim = case["kv"], case["dim"]
        h["cache"] = ops.KvCache(h["k"], h["v"], h["k_scale"], h["v_scale"], dim)
        if case["kind"] == "write":
            rows = len(s["t"]["rows"])
            h["k_rows"], h["v_rows"] = (ops.Rows(h["rows"], i * kv * dim, 2 * kv * dim, rows, kv, dim) for i in range(2))
            n = len(s["t"]["k_out"])
            h["k_out"], h["v_out"] = (ops.Rows(h[name], 0, kv * dim, n, kv, dim) for name in ("k_out", "v_out"))
            h["most"] = int((s["t"]["seen"][1:] - s["t"]["seen"][:-1]).max())
        else:
            heads = kv * case["group"]
            h["queries"] = ops.Rows(h["q"], 0, heads * dim, len(s["t"]["q"]), heads, dim)
    s["handles"] = h
    return h


def _run_own(s):
    h, t, kind = s.get("handles") or _handles(s), s["t"], s["case"]["kind"]
    ops = h["ops"]
    if kind == "linear4":
        h["layer"].forward(h["x"], h["y"])
        return t["y"]
    if kind == "write":
        ops.kv_write(h["cache"], h["table"], h["k_rows"], h["v_rows"], h["starts"], h["past"], s["new"])
        ops.kv_read(h["cache"], h["table"], h["seen"], h["first"], h["most"], h["k_out"], h["v_out"])
        return t["k_out"], t["v_out"], t["k_scale"], t["v_scale"]
    ops.kv_attention(h["cache"], h["table"], h["queries"], h["starts"], h["lengths"], s["new"], h["out"], max_len=s["keys"],
                     window=s["case"].get("window", 0), mask=h.get("mask"), lse=h.get("lse"))
    return (t["out"], t["lse"]) if "lse" in t else t["out"]


# ---- the plain form -----------------------------------------------------------------------------------------------------

def _row_index(starts, count):
    """For each sequence and each of its up to `count` rows: the row, and whether it has one."""
    j = torch.arange(count, device=starts.device)[None, :]
    return (starts[:-1, None] + j).clamp_max(max(int(starts[-1]) - 1, 0)).long(), j < (starts[1:] - starts[:-1])[:, None]


def _plain_linear4(t, case):
    n, half = t["codes"].shape
    codes = torch.stack([t["codes"] & 15, t["codes"] >> 4], -1).reshape(n, -1, case["group"]).float()
    scale = t["scale"].float()[:, :, None]
    w = scale * codes - t["mins"].float()[:, :, None] if case["mins"] else scale * (codes - 8)
    return (t["x"].float() @ w.reshape(n, 2 * half).t() + t["bias"]).to(t["x"].dtype)


def _plain_write_side(codes, scales, new, fresh, kept, dim):
    """One side (keys or values): codes [blocks, kv, 64, width] of the touched blocks and their scales, the new tokens'
    values [blocks, 64, kv, dim] where `fresh`; old tokens where `kept`. Returns the blocks' codes and scales after."""
    new = torch.where(fresh[:, :, None, None], new, torch.zeros_like(new)).permute(0, 2, 1, 3)      # [blocks, kv, 64, dim]
    most = new.abs().amax((2, 3))
    most = most / torch.full_like(most, 127)                        # (by a number, torch multiplies by its reciprocal)
    old = torch.where(kept.any(1)[:, None], scales, torch.zeros_like(scales))
    s = torch.maximum(torch.maximum(most, old), torch.full_like(most, FLOOR))
    again = (codes.float() * (old / s)[:, :, None, None]).round()
    again = torch.where(kept[:, None, :, None], again, torch.zeros_like(again))
    fill = torch.zeros_like(again)
    fill[..., :dim] = (new / s[:, :, None, None]).round().clamp(-127, 127)
    return torch.where(fresh[:, None, :, None], fill, again).to(torch.int8), s


def _plain_write(t, case, most_new):
    kv, dim = case["kv"], case["dim"]
    past, total = t["past"].long(), t["lengths"].long()
    first = past // BLOCK
    count = _blocks(most_new + BLOCK - 1)
    j = first[:, None] + torch.arange(count, device="cuda")[None, :]                                  # block of the sequence
    touched = j * BLOCK < total[:, None]
    pages = torch.gather(t["table"].long(), 1, j.clamp_max(t["table"].shape[1] - 1))[touched]
    at = (j[:, :, None] * BLOCK + torch.arange(BLOCK, device="cuda"))                                 # [seqs, count, 64]
    fresh = ((at >= past[:, None, None]) & (at < total[:, None, None]))[touched]
    kept = (at < past[:, None, None])[touched]
    row = (t["starts"].long()[:-1, None, None] + at - past[:, None, None])[touched].clamp(0, len(t["rows"]) - 1)
    x = t["rows"].float().reshape(len(t["rows"]), 2, kv, dim)
    k, ks = _plain_write_side(t["k"][pages], t["k_scale"][pages], x[:, 0][row], fresh, kept, dim)
    v, vs = _plain_write_side(t["v"][pages].transpose(2, 3), t["v_scale"][pages], x[:, 1][row], fresh, kept, dim)
    t["k"][pages], t["k_scale"][pages] = k, ks
    t["v"][pages], t["v_scale"][pages] = v.transpose(2, 3), vs
    # the touched blocks' tokens as values
    valid = (fresh | kept)
    t["k_out"].copy_((k.float() * ks[:, :, None, None]).permute(0, 2, 1, 3)[valid][:, :, :dim].reshape(-1, kv * dim))
    t["v_out"].copy_((v.float() * vs[:, :, None, None]).permute(0, 2, 1, 3)[valid][:, :, :dim].reshape(-1, kv * dim))
    return t["k_out"], t["v_out"], t["k_scale"], t["v_scale"]


def _plain_attention(t, case, most_new, most_keys):
    kv, dim, group, seqs = case["kv"], case["dim"], case["group"], case["seqs"]
    width, wide = t["k"].shape[3], _blocks(most_keys)
    pages = t["table"][:, :wide].long()
    there = (pages >= 0)
    pages = pages.clamp_min(0)
    k = t["k"][pages].float() * t["k_scale"][pages][..., None, None]                                  # [seqs, wide, kv, 64, width]
    k = k.permute(0, 2, 1, 3, 4).reshape(seqs, kv, wide * BLOCK, width)[..., :dim]
    v = t["v"][pages].float() * t["v_scale"][pages][..., None, None]                                  # [seqs, wide, kv, width, 64]
    v = v.permute(0, 2, 1, 4, 3).reshape(seqs, kv, wide * BLOCK, width)[..., :dim]
    row, real = _row_index(t["starts"], most_new)
    q = t["q"].float().reshape(-1, kv, group, dim)[row]                                               # [seqs, new, kv, group, dim]
    q = q.permute(0, 2, 3, 1, 4).reshape(seqs, kv, group * most_new, dim)
    s = torch.matmul(q, k.transpose(2, 3)).reshape(seqs, kv, group, most_new, wide * BLOCK) * dim ** -0.5
    at = torch.arange(wide * BLOCK, device="cuda")
    where = t["lengths"].long()[:, None] - (t["starts"][1:] - t["starts"][:-1]).long()[:, None] + torch.arange(most_new, device="cuda")
    seen = (at <= where[:, :, None]) & there.repeat_interleave(BLOCK, 1)[:, None, :]                  # [seqs, new, keys]
    if case.get("window"):
        seen &= at > where[:, :, None] - case["window"]
    if case.get("mask"):
        seen &= t["mask"][:, None, : wide * BLOCK] != 0
    s = s.masked_fill(~seen[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = torch.exp(s - top)
    total = p.sum(-1, keepdim=True)
    y = torch.matmul(p.reshape(seqs, kv, group * most_new, -1), v).reshape(seqs, kv, group, most_new, dim)
    y = torch.where(total > 0, y / total, torch.zeros_like(y))
    t["out"].copy_(y.permute(0, 3, 1, 2, 4)[real].reshape(-1, kv * group * dim))
    if "lse" in t:
        t["lse"].copy_((top + torch.log(total)).squeeze(-1).permute(0, 3, 1, 2)[real].reshape(-1, kv * group))
        return t["out"], t["lse"]
    return t["out"]


def run(state):
    if own:
        return _run_own(state)
    t, case = state["t"], state["case"]
    if case["kind"] == "linear4":
        return _plain_linear4(t, case)
    if case["kind"] == "write":
        return _plain_write(t, case, state["new"])
    return _plain_attention(t, case, state["new"], state["keys"])


# ---- what a pass cannot do without ----------------------------------------------------------------------------------------

def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    if case["kind"] == "linear4":
        (k, n), m = LAYERS[case["layer"]], case["m"]
        groups = n * (k // case["group"]) * (4 if case["mins"] else 2)
        return {"bytes": n * k // 2 + groups + 4 * n + size * m * (k + n), "flops": 2 * m * n * k}
    new, lengths = _lengths(case)
    kv, dim = case["kv"], case["dim"]
    if case["kind"] == "write":
        # the rows in, the kept tokens' codes in, the touched blocks' codes out, and their values out
        kept = sum((l - n) % BLOCK for n, l in zip(new, lengths))
        after = sum(new) + kept
        return {"bytes": 2 * kv * dim * (size * sum(new) + kept + after + 4 * after), "flops": 0}
    heads, window = kv * case["group"], case.get("window") or (1 << 60)
    read = sum(min(l, n + window - 1) for n, l in zip(new, lengths))
    pairs = sum(sum(min(l - n + 1 + i, window) for i in range(n)) for n, l in zip(new, lengths))
    return {"bytes": 2 * kv * dim * read + 2 * size * sum(new) * heads * dim, "flops": 4 * heads * dim * pairs}


# ---- the same in 64 bits ----------------------------------------------------------------------------------------------

def _exact_linear4(t, case):
    k, n = LAYERS[case["layer"]]
    x, parts = t["x"].double(), []
    for r in range(0, n, 8192):
        packed = t["codes"][r:r + 8192].to(torch.int64)
        c = torch.empty(len(packed), k, dtype=torch.float64, device="cuda")
        c[:, 0::2], c[:, 1::2] = (packed % 16).double(), (packed // 16).double()
        s = t["scale"][r:r + 8192].double().repeat_interleave(case["group"], 1)
        less = t["mins"][r:r + 8192].double().repeat_interleave(case["group"], 1) if case["mins"] else 8 * s
        parts.append(x @ (s * c - less).t())
    return torch.cat(parts, 1) + t["bias"].double()


def _exact_write(t, case):
    """By blocks, one after another. The scale, the ratio of two scales and the quotients are float32 by definition."""
    kv, dim = case["kv"], case["dim"]
    values, scales = ([], []), (t["k_scale"].clone(), t["v_scale"].clone())
    past, total, starts, table = (t[name].tolist() for name in ("past", "lengths", "starts", "table"))
    sides = t["rows"].double().reshape(-1, 2, kv, dim)
    f32 = lambda x: x.float().double()  # noqa: E731
    for b in range(case["seqs"]):
        for j in range(past[b] // BLOCK, _blocks(total[b])):
            lo, hi = j * BLOCK, min(total[b], j * BLOCK + BLOCK)
            keep, page = max(0, past[b] - lo), table[b][j]
            for i, side in enumerate(("k", "v")):
                x = sides[starts[b] + lo + keep - past[b]:starts[b] + hi - past[b], i].transpose(0, 1)    # [kv, new, dim]
                s = f32(x.abs().amax((1, 2)) / 127).clamp_min(f32(torch.tensor(FLOOR)).item())
                c = f32(x / s[:, None, None]).round().clamp(-127, 127)
                if keep:
                    was = t[side + "_scale"][page].double()
                    s = torch.maximum(s, was)
                    old = t[side][page].double() if side == "k" else t[side][page].double().transpose(1, 2)
                    c = torch.cat([f32(old[:, :keep, :dim] * f32(was / s)[:, None, None]).round(),
                                   f32(x / s[:, None, None]).round().clamp(-127, 127)], 1)
                scales[i][page] = s.float()
                values[i].append((c * s[:, None, None]).transpose(0, 1).reshape(-1, kv * dim))
    return torch.cat(values[0]), torch.cat(values[1]), scales[0].double(), scales[1].double()


def _exact_attention(t, case):
    kv, dim, group = case["kv"], case["dim"], case["group"]
    out = torch.zeros(t["out"].shape, dtype=torch.float64, device="cuda")
    lse = torch.zeros(len(out), kv * group, dtype=torch.float64, device="cuda")
    lengths, starts = t["lengths"].tolist(), t["starts"].tolist()
    for b in range(case["seqs"]):
        n, length = starts[b + 1] - starts[b], lengths[b]
        pages = t["table"][b, :_blocks(length)].long()
        at = torch.arange(length, device="cuda")
        where = torch.arange(length - n, length, device="cuda")
        hide = at[None, :] > where[:, None]
        if case.get("window"):
            hide |= at[None, :] <= where[:, None] - case["window"]
        if case.get("mask"):
            hide |= t["mask"][b, None, :length] == 0
        for h in range(kv):
            k = (t["k"][pages, h].double() * t["k_scale"][pages, h].double()[:, None, None]).reshape(-1, t["k"].shape[3])[:length, :dim]
            v = (t["v"][pages, h].double() * t["v_scale"][pages, h].double()[:, None, None]).transpose(1, 2).reshape(-1, t["k"].shape[3])[:length, :dim]
            for g in range(h * group, (h + 1) * group):
                s = t["q"][starts[b]:starts[b + 1], g * dim:(g + 1) * dim].double() @ k.t().contiguous() / math.sqrt(dim)
                s[hide] = -math.inf
                lse[starts[b]:starts[b + 1], g] = torch.logsumexp(s, 1)
                out[starts[b]:starts[b + 1], g * dim:(g + 1) * dim] = torch.nan_to_num(torch.softmax(s, 1), nan=0.0) @ v
    return (out, lse) if "lse" in t else out


def exact(case, seed):
    t = _inputs(case, seed)
    return {"linear4": _exact_linear4, "write": _exact_write, "attention": _exact_attention}[case["kind"]](t, case)
