"""Decoding from fewer bits, as cases that can be timed and compared: a key/value cache held in 8- or 4-bit codes (quantised as it is
written, read back, attended to) and projections in 8-bit integers.  What a decode step streams from memory is its weights and its
cache; both are held here in a half or a quarter of the bytes.

The formats.  A row of a cache (one token's key or value of one head, `dim` values x) with Q = 2^bits - 1 and its range widened to
hold zero, low = min(0, min x), high = max(0, max x):
    scale = bf16((high - low) / Q)    the difference in fp32; 0 where that is 0, and every code with it
    zero  = rint(-low / scale)        cut to 0 .. Q
    code  = rint(x / scale) + zero    cut to 0 .. Q; it stands for scale * (code - zero)
Codes of 8 bits lie one to a byte, codes of 4 bits two (feature 2 i in the low half); a row's two parameters lie in 32 bits, the bf16
pattern of the scale in the lower 16, zero in the upper 16.  A row of a matrix in 8-bit integers: scale = bf16(max |x| / 127), held in
fp32, code = rint(x / scale) cut to -127 .. 127.

A scale of 8 significant bits makes fp32 enough for all of this: a quotient x / scale that is not half way between two integers is
further from it than fp32's rounding, so codes are those of exact arithmetic."""
import math

import torch

own = False  # set from outside: run() then makes the framework's calls

EPI_NONE, EPI_RES, EPI_SWIGLU = 0, 4, 5
CAUSAL, TREE = 0, 1


def _rd():
    import os
    import sys

    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ml-recurrent-drafter_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import recurrent_drafting

    return recurrent_drafting


# Heads and widths are those of this repository's decoders: 2048 (16 heads on 4), 4096 (32 on 8, 32 on 32), feed-forward 5632 and 11008.
def listed():
    return [
        # what one decode step of eight requests adds to a layer's cache, and reads back: latency
        dict(name="append step", kind="append", bits=4, kv=32, dim=128, dtype="bfloat16", new="1,1,1,1,1,1,1,1", base="500,37,433,256,500,311,90,128"),
        # prompts of different lengths, in portions, on what is there already
        dict(name="append prompts", kind="append", bits=8, kv=8, dim=128, dtype="bfloat16", new="8192,17,700,2048,3001,333,5000,1", base="0,4000,0,1024,0,64,900,8191"),
        # a 32-bit model's short cache, its layer handed to code that wants plain keys and values
        dict(name="read short fp32", kind="read", bits=8, kv=4, dim=64, dtype="float32", length="333,1,96"),
        # a large server's layer
        dict(name="read long", kind="read", bits=4, kv=32, dim=128, dtype="bfloat16", length="8192,7001,8190,4096,16000,5555,12288,9999"),
        # one user, a short chat: latency of a step
        dict(name="attention one user", kind="attention", bits=4, heads=32, kv=8, dim=128, new="1", base="1000", mode="causal"),
        # one user, a long document
        dict(name="attention one user long", kind="attention", bits=4, heads=32, kv=8, dim=128, new="1", base="131071", mode="causal"),
        # a server's batch, every head with keys of its own, rows of very different lengths, one of them new
        dict(name="attention server batch", kind="attention", bits=8, heads=32, kv=32, dim=128,
             new="1,1,1,1,1,1,1,1,1,1,1,1,1,1,1,1", base="500,16001,8191,333,1,12000,4096,9999,700,0,3001,15000,64,2500,6000,10240", mode="causal"),
        # the verify step of the headline workload: eight requests, packed draft trees
        dict(name="attention draft trees", kind="attention", bits=4, heads=32, kv=32, dim=128, new="97,120,64,101,88,140,79,93",
             base="500,521,433,256,500,311,490,128", mode="tree"),
        # a long prompt in portions, grouped heads
        dict(name="attention portion", kind="attention", bits=8, heads=32, kv=8, dim=128, new="2048,333", base="6143,1000", mode="causal"),
        # one token through the q, k, v projection: the weights' bytes
        dict(name="product one token", kind="product", rows=1, k=4096, n=12288, out="bfloat16", epilogue="none"),
        # a packed draft through the second half of the feed-forward, added to the residual stream
        dict(name="product draft residual", kind="product", rows=110, k=11008, n=4096, out="bfloat16", epilogue="residual"),
        # a prompt through gate and up, interleaved
        dict(name="product prompt gated", kind="product", rows=4095, k=4096, n=22016, out="bfloat16", epilogue="swiglu"),
    ]


def draw(rng):
    def spread(low, high):
        return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))

    def texts(values):
        return ",".join(str(v) for v in values)

    kind = rng.choice(["append", "read", "attention", "attention", "attention", "product", "product"])
    bits = rng.choice([4, 8])
    if kind == "product":
        k, n = rng.choice([2048, 4096, 5632, 11008, 16 * spread(16, 688)]), rng.choice([4096, 6144, 12288, 22016, 2 * spread(64, 11008)])
        return dict(kind=kind, rows=spread(1, min(4095, 300000000000 // (k * n))), k=k, n=n, out=rng.choice(["bfloat16", "bfloat16", "float32"]), epilogue=rng.choice(["none", "residual", "swiglu"]))
    kv, dim, batch = rng.choice([2, 4, 8, 32]), rng.choice([64, 128, 128]), spread(1, 24)
    if kind == "append":
        most = max(1, min(8192, 120000 // (batch * kv)))
        return dict(kind=kind, bits=bits, kv=kv, dim=dim, dtype=rng.choice(["bfloat16", "bfloat16", "float32"]), new=texts(spread(1, most) for _ in range(batch)),
                    base=texts(rng.randint(0, 8000) for _ in range(batch)))
    if kind == "read":
        most = max(1, min(16000, 2000000 // (batch * kv)))
        return dict(kind=kind, bits=bits, kv=kv, dim=dim, dtype=rng.choice(["bfloat16", "bfloat16", "float32"]), length=texts(spread(1, most) for _ in range(batch)))
    heads = kv * rng.choice([g for g in (1, 2, 4, 8) if kv * g <= 32])
    shape = rng.choice(["step", "step", "trees", "portion"])
    if shape == "step":
        most = max(64, min(131071, 2600000 // (batch * kv)))
        return dict(kind=kind, bits=bits, heads=heads, kv=kv, dim=dim, new=texts([1] * batch), base=texts(spread(1, most) - 1 for _ in range(batch)), mode="causal")
    if shape == "trees":
        batch = min(batch, 16)
        return dict(kind=kind, bits=bits, heads=heads, kv=kv, dim=dim, new=texts(spread(2, 225) for _ in range(batch)),
                    base=texts(spread(1, 2000) for _ in range(batch)), mode="tree")
    batch = min(batch, 4)
    return dict(kind=kind, bits=bits, heads=heads, kv=kv, dim=dim, new=texts(spread(2, 1024) for _ in range(batch)),
                base=texts(spread(1, 6000) - 1 for _ in range(batch)), mode="causal")


def _numbers(text):
    return [int(v) for v in text.split(",")]


# ---------------------------------------------------------------------------------------------- the plain forms
def _quantised(x, bits):
    """Codes (int64, one each), scale and zero (fp32, [..., 1]) of rows x (fp32)."""
    q = float(2 ** bits - 1)
    low, high = x.amin(-1, keepdim=True).clamp(max=0.0), x.amax(-1, keepdim=True).clamp(min=0.0)
    scale = ((high - low) / q).to(torch.bfloat16).float()
    divisor = torch.where(scale > 0, scale, torch.ones_like(scale))
    zero = torch.round(-low / divisor).clamp(0.0, q) * (scale > 0)
    code = (torch.round(x / divisor) + zero).clamp(0.0, q) * (scale > 0)
    return code.to(torch.int64), scale, zero


def _packed(code, bits):
    code = code.to(torch.uint8)
    return code if bits == 8 else code[..., 0::2] | (code[..., 1::2] << 4)


def _parameters(scale, zero):
    """[..., 2] int16: the scale's bf16 pattern, zero."""
    return torch.cat([scale.to(torch.bfloat16).view(torch.int16), zero.to(torch.int16)], dim=-1)


def _unpacked(codes, bits):
    return codes if bits == 8 else torch.stack([codes & 15, codes >> 4], dim=-1).flatten(-2)


def _values(codes, parameters, bits):
    """fp32: scale * (code - zero)."""
    scale = parameters[..., 0:1].contiguous().view(torch.bfloat16).float()
    return scale * (_unpacked(codes, bits).float() - parameters[..., 1:2].float())


def _int8(x):
    scale = (x.abs().amax(-1, keepdim=True) / 127.0).to(torch.bfloat16).float()
    divisor = torch.where(scale > 0, scale, torch.ones_like(scale))
    return torch.round(x / divisor).clamp(-127.0, 127.0) * (scale > 0), scale


def _attention(q, k, v, visible, scale):
    """q [B, n, heads, dim], k and v [B, kv, S, dim], visible [B, n, S] -> [B, n, heads, dim], all fp32."""
    B, n, heads, dim = q.shape
    kv = k.shape[1]
    s = torch.matmul(q.reshape(B, n, kv, heads // kv, dim).permute(0, 2, 3, 1, 4).reshape(B, kv, -1, dim), k.transpose(-1, -2)) * scale
    s = s.reshape(B, kv, heads // kv, n, -1).masked_fill(~visible[:, None, None], float("-inf"))
    p = torch.exp(s - s.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    o = torch.matmul(p.reshape(B, kv, (heads // kv) * n, -1), v)
    return o.reshape(B, kv, heads // kv, n, dim).permute(0, 3, 1, 2, 4).reshape(B, n, heads, dim)


# ---------------------------------------------------------------------------------------------- states
def _rows(generator, shape, dtype):
    """Keys or values as layers have them: bell-shaped, some features larger throughout."""
    x = torch.randn(shape, generator=generator, device="cuda")
    wide = 1.0 + 3.0 * (torch.rand(shape[-1], generator=generator, device="cuda") < 0.05)
    return (x * wide).to(dtype)


def _cache(case, capacity, batch):
    """Storage of one layer."""
    if own:
        return _rd().kv_cache.QuantizedCache(batch, capacity, 1, case["kv"], case["dim"], case["bits"], torch.device("cuda"))
    return None


def _filled(case, generator, batch, capacity):
    """Codes and parameters of `capacity` keys and values of every row and head."""
    got = []
    for _ in range(2):
        codes, params = [], []
        for _ in range(batch):  # a row at a time: the 32-bit values of all need not be there at once
            code, scale, zero = _quantised(_rows(generator, (case["kv"], capacity, case["dim"]), torch.bfloat16).float(), case["bits"])
            codes.append(_packed(code, case["bits"]))
            params.append(_parameters(scale, zero))
        got += [torch.stack(codes), torch.stack(params)]
    return got


def _slots(counts, first):
    """(batch row, slot) of every new token, row after row."""
    rows = [b for b, c in enumerate(counts) for _ in range(c)]
    slots = [first[b] + i for b, c in enumerate(counts) for i in range(c)]
    return torch.tensor(rows, dtype=torch.int32, device="cuda"), torch.tensor(slots, dtype=torch.int32, device="cuda")


def _starts(counts):
    got = [0]
    for c in counts:
        got.append(got[-1] + c)
    return torch.tensor(got, dtype=torch.int32, device="cuda")


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _tree(counts, seed):
    """Ancestors (themselves included) of the packed tokens of each row: lists of lists."""
    import random

    r, rows = random.Random(seed), []
    for n in counts:
        sees, depth = [], []
        for i in range(n):
            parents = [j for j in range(max(0, i - 40), i) if depth[j] < 4]
            j = r.choice(parents) if i and parents else None
            depth.append(0 if j is None else depth[j] + 1)
            sees.append(([] if j is None else sees[j]) + [i])
        rows.append(sees)
    return rows


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind = case["kind"]
    st = dict(case=case)
    if kind == "product":
        rows, k, n = case["rows"], case["k"], case["n"]
        out = getattr(torch, case["out"])
        st["x"] = (torch.randn(rows, k, generator=g, device="cuda") * (1.0 + 7.0 * (torch.rand(k, generator=g, device="cuda") < 0.01))).to(torch.bfloat16)
        w = torch.randn(n, k, generator=g, device="cuda") * 0.02
        codes, scales = _int8(w)
        st["w_codes"], st["w_scales"] = codes.to(torch.int8), scales.view(-1).contiguous()
        wide = n // 2 if case["epilogue"] == "swiglu" else n
        st["residual"] = torch.randn(rows, wide, generator=g, device="cuda").to(out) if case["epilogue"] == "residual" else None
        st["out"] = torch.empty(rows, wide, dtype=out, device="cuda")
        if own:
            st["linear"] = _rd().modeling_common.Int8Linear.from_codes(st["w_codes"], st["w_scales"])
        return st
    if kind == "append":
        new, base = _numbers(case["new"]), _numbers(case["base"])
        m, dtype, kv, dim = sum(new), getattr(torch, case["dtype"]), case["kv"], case["dim"]
        both = _rows(g, (m, 2, kv, dim), dtype)  # as a projection leaves them: a token's keys, then its values
        st["k"], st["v"] = both[:, 0], both[:, 1]
        st["tok_row"], st["tok_slot"] = _slots(new, base)
        capacity = (max(b + n for b, n in zip(base, new)) + 63) // 64 * 64
        st["begin"], st["length"] = _i32(base), _i32(new)
        st["cache"] = _cache(case, capacity, len(new))
        if not own:
            codes = dim * case["bits"] // 8
            st["codes"] = torch.zeros(2, len(new), kv, capacity, codes, dtype=torch.uint8, device="cuda")
            st["params"] = torch.zeros(2, len(new), kv, capacity, 2, dtype=torch.int16, device="cuda")
        st["k_out"], st["v_out"] = (torch.zeros(len(new), kv, max(new), dim, dtype=dtype, device="cuda") for _ in range(2))
        return st
    if kind == "read":
        length = _numbers(case["length"])
        capacity = (max(length) + 63) // 64 * 64
        st["held"] = _filled(case, g, len(length), capacity)
        st["begin"], st["length"] = _i32([0] * len(length)), _i32(length)
        dtype = getattr(torch, case["dtype"])
        st["k_out"], st["v_out"] = (torch.zeros(len(length), case["kv"], max(length), case["dim"], dtype=dtype, device="cuda") for _ in range(2))
    else:
        new, base = _numbers(case["new"]), _numbers(case["base"])
        batch, m, most = len(new), sum(new), max(b + n for b, n in zip(base, new))
        capacity = (most + 63) // 64 * 64
        st["held"] = _filled(case, g, batch, capacity)
        st["q"] = torch.randn(m, case["heads"] * case["dim"], generator=g, device="cuda").to(torch.bfloat16)
        st["out"] = torch.empty_like(st["q"])
        st["row_start"], st["kv_begin"], st["base_len"] = _starts(new), _i32([0] * batch), _i32(base)
        st["max_new"], st["max_kv"], st["most"] = max(new), most, most
        st["tree_mask"] = None
        if case["mode"] == "tree":
            words = (max(new) + 31) // 32
            bits = [[0] * words for _ in range(m)]
            t = 0
            for sees in _tree(new, seed):
                for seen in sees:
                    for j in seen:
                        bits[t][j >> 5] |= 1 << (j & 31)
                    t += 1
            st["tree_mask"] = torch.tensor(bits, dtype=torch.int64, device="cuda").to(torch.int32)
        # where a token of the padded batch [B, max_new] lies among the packed ones
        st["tok_row"], tok_index = _slots(new, [0] * batch)
        st["place"] = st["tok_row"].long() * max(new) + tok_index.long()
    if own:
        st["cache"] = _cache(case, capacity, st["held"][0].shape[0])
        layer = st["cache"].layers[0]
        for plane, held in zip((layer.k_codes, layer.k_params, layer.v_codes, layer.v_params), st["held"]):
            plane[:, :, :capacity].copy_(held)
    return st


def _visible(st, case):
    """[B, max_new, most] bool: which keys each query of the padded batch sees (one, where there is no query: it is not looked at)."""
    new = (st["row_start"][1:] - st["row_start"][:-1])[:, None, None]
    base = st["base_len"][:, None, None]
    i = torch.arange(st["max_new"], device="cuda")[None, :, None]
    j = torch.arange(st["most"], device="cuda")[None, None, :]
    if case["mode"] == "causal":
        seen = j <= base + i
    else:
        padded = torch.zeros(new.shape[0] * st["max_new"], st["tree_mask"].shape[1], dtype=torch.int32, device="cuda")
        padded[st["place"]] = st["tree_mask"]
        padded = padded.view(new.shape[0], st["max_new"], -1)
        among = (j - base).clamp(0, st["max_new"] - 1).expand(-1, st["max_new"], -1)
        bit = (torch.gather(padded, 2, among >> 5) >> (among & 31)) & 1
        seen = (j < base) | ((bit != 0) & (j < base + new))
    return seen | ((i >= new) & (j == 0))


def _run_plain(st):
    case = st["case"]
    kind = case["kind"]
    if kind == "product":
        codes, scale = _int8(st["x"].float())
        c = torch.matmul(codes, st["w_codes"].float().t()) * (scale * st["w_scales"])
        if case["epilogue"] == "residual":
            c = c + st["residual"].float()
        elif case["epilogue"] == "swiglu":
            gate, up = c[:, 0::2], c[:, 1::2]
            c = gate / (1.0 + torch.exp(-gate)) * up
        st["out"].copy_(c)
        return st["out"]
    bits = case["bits"]
    if kind == "append":
        code, scale, zero = _quantised(torch.stack([st["k"], st["v"]]).float(), bits)
        row, slot = st["tok_row"].long(), st["tok_slot"].long()
        st["codes"][:, row, :, slot] = _packed(code, bits).transpose(0, 1)
        st["params"][:, row, :, slot] = _parameters(scale, zero).transpose(0, 1)
        index = slot - st["begin"].long()[row]
        for out, codes, params in ((st["k_out"], st["codes"][0], st["params"][0]), (st["v_out"], st["codes"][1], st["params"][1])):
            out[row, :, index] = _values(codes[row, :, slot], params[row, :, slot], bits).to(out.dtype)
        return st["k_out"], st["v_out"]
    if kind == "read":
        n = st["k_out"].shape[2]
        there = (torch.arange(n, device="cuda")[None, :] < st["length"][:, None])[:, None, :, None]
        for out, codes, params in ((st["k_out"], st["held"][0], st["held"][1]), (st["v_out"], st["held"][2], st["held"][3])):
            out.copy_(torch.where(there, _values(codes[:, :, :n], params[:, :, :n], bits), out))
        return st["k_out"], st["v_out"]
    heads, dim, most = case["heads"], case["dim"], st["most"]
    batch = st["base_len"].shape[0]
    q = torch.zeros(batch * st["max_new"], heads, dim, device="cuda")
    q[st["place"]] = st["q"].float().view(-1, heads, dim)
    k = _values(st["held"][0][:, :, :most], st["held"][1][:, :, :most], bits)
    v = _values(st["held"][2][:, :, :most], st["held"][3][:, :, :most], bits)
    o = _attention(q.view(batch, st["max_new"], heads, dim), k, v, _visible(st, case), 1.0 / math.sqrt(dim))
    st["out"].copy_(o.reshape(-1, heads * dim)[st["place"]])
    return st["out"]


def _run_own(st):
    case = st["case"]
    kind = case["kind"]
    if kind == "product":
        st["linear"](st["x"], st["out"], {"none": EPI_NONE, "residual": EPI_RES, "swiglu": EPI_SWIGLU}[case["epilogue"]], residual=st["residual"])
        return st["out"]
    if kind == "append":
        st["cache"].append(0, st["k"], st["v"], st["tok_row"], st["tok_slot"])
    if kind in ("append", "read"):
        st["cache"].read(0, st["begin"], st["length"], st["k_out"], st["v_out"])
        return st["k_out"], st["v_out"]
    st["cache"].attend(0, st["q"], st["out"], st["row_start"], st["kv_begin"], st["base_len"], st["max_new"], st["max_kv"],
                       mode=CAUSAL if case["mode"] == "causal" else TREE, tree_mask=st["tree_mask"])
    return st["out"]


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---------------------------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    kind = case["kind"]
    if kind == "product":
        rows, k, n = case["rows"], case["k"], case["n"]
        wide = n // 2 if case["epilogue"] == "swiglu" else n
        size = 2 if case["out"] == "bfloat16" else 4
        return {"bytes": rows * k * 2 + n * (k + 4) + rows * wide * size * (2 if case["epilogue"] == "residual" else 1), "flops": 2 * rows * k * n}
    row = case["dim"] * case["bits"] // 8 + 4  # a key or a value as it is held
    if kind in ("append", "read"):
        m = sum(_numbers(case["new" if kind == "append" else "length"]))
        plain = case["dim"] * (2 if case["dtype"] == "bfloat16" else 4)
        each = 2 * plain + row if kind == "append" else row + plain  # append: read, written as codes, and the values that these stand for
        return {"bytes": 2 * m * case["kv"] * each, "flops": 2 * m * case["kv"] * case["dim"] * 2}
    new, base = _numbers(case["new"]), _numbers(case["base"])
    keys = sum(b + n for b, n in zip(base, new))
    if case["mode"] == "causal":
        pairs = sum(n * b + n * (n + 1) // 2 for b, n in zip(base, new))
    else:
        pairs = sum(n * b + 3 * n for b, n in zip(base, new))
    return {"bytes": 2 * keys * case["kv"] * row + 2 * sum(new) * case["heads"] * case["dim"] * 2, "flops": 4 * pairs * case["heads"] * case["dim"]}


# ---------------------------------------------------------------------------------------------- in 64 bits
def _exact_bf16(x):
    """The 64-bit numbers x rounded once to 8 significant bits, ties to even."""
    mantissa, exponent = torch.frexp(x)
    return torch.ldexp(torch.round(mantissa * 256.0), exponent - 8)


def _exact_held(x, bits):
    """What rows x (64 bits) come to as codes; the range's difference is rounded to 32 bits by definition."""
    top = 2 ** bits - 1
    low = torch.minimum(x.min(dim=-1, keepdim=True).values, torch.zeros((), dtype=x.dtype, device=x.device))
    high = torch.maximum(x.max(dim=-1, keepdim=True).values, torch.zeros((), dtype=x.dtype, device=x.device))
    scale = _exact_bf16((high - low).float().double() / top)
    zero = torch.round(-low / scale).clamp(0, top)
    value = ((torch.round(x / scale) + zero).clamp(0, top) - zero) * scale
    return torch.where(scale > 0, value, torch.zeros_like(value))


def _exact_stored(codes, params, bits):
    n = codes.shape[-1] * 8 // bits
    at = torch.arange(n, device=codes.device)
    shift = (at * bits % 8).to(torch.uint8)
    code = (codes.index_select(-1, at * bits // 8) >> shift) & (2 ** bits - 1)
    pattern = params[..., 0].to(torch.int32) << 16
    return (code.double() - params[..., 1:].double()) * pattern.view(torch.float32).double()[..., None]


def exact(case, seed):
    st = prepare(case, seed)
    kind = case["kind"]
    if kind == "product":
        if case["rows"] * case["n"] * case["k"] > 5e11:
            return None
        def held(x):
            scale = _exact_bf16(x.abs().max(dim=-1, keepdim=True).values / 127)
            return torch.round(x / scale).clamp(-127, 127), scale

        codes, scale = held(st["x"].double())
        c = (codes @ st["w_codes"].double().t()) * scale * st["w_scales"].double()[None, :]
        if st["residual"] is not None:
            c = c + st["residual"].double()
        if case["epilogue"] == "swiglu":
            pair = c.view(c.shape[0], -1, 2)
            c = pair[..., 1] * pair[..., 0] * torch.sigmoid(pair[..., 0])
        return c
    if kind == "append":
        got = []
        for x, out in ((st["k"], st["k_out"]), (st["v"], st["v_out"])):
            values, want = _exact_held(x.double(), case["bits"]), out.double()
            t = 0
            for b, n in enumerate(_numbers(case["new"])):
                want[b, :, :n] = values[t : t + n].transpose(0, 1)
                t += n
            got.append(want)
        return tuple(got)
    k_codes, k_params, v_codes, v_params = st["held"]
    if kind == "read":
        got = []
        for codes, params, out in ((k_codes, k_params, st["k_out"]), (v_codes, v_params, st["v_out"])):
            want = out.double()
            for b, n in enumerate(_numbers(case["length"])):
                want[b, :, :n] = _exact_stored(codes[b, :, :n], params[b, :, :n], case["bits"])
            got.append(want)
        return tuple(got)
    new, base = _numbers(case["new"]), _numbers(case["base"])
    heads, kv, dim = case["heads"], case["kv"], case["dim"]
    if sum(n * (b + n) for b, n in zip(base, new)) * heads * dim > 2e12:
        return None
    trees = _tree(new, seed) if case["mode"] == "tree" else None
    want, t = torch.empty(sum(new), heads, dim, dtype=torch.float64, device="cuda"), 0
    for b, n in enumerate(new):
        end = base[b] + n
        hidden = torch.ones(n, n, dtype=torch.bool).triu(1) if trees is None else torch.ones(n, n, dtype=torch.bool)
        for i, seen in enumerate(trees[b] if trees is not None else ()):
            hidden[i, seen] = False
        hidden = hidden.cuda()
        for g in range(kv):
            keys = _exact_stored(k_codes[b, g, :end], k_params[b, g, :end], case["bits"])
            values = _exact_stored(v_codes[b, g, :end], v_params[b, g, :end], case["bits"])
            for h in range(g * (heads // kv), (g + 1) * (heads // kv)):
                s = st["q"].view(-1, heads, dim)[t : t + n, h].double() @ keys.t() / math.sqrt(dim)
                s[:, base[b] :].masked_fill_(hidden, float("-inf"))
                want[t : t + n, h] = torch.softmax(s, dim=-1) @ values
        t += n
    return want.view(sum(new), heads * dim)
