"""The attention operators' cases: what is measured, the plain form of each operator and its result in
64 bits.

Attention of query rows over states of another length (forward and backward), the 8-bit cache of such
states, and attention over that cache.  Where `own` is false, run() computes an operator with
elementary torch operations in 32 bits; where it is true, it calls the library.
"""
import math
import os
import sys

import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
E4M3_MAX = 448.0


def listed():
    return [
        # one request's single token over a short encoder output: nothing but latency
        _attend("attend-token", "bf16", 1, 1, 8, 8, 64, 64, "none"),
        # a decoding step of 32 sequences: one token each over 1500 encoder states, ragged lengths
        _attend("attend-step", "fp16", 32, 1, 16, 16, 1500, 64, "counts"),
        # a padded batch with odd sizes and a head of 80 dimensions; the mask leaves one sequence nothing
        _attend("attend-odd", "fp16", 3, 333, 12, 4, 1001, 80, "mask"),
        # a long target text over a long source, heads shared four to one: the arithmetic bound
        _attend("attend-long", "bf16", 4, 2048, 16, 4, 8192, 128, "none"),
        # the training step of a small padded batch
        _attend("grad-short", "fp16", 2, 65, 8, 2, 257, 64, "mask", op="grad"),
        # the training step at the lengths of attend-long
        _attend("grad-long", "bf16", 2, 2048, 16, 4, 8192, 128, "counts", op="grad"),
        # one short sequence enters the cache
        _cache("store-short", "store", "fp16", 1, 0, 8, 8, 200, 64, 16, "ragged"),
        # a full batch of long sequences enters the cache: the memory bound of writing
        _cache("store-long", "store", "bf16", 32, 0, 8, 8, 8192, 128, 64, "full"),
        # one token over one short cached sequence
        _cache("cached-token", "cached", "bf16", 1, 1, 8, 2, 1000, 128, 16, "ragged"),
        # a decoding step of 64 sequences over long caches: the memory bound of reading
        _cache("cached-step", "cached", "bf16", 64, 1, 32, 8, 8192, 128, 64, "ragged"),
        # every query reads the 16 blocks that a search found for it, some of them missing
        _cache("cached-found", "cached", "fp16", 1024, 1, 8, 8, 512, 64, 32, "found"),
        # a chunk of 512 target tokens over cached states
        _cache("cached-rows", "cached", "fp16", 4, 512, 16, 4, 4096, 128, 32, "ragged"),
    ]


def _attend(name, dtype, batch, q, heads, state_heads, n, dim, masked, layout="heads", op="attend"):
    case = dict(op=op, dtype=dtype, batch=batch, q=q, heads=heads, state_heads=state_heads, n=n, dim=dim,
                masked=masked, layout=layout)
    return dict(case, name=name) if name else case


def _cache(name, op, dtype, batch, q, heads, state_heads, n, dim, block, table):
    case = dict(op=op, dtype=dtype, batch=batch, q=q, heads=heads, state_heads=state_heads, n=n, dim=dim,
                block=block, table=table)
    return dict(case, name=name) if name else case


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    limits = {case["op"]: {"bytes": 0.0, "flops": 0.0} for case in listed()}
    for case in listed():
        for kind, amount in work(case).items():
            limits[case["op"]][kind] = max(limits[case["op"]][kind], amount)
    while True:
        op = rng.choice(sorted(limits))
        dtype = rng.choice(sorted(TYPES))
        dim = rng.choice([64, 128, 8 * rng.randint(2, 16)])
        state_heads = rng.choice([1, 2, 3, 4, 8, 16])
        heads = state_heads * rng.choice([1, 1, 2, 4, 5, 8])
        if op in ("attend", "grad"):
            q = rng.choice([1, _log(rng, 2, 2048)]) if op == "attend" else _log(rng, 1, 2048)
            case = _attend(None, dtype, _log(rng, 1, 32), q, heads, state_heads, _log(rng, 1, 8192), dim,
                           rng.choice(["none", "counts", "mask"]), rng.choice(["heads", "rows"]), op)
        else:
            table = rng.choice(["full", "ragged"]) if op == "store" else rng.choice(["ragged", "found"])
            q = 0 if op == "store" else rng.choice([1, 1, _log(rng, 2, 512)])
            case = _cache(None, op, dtype, _log(rng, 1, 64), q, state_heads if op == "store" else heads,
                          state_heads, _log(rng, 1, 8192), dim, rng.choice([16, 32, 64, 128]), table)
        scores = case["batch"] * case["heads"] * q * case["n"]
        if scores <= 2 ** 30 and all(amount <= limits[op][kind] for kind, amount in work(case).items()):
            return case


def _valid_share(case):
    """The share of the states that take part, on average: what the operator has to read and compute."""
    return {"none": 1.0, "full": 1.0, "counts": 0.75, "ragged": 0.75, "mask": 0.75, "found": 0.9}[
        case.get("masked") or case.get("table")]


def work(case):
    b, q, h, hs, n, d = (case[x] for x in ("batch", "q", "heads", "state_heads", "n", "dim"))
    states = b * hs * n * d * _valid_share(case)
    rows = b * h * q * d
    products = 2.0 * b * h * q * n * d * _valid_share(case)
    if case["op"] == "attend":
        return {"bytes": 4.0 * states + 4.0 * rows + 4.0 * b * h * q, "flops": 2 * products}
    if case["op"] == "grad":
        # queries, their gradient, out and its gradient; keys and values read, their gradients written whole
        return {"bytes": 4.0 * states + 4.0 * b * hs * n * d + 8.0 * rows + 4.0 * b * h * q, "flops": 5 * products}
    if case["op"] == "store":
        return {"bytes": 4.0 * states + 2.0 * states, "flops": 0.0}
    return {"bytes": 2.0 * states + 4.0 * rows + 4.0 * b * h * q, "flops": 2 * products}


# ---- inputs --------------------------------------------------------------------------------------


def _normal(gen, shape, dtype, spread=1.0):
    return (torch.randn(shape, generator=gen, device="cuda") * spread).to(dtype)


def _states(gen, shape, dtype):
    """Keys or values: every head has a magnitude of its own and a few channels that stand out."""
    b, h, n, d = shape
    x = torch.randn(shape, generator=gen, device="cuda")
    x *= torch.exp(0.3 * torch.randn((1, h, 1, 1), generator=gen, device="cuda"))
    x *= 1 + 3 * (torch.rand((1, h, 1, d), generator=gen, device="cuda") < 0.02)
    return x.to(dtype)


def _laid(x, layout):
    """(batch, heads, rows, dim) as it is, or as a view of (batch, rows, heads, dim)."""
    return x if layout == "heads" else x.transpose(1, 2).contiguous().transpose(1, 2)


def _counts(gen, batch, n):
    """Lengths between half of n and n, their mean three quarters of it."""
    low = (n + 1) // 2
    return torch.randint(low, n + 1, (batch,), generator=gen, device="cuda", dtype=torch.int32)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    if case["op"] in ("attend", "grad"):
        return _prepare_attend(case, gen)
    return _prepare_cache(case, gen)


def _prepare_attend(case, gen):
    b, q, h, hs, n, d = (case[x] for x in ("batch", "q", "heads", "state_heads", "n", "dim"))
    dtype = TYPES[case["dtype"]]
    s = {"op": case["op"], "counts": None, "mask": None, "scale": d ** -0.5}
    s["queries"] = _laid(_normal(gen, (b, h, q, d), dtype, 1.5), case["layout"])
    s["keys"] = _laid(_states(gen, (b, hs, n, d), dtype), case["layout"])
    s["values"] = _laid(_states(gen, (b, hs, n, d), dtype), case["layout"])
    if case["masked"] == "counts":
        s["counts"] = _counts(gen, b, n)
    if case["masked"] == "mask":
        s["mask"] = torch.rand((b, n), generator=gen, device="cuda") < 0.75
        if b > 1:
            s["mask"][b // 2] = False
    if case["op"] == "grad":
        # what the forward pass left behind, and the gradient that arrives
        s["out"], s["lse"] = _plain_attend(s)
        s["grad_out"] = _laid(_normal(gen, (b, h, q, d), dtype), case["layout"])
    return s


def _prepare_cache(case, gen):
    b, q, h, hs, n, d, block = (case[x] for x in ("batch", "q", "heads", "state_heads", "n", "dim", "block"))
    dtype = TYPES[case["dtype"]]
    slots = -(-n // block)
    blocks = b * slots
    s = {"op": case["op"], "block": block, "scale": d ** -0.5, "counts": None}
    if case["table"] != "full":
        s["counts"] = _counts(gen, b, n)
    s["table"] = torch.randperm(blocks, generator=gen, device="cuda").to(torch.int32).view(b, slots)
    cache = {
        "key_codes": torch.zeros((blocks, hs, block, d), dtype=torch.uint8, device="cuda"),
        "value_codes": torch.zeros((blocks, hs, block, d), dtype=torch.uint8, device="cuda"),
        "key_scales": torch.ones((blocks, hs), dtype=torch.float32, device="cuda"),
        "value_scales": torch.ones((blocks, hs), dtype=torch.float32, device="cuda"),
        "block_counts": torch.zeros(blocks, dtype=torch.int32, device="cuda"),
    }
    s["cache"] = cache
    if case["op"] == "store":
        s["keys"] = _states(gen, (b, hs, n, d), dtype)
        s["values"] = _states(gen, (b, hs, n, d), dtype)
        return s
    s["queries"] = _normal(gen, (b, h, q, d), dtype, 1.5)
    # the cache's content, written block by block as the states would have been
    for name in ("key", "value"):
        x = _states(gen, (blocks, hs, block, d), torch.float32)
        scales = _power_of_two(x.abs().amax((2, 3)))
        cache[name + "_codes"].copy_((x / scales[..., None, None]).to(torch.float8_e4m3fn).view(torch.uint8))
        cache[name + "_scales"].copy_(scales)
    cache["block_counts"].fill_(block)
    if case["table"] == "found":
        # blocks that a search named: any block, some of them not full, one entry in ten names none
        cache["block_counts"].sub_(torch.randint(0, 3, (blocks,), generator=gen, device="cuda", dtype=torch.int32))
        found = torch.randint(0, blocks, (b, slots), generator=gen, device="cuda", dtype=torch.int32)
        none = torch.rand((b, slots), generator=gen, device="cuda") < 0.1
        s["table"] = torch.where(none, torch.full_like(found, 2 ** 31 - 1), found)
        s["counts"] = None
    return s


# ---- one pass ------------------------------------------------------------------------------------


def run(s):
    if own:
        return _library(s)
    if s["op"] == "attend":
        out, lse = _plain_attend(s)
        return {"out": out, "lse": lse}
    if s["op"] == "grad":
        return _plain_grad(s)
    if s["op"] == "store":
        return _plain_store(s)
    return _plain_cached(s)


def _library(s):
    bitsknn = _bitsknn()
    if s["op"] == "attend":
        out, lse = bitsknn.cross_attention(s["queries"], s["keys"], s["values"], counts=s["counts"], mask=s["mask"],
                                           scale=s["scale"])
        return {"out": out, "lse": lse}
    if s["op"] == "grad":
        dq, dk, dv = bitsknn.cross_attention_backward(s["grad_out"], s["queries"], s["keys"], s["values"], s["out"],
                                                      s["lse"], counts=s["counts"], mask=s["mask"], scale=s["scale"])
        return {"queries": dq, "keys": dk, "values": dv}
    cache = bitsknn.StateCache(**s["cache"])
    if s["op"] == "store":
        bitsknn.cache_store(cache, s["keys"], s["values"], s["table"], counts=s["counts"])
        return _cache_values(s["cache"])
    out, lse = bitsknn.cached_attention(s["queries"], cache, s["table"], counts=s["counts"], scale=s["scale"])
    return {"out": out, "lse": lse}


def _bitsknn():
    package = os.path.join(ROOT, "bits-knn-jpdc2024_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    import bitsknn
    return bitsknn


def _cache_values(cache):
    """The cache with its codes as the numbers that they stand for (times their block's scale)."""
    return {
        "key_codes": cache["key_codes"].view(torch.float8_e4m3fn),
        "value_codes": cache["value_codes"].view(torch.float8_e4m3fn),
        "key_scales": cache["key_scales"],
        "value_scales": cache["value_scales"],
        "block_counts": cache["block_counts"],
    }


# ---- the plain forms, in 32 bits -------------------------------------------------------------------


def _power_of_two(amax):
    """The smallest power of two that is at least amax / 448, and at least 2^-126."""
    mantissa, exponent = torch.frexp(amax / E4M3_MAX)
    exponent = torch.where(mantissa == 0.5, exponent - 1, exponent)
    exponent = torch.where(amax > 0, exponent, torch.full_like(exponent, -126)).clamp_min(-126)
    return torch.ldexp(torch.ones_like(amax), exponent)


def _valid(s, batch, n, device):
    valid = torch.ones((batch, n), dtype=torch.bool, device=device)
    if s.get("counts") is not None:
        valid = valid & (torch.arange(n, device=device)[None] < s["counts"][:, None])
    if s.get("mask") is not None:
        valid = valid & s["mask"]
    return valid


def _grouped(x, state_heads):
    """(batch, heads, rows, dim) -> (batch, state heads, rows of all heads that share them, dim), 32 bits"""
    b, h, rows, d = x.shape
    return x.float().reshape(b, state_heads, h // state_heads * rows, d)


def _softmax_product(q, k, v, valid, scale):
    """q (b, hs, m, d) over k, v (b, hs, n, d) where valid (b, n): the weighted sum and the log-sum-exp."""
    gone = ~valid[:, None, None, :]
    v = v.masked_fill(gone.transpose(2, 3), 0.0)
    scores = torch.matmul(q, k.transpose(2, 3)).mul_(scale).masked_fill_(gone, -math.inf)
    top = scores.amax(-1, keepdim=True)
    base = torch.where(top == -math.inf, torch.zeros_like(top), top)
    weights = scores.sub_(base).exp_()
    total = weights.sum(-1, keepdim=True)
    out = torch.matmul(weights, v) / torch.where(total > 0, total, torch.ones_like(total))
    return out, (base + total.log()).squeeze(-1)


def _plain_attend(s):
    b, h, rows, d = s["queries"].shape
    hs, n = s["keys"].shape[1:3]
    out, lse = _softmax_product(_grouped(s["queries"], hs), s["keys"].float(), s["values"].float(),
                                _valid(s, b, n, s["keys"].device), s["scale"])
    return out.reshape(b, h, rows, d).to(s["queries"].dtype), lse.reshape(b, h, rows)


def _plain_grad(s):
    b, h, rows, d = s["queries"].shape
    hs, n = s["keys"].shape[1:3]
    gone = ~_valid(s, b, n, s["keys"].device)[:, None, None, :]
    q, grad_out, out = (_grouped(s[name], hs) for name in ("queries", "grad_out", "out"))
    k = s["keys"].float().masked_fill(gone.transpose(2, 3), 0.0)
    v = s["values"].float().masked_fill(gone.transpose(2, 3), 0.0)
    lse = s["lse"].reshape(b, hs, -1, 1)
    weights = torch.matmul(q, k.transpose(2, 3)).mul_(s["scale"]).sub_(lse).exp_().masked_fill_(gone, 0.0)
    grad_v = torch.matmul(weights.transpose(2, 3), grad_out)
    delta = (grad_out * out).sum(-1, keepdim=True)
    grad_s = torch.matmul(grad_out, v.transpose(2, 3)).sub_(delta).mul_(weights).mul_(s["scale"])
    grad_q = torch.matmul(grad_s, k).reshape(b, h, rows, d)
    grad_k = torch.matmul(grad_s.transpose(2, 3), q)
    dtype = s["queries"].dtype
    return {"queries": grad_q.to(dtype), "keys": grad_k.to(dtype), "values": grad_v.to(dtype)}


def _plain_store(s):
    cache, table, block = s["cache"], s["table"].long(), s["block"]
    b, hs, n, d = s["keys"].shape
    slots = table.shape[1]
    valid = _valid(s, b, n, table.device)
    valid = torch.nn.functional.pad(valid, (0, slots * block - n)).view(b, slots, block)
    used = valid[:, :, 0]  # the blocks that hold a state at all
    names = table[used]
    for name in ("key", "value"):
        x = torch.nn.functional.pad(s[name + "s"].float(), (0, 0, 0, slots * block - n))
        x = x.view(b, hs, slots, block, d).transpose(1, 2)
        inside = valid[:, :, None, :, None]
        x = x.masked_fill(~inside, 0.0)
        scales = _power_of_two(x.abs().amax((3, 4)))
        codes = (x / scales[..., None, None]).to(torch.float8_e4m3fn).view(torch.uint8)
        codes = torch.where(inside, codes, cache[name + "_codes"][table])
        cache[name + "_codes"][names] = codes[used]
        cache[name + "_scales"][names] = scales[used]
    cache["block_counts"][names] = valid.sum(-1, dtype=torch.int32)[used]
    return _cache_values(cache)


def _plain_cached(s):
    cache, table, block = s["cache"], s["table"], s["block"]
    b, h, rows, d = s["queries"].shape
    blocks, hs = cache["key_scales"].shape
    slots = table.shape[1]
    there = (table >= 0) & (table < blocks)
    names = torch.where(there, table, torch.zeros_like(table)).long()
    held = torch.where(there, cache["block_counts"][names], torch.zeros_like(table))
    valid = torch.arange(block, device=table.device)[None, None] < held[:, :, None]
    valid = valid.view(b, slots * block) & _valid(s, b, slots * block, table.device)
    states = []
    for name in ("key", "value"):
        x = cache[name + "_codes"][names].view(torch.float8_e4m3fn).float()
        x = x * cache[name + "_scales"][names][..., None, None]
        states.append(x.transpose(1, 2).reshape(b, hs, slots * block, d))
    out, lse = _softmax_product(_grouped(s["queries"], hs), states[0], states[1], valid, s["scale"])
    return {"out": out.reshape(b, h, rows, d).to(s["queries"].dtype), "lse": lse.reshape(b, h, rows)}


# ---- the definitions in 64 bits --------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] == "store":
        return _exact_store(s)
    parts = []
    for b in range(case["batch"]):
        if s["op"] == "cached":
            keys, values = _exact_cached_states(s, b)
        else:
            take = torch.arange(case["n"], device="cuda")
            if s["counts"] is not None:
                take = take[: int(s["counts"][b])]
            if s["mask"] is not None:
                take = take[s["mask"][b][take]]
            keys, values = s["keys"][b].double()[:, take], s["values"][b].double()[:, take]
        share = case["heads"] // case["state_heads"]
        keys, values = (x.repeat_interleave(share, 0) for x in (keys, values))
        q = s["queries"][b].double()
        scores = torch.bmm(q, keys.mT.contiguous()) * s["scale"]
        if s["op"] != "grad":
            weights = torch.softmax(scores, -1)
            parts.append((torch.bmm(weights, values), torch.logsumexp(scores, -1)))
            continue
        grad_out = s["grad_out"][b].double()
        weights = torch.exp(scores - s["lse"][b].double()[..., None])
        slope = torch.bmm(grad_out, values.mT.contiguous())
        slope = weights * (slope - (grad_out * s["out"][b].double()).sum(-1, keepdim=True)) * s["scale"]
        hs, n, d = s["keys"].shape[1:]
        grads = [torch.bmm(slope, keys)]
        for x, y in ((slope, q), (weights, grad_out)):
            one = torch.zeros((hs, n, d), dtype=torch.float64, device="cuda")
            one[:, take] = torch.bmm(x.mT.contiguous(), y).view(hs, share, len(take), d).sum(1)
            grads.append(one)
        parts.append(tuple(grads))
    names = ("queries", "keys", "values") if s["op"] == "grad" else ("out", "lse")
    return {name: torch.stack(column) for name, column in zip(names, zip(*parts))}


def _exact_cached_states(s, b):
    cache, picked = s["cache"], [[], []]
    held_by = cache["block_counts"].tolist()
    left = s["table"].shape[1] * s["block"] if s["counts"] is None else int(s["counts"][b])
    for name in s["table"][b].tolist():
        if 0 <= name < len(held_by) and left > 0:
            held = min(left, held_by[name])
            for one, kind in zip(picked, ("key", "value")):
                codes = cache[kind + "_codes"][name, :, :held].view(torch.float8_e4m3fn).double()
                one.append(codes * cache[kind + "_scales"][name].double()[:, None, None])
        left -= s["block"]
    empty = torch.zeros((cache["key_codes"].shape[1], 0, cache["key_codes"].shape[3]), dtype=torch.float64,
                        device="cuda")
    return [torch.cat([empty] + one, 1) for one in picked]


def _exact_store(s):
    blocks, hs, block, d = s["cache"]["key_codes"].shape
    b, slots = s["table"].shape
    n = s["keys"].shape[2]
    counts = [n] * b if s["counts"] is None else s["counts"].tolist()
    result = {}
    for kind in ("key", "value"):
        codes = torch.zeros((blocks, hs, block, d), dtype=torch.float64, device="cuda")
        scales = torch.ones((blocks, hs), dtype=torch.float64, device="cuda")
        for i in range(b):
            for slot, name in enumerate(s["table"][i].tolist()):
                x = s[kind + "s"][i, :, slot * block:min(counts[i], (slot + 1) * block)].double()
                if x.shape[1] <= 0:
                    break
                # frexp: top = mantissa 2^exponent with the mantissa in [1/2, 1)
                mantissa, exponent = torch.frexp((x.abs().amax((1, 2)) / E4M3_MAX).clamp_min(2.0 ** -126))
                power = torch.exp2(exponent.double() - (mantissa == 0.5).double())
                x = x / power[:, None, None]
                step = torch.exp2(torch.frexp(x.abs().clamp_min(2.0 ** -6))[1].double() - 4)
                codes[name, :, : x.shape[1]] = torch.round(x / step) * step
                scales[name] = power
        result[kind + "_codes"], result[kind + "_scales"] = codes, scales
    result["block_counts"] = None
    return result
