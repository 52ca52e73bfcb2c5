"""Operators over a key/value cache held in 8 bits with one scale per block of tokens and head, as cases that can be timed and compared.

* ``append``: a step's keys and values are quantized into the cache (`swlm_op_kv8_append_dev`).
* ``attend``: attention of a step's queries over the cache, with or without each cached token's weight added to its running sum
  (`swlm_op_kv8_attend_dev`).
* ``evict``: the tokens that keep their place in a smaller cache, by accumulated weight (`swlm_op_kv8_evict_dev`).

A cached value is code * scale, the code an int8 of -127..127 or an e4m3 number. `run` returns codes as they are held beside the
scales; together they are the values. Head layouts are those of the framework's own configurations (32 query and 8 KV heads of 128 or
64) and generic ones; a step's tokens lie one after the other, `starts` says where each sequence's begin.
"""
import math

import torch

own = False

INT8, E4M3 = "int8", "e4m3"
TOP = {INT8: 127.0, E4M3: 448.0}
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    llama = {"heads": 32, "kv_heads": 8, "head_dim": 128, "code": INT8, "block": 64, "dtype": "bf16"}
    small = {"heads": 32, "kv_heads": 8, "head_dim": 64, "code": E4M3, "block": 32, "dtype": "fp16"}
    return [
        # the token of one decoding user: the smallest call, its block partly filled
        {"name": "append_1x1", "kind": "append", "batch": 1, "tokens": 1, "context": 2047, "ragged": False, **llama},
        # a serving batch's step, every sequence at its own place
        {"name": "append_48x1_ragged", "kind": "append", "batch": 48, "tokens": 1, "context": 1531, "ragged": True, **small},
        # portions of four prompts of unequal length
        {"name": "append_4x2048_ragged", "kind": "append", "batch": 4, "tokens": 2048, "context": 1000, "ragged": True, **llama, "block": 128},
        # one user, a short context: latency
        {"name": "attend_1x1000", "kind": "attend", "batch": 1, "tokens": 1, "context": 1000, "ragged": False, "weights": False, **llama},
        # a serving batch with long contexts whose tokens' weights are kept for eviction
        {"name": "attend_8x8192_weights", "kind": "attend", "batch": 8, "tokens": 1, "context": 8192, "ragged": False, "weights": True, **llama},
        # a larger batch of no round size, lengths from all of the context to a quarter, small heads
        {"name": "attend_41x4091_ragged", "kind": "attend", "batch": 41, "tokens": 1, "context": 4091, "ragged": True, "weights": False, **small},
        # one user with a very long document
        {"name": "attend_1x131071_weights", "kind": "attend", "batch": 1, "tokens": 1, "context": 131071, "ragged": False, "weights": True, **llama, "block": 128},
        # five drafted tokens per sequence, to be checked together
        {"name": "attend_6x5_over_16384", "kind": "attend", "batch": 6, "tokens": 5, "context": 16384, "ragged": True, "weights": False, **llama, "block": 16},
        # a portion of a long prompt
        {"name": "attend_prompt_2048_over_8192", "kind": "attend", "batch": 1, "tokens": 2048, "context": 6144, "ragged": False, "weights": False, **llama},
        # portions of three prompts, weights kept from the first token on
        {"name": "attend_prompt_3x777_weights", "kind": "attend", "batch": 3, "tokens": 777, "context": 2100, "ragged": True, "weights": True, **small},
        # a bounded cache that has run over by 256 tokens since its last eviction
        {"name": "evict_1x4352_to_4096", "kind": "evict", "batch": 1, "context": 4352, "keep": 4096, "ragged": False, "mixed": True, **llama},
        # four prompts brought down to a small cache each
        {"name": "evict_4x32768_to_4096", "kind": "evict", "batch": 4, "context": 32768, "keep": 4096, "ragged": True, "mixed": False, **llama, "block": 32},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kv_heads = rng.choice([1, 2, 4, 8])
    case = {"kind": rng.choice(["append", "attend", "attend", "attend", "evict"]), "heads": kv_heads * rng.choice([1, 2, 4, 4, 7, 8]), "kv_heads": kv_heads,
            "head_dim": rng.choice([64, 128]), "code": rng.choice([INT8, E4M3]), "block": rng.choice([16, 32, 64, 128]), "dtype": rng.choice(["bf16", "fp16"]),
            "ragged": rng.random() < 0.6}
    batch = case["batch"] = _log(rng, 1, 48)
    if case["kind"] == "append":
        return {**case, "tokens": rng.choice([1, _log(rng, 1, max(1, 8192 // batch))]), "context": _log(rng, 1, 8192)}
    if case["kind"] == "evict":
        context = max(64, min(32768, _log(rng, 256, 131072) // batch + rng.randrange(64)))
        return {**case, "context": context, "keep": max(8, min(context, 131072 // batch, _log(rng, context / 16 + 1, context))), "mixed": rng.random() < 0.5}
    case["weights"] = rng.random() < 0.5
    how = rng.choice(["one", "one", "few", "portion"])
    if how == "portion":
        batch = case["batch"] = _log(rng, 1, 4)
        return {**case, "tokens": _log(rng, 17, (2048 if case["heads"] <= 32 else 1024) // batch), "context": _log(rng, 1, 4096)}
    return {**case, "tokens": 1 if how == "one" else rng.randint(2, 16), "context": max(1, _log(rng, 64, 131072) // batch + rng.randrange(64))}


# ---- inputs ------------------------------------------------------------------------------------------------------------

def _generator(seed, salt):
    return torch.Generator(device="cuda").manual_seed((seed * 1000003 + salt) & 0x7FFFFFFF)


def _lengths(case):
    """Tokens in the cache of each sequence before the step: all alike, or from the whole context down to a quarter of it."""
    b, context = case["batch"], case["context"]
    return [max(1, round(context * (1.0 - 0.75 * i / max(1, b - 1)))) if case["ragged"] else context for i in range(b)]


def _counts(case):
    """Tokens of the step of each sequence: all alike, or up to half of them missing."""
    b, n = case["batch"], case.get("tokens", 0)
    return [max(1, n - (i * 5 * n // (8 * b)) if n > 1 else 1) if case["ragged"] else n for i in range(b)]


def _seen(case):
    """Position of the next token of each sequence of an eviction."""
    return [case["context"]] * case["batch"] if case["mixed"] else _lengths(case)


def _capacity(case):
    return (case["context"] + case.get("tokens", 0)) // case["block"] * case["block"] + 2 * case["block"]


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _codes(case, shape, generator):
    """Codes of one cache, their spread a quarter of the range, as in a block whose largest value is four deviations out."""
    out = torch.empty(shape, dtype=torch.int8 if case["code"] == INT8 else torch.float8_e4m3fn, device="cuda")
    for b in range(shape[0]):
        x = torch.randn(shape[1:], generator=generator, device="cuda") * (TOP[case["code"]] / 4)
        out[b] = (x.round() if case["code"] == INT8 else x).clamp(-TOP[case["code"]], TOP[case["code"]]).to(out.dtype)
    return out


def _cache(case, seed):
    b, h, d, cap, t = case["batch"], case["kv_heads"], case["head_dim"], _capacity(case), case["block"]
    g = _generator(seed, 1)
    cache = {"k": _codes(case, (b, h, cap, d), g), "v": _codes(case, (b, h, cap, d), g)}
    unit = 4.0 / TOP[case["code"]]   # keys of deviation 2 (attention is not a plain mean), values of deviation 1; blocks differ by some tenths
    cache["k_scale"] = 2.0 * unit * torch.exp(0.2 * torch.randn((b, h, cap // t), generator=g, device="cuda"))
    cache["v_scale"] = unit * torch.exp(0.3 * torch.randn((b, h, cap // t), generator=g, device="cuda"))
    # attention weights are far from even: most tokens were hardly looked at
    cache["weight"] = torch.exp(2.0 * torch.randn((b, h, cap), generator=g, device="cuda"))
    cache["slot_pos"] = torch.arange(cap, dtype=torch.int32, device="cuda").expand(b, h, cap).contiguous()
    if case.get("mixed"):   # slots that earlier evictions have filled out of order, each head on its own
        n = case["context"]
        cache["slot_pos"][:, :, :n] = torch.rand((b, h, n), generator=g, device="cuda").argsort(dim=-1).int()
    return cache


def _rows(case, seed, salt, heads, spread=1.0):
    return (spread * torch.randn((sum(_counts(case)), heads, case["head_dim"]), generator=_generator(seed, salt), device="cuda")).to(DTYPES[case["dtype"]])


def prepare(case, seed):
    state = {"case": case, "cache": _cache(case, seed), "lengths": _ints(_lengths(case)), "counts": _ints(_counts(case)),
             "starts": _ints([sum(_counts(case)[:i]) for i in range(case["batch"])])}
    cache = state["cache"]
    if case["kind"] == "append":
        state["k"], state["v"] = _rows(case, seed, 2, case["kv_heads"], 2.0), _rows(case, seed, 3, case["kv_heads"])
        state["seen"] = state["lengths"] + 5   # sequences that have lost five tokens to an eviction
    elif case["kind"] == "attend":
        state["q"] = _rows(case, seed, 4, case["heads"])
        state["out"] = torch.zeros_like(state["q"])
        state["before"] = cache["weight"].clone()
    else:
        t = case["block"]
        capacity = (case["keep"] + 2 * t - 1) // t * t
        state["seen"] = _ints(_seen(case))
        state["kept"] = {name: torch.zeros((*x.shape[:2], capacity // t if name.endswith("scale") else capacity, *x.shape[3:]), device="cuda").to(x.dtype)
                         for name, x in cache.items()}
    if own:
        _prepare_own(state)
    torch.cuda.synchronize()
    return state


# ---- the framework's calls ----------------------------------------------------------------------------------------------

def _context():
    """The package and the context of the device: a program makes them once."""
    if not hasattr(_context, "made"):
        import __graft_entry__
        pkg = __graft_entry__.load_package()
        _context.made = pkg, pkg.WeightStore(0)
    return _context.made


def _prepare_own(state):
    _context()
    if state["case"]["kind"] == "append":
        _hold_last_blocks(state)


def _hold_last_blocks(state):
    """Codes and scales of the blocks that sequences end in, which an append may scale anew: every pass finds them as they were before the step. The cache
    lies in one allocation of words, so that one copy brings them back."""
    case, cache = state["case"], state["cache"]
    b, h, cap, d = cache["k"].shape
    t, codes, scales = case["block"], cache["k"].numel() // 4, cache["k_scale"].numel()
    state["words"] = words = torch.cat([cache[x].reshape(-1).view(torch.int32) for x in ("k", "v", "k_scale", "v_scale")])
    for x, part in zip(("k", "v", "k_scale", "v_scale"), words.split([codes, codes, scales, scales])):
        cache[x] = part.view(cache[x].dtype).view(cache[x].shape)
    head = torch.arange(b * h, device="cuda")
    block = (state["lengths"].long() // t).repeat_interleave(h)
    of_codes = ((head * cap + block * t)[:, None] * (d // 4) + torch.arange(t * d // 4, device="cuda")).reshape(-1)
    of_scales = 2 * codes + head * (cap // t) + block
    state["last"] = torch.cat([of_codes, of_codes + codes, of_scales, of_scales + scales])
    state["held"] = words[state["last"]]


def _described(pkg, case, cache):
    return pkg.Kv8Cache(k=cache["k"].data_ptr(), v=cache["v"].data_ptr(), k_scale=cache["k_scale"].data_ptr(), v_scale=cache["v_scale"].data_ptr(),
                        weight=cache["weight"].data_ptr(), slot_pos=cache["slot_pos"].data_ptr(), batch=case["batch"], kv_heads=case["kv_heads"],
                        head_dim=case["head_dim"], capacity=cache["k"].shape[2], block=case["block"],
                        code=pkg.KV8_INT8 if case["code"] == INT8 else pkg.KV8_E4M3)


def _run_own(state):
    pkg, store = _context()
    # (a null stream stands for the context's own; 1 is CUDA's handle of the default stream that torch works on)
    lib, handle, stream = store.lib, store.handle, torch.cuda.current_stream().cuda_stream or 1
    case, cache = state["case"], state["cache"]
    if case["kind"] == "append":
        state["words"].index_copy_(0, state["last"], state["held"])
    described, lengths = _described(pkg, case, cache), state["lengths"].data_ptr()
    if case["kind"] == "append":
        stride = case["kv_heads"] * case["head_dim"]
        call = pkg.Kv8Append(k=state["k"].data_ptr(), v=state["v"].data_ptr(), k_stride=stride, v_stride=stride, lengths=lengths, counts=state["counts"].data_ptr(),
                             starts=state["starts"].data_ptr(), seen=state["seen"].data_ptr(), dtype=pkg.KV8_BF16 if case["dtype"] == "bf16" else pkg.KV8_FP16,
                             n=case["tokens"], rows=state["k"].shape[0])
        lib.check(lib.swlm_op_kv8_append_dev(handle, described, call, stream))
    elif case["kind"] == "attend":
        stride = case["heads"] * case["head_dim"]
        call = pkg.Kv8Attend(q=state["q"].data_ptr(), out=state["out"].data_ptr(), q_stride=stride, out_stride=stride, lengths=lengths,
                             counts=state["counts"].data_ptr(), starts=state["starts"].data_ptr(), scale=case["head_dim"] ** -0.5,
                             dtype=pkg.KV8_BF16 if case["dtype"] == "bf16" else pkg.KV8_FP16, heads=case["heads"], n=case["tokens"],
                             rows=state["q"].shape[0], max_len=case["context"] + case["tokens"], accumulate=int(case["weights"]))
        call.scratch_bytes = lib.swlm_op_kv8_attend_scratch_bytes(described, call)
        scratch = torch.empty(max(16, call.scratch_bytes), dtype=torch.uint8, device="cuda")
        call.scratch = scratch.data_ptr()
        lib.check(lib.swlm_op_kv8_attend_dev(handle, described, call, stream))
    else:
        call = pkg.Kv8Evict(lengths=lengths, seen=state["seen"].data_ptr(), keep=case["keep"], sink=min(4, case["keep"] // 4),
                            recent=min(32, case["keep"] // 4), max_len=case["context"])
        call.scratch_bytes = lib.swlm_op_kv8_evict_scratch_bytes(described, call)
        scratch = torch.empty(max(16, call.scratch_bytes), dtype=torch.uint8, device="cuda")
        call.scratch = scratch.data_ptr()
        lib.check(lib.swlm_op_kv8_evict_dev(handle, described, _described(pkg, case, state["kept"]), call, stream))


def run(state):
    case, cache = state["case"], state["cache"]
    if case["kind"] == "attend" and case["weights"]:
        cache["weight"].copy_(state["before"])   # every pass adds to the sums as they were before the step
    if own:
        _run_own(state)
    else:
        {"append": _plain_append, "attend": _plain_attend, "evict": _plain_evict}[case["kind"]](state)
    if case["kind"] == "attend":
        return {"out": state["out"], "weight": cache["weight"]} if case["weights"] else {"out": state["out"]}
    return dict(cache if case["kind"] == "append" else state["kept"])


# ---- the plain forms ----------------------------------------------------------------------------------------------------

def _to_codes(x, code):
    """The nearest code of each value x, given in units of its block's scale."""
    return (x.round() if code == INT8 else x).clamp(-TOP[code], TOP[code]).to(torch.int8 if code == INT8 else torch.float8_e4m3fn)


def _bits(x):
    return x.view(torch.int8)   # (one byte either way; gathers and scatters move bytes)


def _per_slot(scale, block):
    return scale.repeat_interleave(block, dim=2)


def _plain_append(state):
    """The blocks that the step touches, from each sequence's last one on, as a window of the cache."""
    case, cache = state["case"], state["cache"]
    t, code, b, h, d = case["block"], case["code"], case["batch"], case["kv_heads"], case["head_dim"]
    lengths, counts = state["lengths"].long(), state["counts"].long()
    blocks = (case["tokens"] + t - 2) // t + 1
    first = lengths // t
    slot = first[:, None] * t + torch.arange(blocks * t, device="cuda")
    at_block = first[:, None] + torch.arange(blocks, device="cuda")
    old, new = slot < lengths[:, None], (slot >= lengths[:, None]) & (slot < (lengths + counts)[:, None])
    row = (state["starts"].long()[:, None] + slot - lengths[:, None]).clamp(0, state["k"].shape[0] - 1)
    top = torch.tensor(TOP[code], device="cuda")
    at = slot[:, None, :, None].expand(b, h, -1, d)
    at_scale = at_block[:, None, :].expand(b, h, -1)
    has_old, touched = old.view(b, 1, blocks, t).any(dim=3), new.view(b, 1, blocks, t).any(dim=3)
    for name in ("k", "v"):
        x = torch.where(new[:, None, :, None], state[name][row].transpose(1, 2).float(), 0.0)
        held = _bits(cache[name]).gather(2, at)
        before = cache[name + "_scale"].gather(2, at_scale)
        s0 = torch.where(has_old, before, 0.0)
        s = torch.maximum(s0, x.abs().reshape(b, h, blocks, t * d).amax(dim=3) / top)
        each = _per_slot(s, t)[..., None]
        value = torch.where(old[:, None, :, None], held.view(cache[name].dtype).float() * _per_slot(s0, t)[..., None], x)
        codes = _bits(_to_codes(torch.where(each > 0, value / each, 0.0), code))
        keep = (old | new)[:, None, :, None] & _per_slot(touched, t)[..., None]
        _bits(cache[name]).scatter_(2, at, torch.where(keep, codes, held))
        cache[name + "_scale"].scatter_(2, at_scale, torch.where(touched, s, before))
    at = slot[:, None, :].expand(b, h, -1)
    position = (state["seen"].long()[:, None] + slot - lengths[:, None]).int()
    cache["slot_pos"].scatter_(2, at, torch.where(new[:, None, :], position[:, None, :], cache["slot_pos"].gather(2, at)))
    cache["weight"].scatter_(2, at, torch.where(new[:, None, :], 0.0, cache["weight"].gather(2, at)))


def _places(state):
    """Row of query i of sequence b in the step's arrays [b, i], and whether there is one."""
    i = torch.arange(state["case"]["tokens"], device="cuda")
    valid = i < state["counts"][:, None]
    return torch.where(valid, state["starts"].long()[:, None] + i, state["q"].shape[0]), valid


def _plain_attend(state):
    case, cache = state["case"], state["cache"]
    t, b, h, d, n = case["block"], case["batch"], case["kv_heads"], case["head_dim"], case["tokens"]
    group, rows, span = case["heads"] // h, state["q"].shape[0], case["context"] + n
    row, valid = _places(state)
    q = state["q"][row.clamp(max=rows - 1)].float().view(b, n, h, group, d).permute(0, 2, 1, 3, 4).reshape(b, h, n * group, d)
    s = q @ (cache["k"][:, :, :span].float() * _per_slot(cache["k_scale"], t)[:, :, :span, None]).transpose(2, 3)
    limit = state["lengths"][:, None] + torch.arange(n, device="cuda") + 1
    seen = (torch.arange(span, device="cuda") < limit[:, :, None]) & valid[:, :, None]
    s = (s * d ** -0.5).view(b, h, n, group, span).masked_fill_(~seen[:, None, :, None, :], -math.inf)
    top = s.amax(dim=-1, keepdim=True)
    p = s.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    p /= p.sum(dim=-1, keepdim=True).clamp(min=1e-30)
    o = p.view(b, h, n * group, span) @ (cache["v"][:, :, :span].float() * _per_slot(cache["v_scale"], t)[:, :, :span, None])
    o = o.view(b, h, n, group, d).permute(0, 2, 1, 3, 4).reshape(b * n, h * group, d)
    out = torch.cat([state["out"], state["out"][:1]])
    out[row.reshape(-1)] = o.to(out.dtype)   # (places without a query go to a row of their own)
    state["out"].copy_(out[:rows])
    if case["weights"]:
        cache["weight"][:, :, :span] += p.sum(dim=(2, 3))


def _plain_evict(state):
    case, cache, kept = state["case"], state["cache"], state["kept"]
    t, code, keep, b, h, d = case["block"], case["code"], case["keep"], case["batch"], case["kv_heads"], case["head_dim"]
    span, top = case["context"], torch.tensor(TOP[case["code"]], device="cuda")
    lengths, seen = state["lengths"].long()[:, None, None], state["seen"].long()[:, None, None]
    slot = torch.arange(span, device="cuda")
    position = cache["slot_pos"][:, :, :span]
    key = cache["weight"][:, :, :span].clone()
    key = torch.where((position < min(4, keep // 4)) | (position >= seen - min(32, keep // 4)), math.inf, key)
    key = torch.where(slot < lengths, key, -math.inf)
    chosen = torch.zeros_like(key, dtype=torch.bool).scatter_(2, key.sort(dim=2, descending=True, stable=True).indices[:, :, :keep], True)
    # the i-th free slot below `keep` takes the i-th chosen one from `keep` on
    free, moves = ~chosen[:, :, :keep], chosen.clone()
    moves[:, :, :keep] = False
    moved = moves.float().sort(dim=2, descending=True, stable=True).indices
    source = torch.where(free, moved.gather(2, (free.long().cumsum(dim=2) - 1).clamp(min=0)), slot[:keep])
    valid = slot[:keep] < lengths
    changed = free & valid & (lengths > keep)
    source = torch.where(changed, source, slot[:keep])
    capacity = kept["k"].shape[2]
    pad = (keep + t - 1) // t * t
    wide = torch.nn.functional.pad
    changed = wide(changed, (0, pad - keep)).view(b, h, pad // t, t).any(dim=3)
    touched = wide(valid.expand(b, h, keep), (0, pad - keep)).view(b, h, pad // t, t).any(dim=3)
    whole = wide(valid.expand(b, h, keep), (0, pad - keep))
    source = wide(source, (0, pad - keep))
    for name in ("k", "v"):
        codes = _bits(cache[name]).gather(2, source[..., None].expand(b, h, pad, d))
        scale = cache[name + "_scale"].gather(2, source // t)
        value = torch.where(whole[..., None], codes.view(cache[name].dtype).float() * scale[..., None], 0.0)
        s = torch.where(changed, value.abs().view(b, h, pad // t, t * d).amax(dim=3) / top, cache[name + "_scale"][:, :, :pad // t])
        each = _per_slot(s, t)[..., None]
        new = _bits(_to_codes(torch.where(each > 0, value / each, 0.0), code))
        new = torch.where(_per_slot(changed, t)[..., None], new, codes)
        _bits(kept[name])[:, :, :pad] = torch.where(whole[..., None], new, _bits(kept[name])[:, :, :pad])
        kept[name + "_scale"][:, :, :pad // t] = torch.where(touched, s, kept[name + "_scale"][:, :, :pad // t])
    for name in ("weight", "slot_pos"):
        kept[name][:, :, :pad] = torch.where(whole, cache[name].gather(2, source), kept[name][:, :, :pad])


# ---- what it takes, and the values in 64 bits ------------------------------------------------------------------------------

def work(case):
    h, d, t, lengths, counts = case["kv_heads"], case["head_dim"], case["block"], _lengths(case), _counts(case)
    if case["kind"] == "append":
        n = sum(counts)
        return {"bytes": h * (n * (2 * d * 3 + 8) + 8.0 * sum(-(-c // t) for c in counts)), "flops": 4.0 * h * n * d}
    if case["kind"] == "attend":
        cached = sum(a + c for a, c in zip(lengths, counts))
        visible = sum(c * a + c * (c + 1) / 2 for a, c in zip(lengths, counts))
        return {"bytes": h * cached * (2 * d + 8 / t + (8 if case["weights"] else 0)) + 4.0 * sum(counts) * case["heads"] * d,
                "flops": 4.0 * case["heads"] * d * visible}
    kept = sum(min(a, case["keep"]) for a in lengths)
    return {"bytes": h * (8.0 * sum(lengths) + kept * (4 * d + 8) + 16 * kept / t), "flops": 4.0 * h * kept * d}


def _double_codes(x, code):
    """Values in units of their scale, rounded to the codes' numbers in 64 bits."""
    if code == INT8:
        return x.round().clamp(-127, 127)
    step = torch.exp2((torch.frexp(x).exponent - 1).clamp(min=-6).double() - 3)
    return ((x / step).round() * step).clamp(-448, 448)


def exact(case, seed):
    cache = _cache(case, seed)
    t, code, top, h, d = case["block"], case["code"], TOP[case["code"]], case["kv_heads"], case["head_dim"]
    lengths, counts = _lengths(case), _counts(case)
    if case["kind"] == "append":
        new = {"k": _rows(case, seed, 2, h, 2.0), "v": _rows(case, seed, 3, h)}
        result = {"k": cache["k"].double(), "v": cache["v"].double(), "k_scale": cache["k_scale"].double(), "v_scale": cache["v_scale"].double()}
        row = 0
        for b, (a, c) in enumerate(zip(lengths, counts)):
            for name in ("k", "v"):
                tokens = new[name][row:row + c].double().transpose(0, 1)
                for block in range(a // t, (a + c - 1) // t + 1):
                    low, mid, high = block * t, max(a, block * t), min(a + c, block * t + t)
                    fresh = tokens[:, mid - a:high - a]
                    held = result[name][b, :, low:mid] * result[name + "_scale"][b, :, block, None, None]
                    s = fresh.abs().amax(dim=(1, 2)) / top
                    s = s if mid == low else torch.maximum(s, result[name + "_scale"][b, :, block])
                    result[name][b, :, low:high] = _double_codes(torch.cat([held, fresh], dim=1) / s[:, None, None], code)
                    result[name + "_scale"][b, :, block] = s
            cache["weight"][b, :, a:a + c] = 0.0
            row += c
        return {**result, "weight": cache["weight"].double(), "slot_pos": None}
    if case["kind"] == "attend":
        group, out, weight = case["heads"] // h, [], cache["weight"].double()
        q = _rows(case, seed, 4, case["heads"]).double().split(counts)
        for b, (a, c) in enumerate(zip(lengths, counts)):
            mask = torch.arange(a + c, device="cuda")[None, :] > a + torch.arange(c, device="cuda")[:, None]
            o = torch.empty((c, case["heads"], d), dtype=torch.float64, device="cuda")
            for head in range(case["heads"]):
                kv = head // group
                k, v = (cache[x][b, kv, :a + c].double() * cache[x + "_scale"][b, kv].double().repeat_interleave(t)[:a + c, None] for x in "kv")
                p = torch.softmax((q[b][:, head] @ k.T / math.sqrt(d)).masked_fill(mask, -math.inf), dim=-1)
                o[:, head] = p @ v
                weight[b, kv, :a + c] += p.sum(dim=0)
            out.append(o)
        return {"out": torch.cat(out), "weight": weight} if case["weights"] else {"out": torch.cat(out)}
    keep = case["keep"]
    capacity = (keep + 2 * t - 1) // t * t
    shape = (case["batch"], h, capacity)
    result = {"k": torch.zeros((*shape, d), dtype=torch.float64, device="cuda"), "k_scale": torch.zeros((*shape[:2], capacity // t), dtype=torch.float64, device="cuda"),
              "weight": torch.zeros(shape, dtype=torch.float64, device="cuda"), "slot_pos": None}
    result["v"], result["v_scale"] = result["k"].clone(), result["k_scale"].clone()
    for b, a in enumerate(lengths):
        for head in range(h):
            position, weight = cache["slot_pos"][b, head, :a], cache["weight"][b, head, :a].double()
            source = torch.arange(min(a, keep), device="cuda")
            if a > keep:
                rank = torch.where((position < min(4, keep // 4)) | (position >= _seen(case)[b] - min(32, keep // 4)), math.inf, weight)
                order = torch.sort(rank, descending=True, stable=True).indices[:keep].sort().values
                stays, comes = order[order < keep], order[order >= keep]
                free = torch.ones(keep, dtype=torch.bool, device="cuda")
                free[stays] = False
                source[free] = comes
            n = source.numel()
            result["weight"][b, head, :n] = weight[source]
            new = (torch.arange(n, device="cuda") != source).double()
            pad = torch.nn.functional.pad
            blocks = -(-n // t)
            for x in "kv":
                codes = cache[x][b, head].double()[source]
                value = pad(codes * cache[x + "_scale"][b, head].double()[source // t, None], (0, 0, 0, blocks * t - n)).view(blocks, t, d)
                mixed = pad(new, (0, blocks * t - n)).view(blocks, t).amax(dim=1) > 0
                s = torch.where(mixed, value.abs().amax(dim=(1, 2)) / top, cache[x + "_scale"][b, head, :blocks].double())
                fresh = _double_codes(value / s[:, None, None], code).view(blocks * t, d)[:n]
                result[x][b, head, :n] = torch.where(mixed.repeat_interleave(t)[:n, None], fresh, codes)
                result[x + "_scale"][b, head, :blocks] = s
    return result
