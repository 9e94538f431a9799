"""The attention operators' work, as cases that can be timed and compared.

Kinds of case:
  store      keys and values of some tokens written into a cache, and the same tokens read back from it
  attention  queries of a batch over a prefix that rows share and over keys and values of their own

Token counts follow from an image size (64 x 64 latent tokens per 1024 x 1024 image at the 640-wide level, 32 x 32 at the
1280-wide one, heads of 64) and from prompts of 77 tokens or several times that; the cases of single tokens and of
shared key heads are generic. The plain forms are elementary torch operations in 32 bits.
"""
import importlib
import math

import torch

own = False

FP8_MAX = {"e4m3": 448.0, "e5m2": 57344.0}
FP8_TYPE = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}


def _store(name, slots, tokens, heads, dim, dtype, capacity, ragged=False):
    return {"name": name, "kind": "store", "slots": slots, "tokens": tokens, "heads": heads, "dim": dim, "dtype": dtype,
            "capacity": capacity, "ragged": ragged}


def _attention(name, batch, queries, q_heads, kv_heads, dim, dtype, prefixes, prefix, own_tokens, ragged=False, causal=False):
    return {"name": name, "kind": "attention", "batch": batch, "queries": queries, "q_heads": q_heads, "kv_heads": kv_heads,
            "dim": dim, "dtype": dtype, "prefixes": prefixes, "prefix": prefix, "own_tokens": own_tokens, "ragged": ragged,
            "causal": causal}


def listed():
    return [
        # K / V of one prompt pair for a block of the 640-wide level: the smallest write, all latency
        _store("store_prompt_int8", 2, 77, 10, 64, "int8", 77),
        # one new token for each of 64 sequences of unlike lengths
        _store("store_token_e4m3", 64, 1, 20, 64, "e4m3", 2048, ragged=True),
        # the tokens of three images of 39 x 39 latent tokens: odd counts
        _store("store_images_e5m2", 3, 1521, 10, 64, "e5m2", 1600),
        # sixteen images at 1024 x 1024: bandwidth
        _store("store_batch_int8", 16, 4096, 10, 64, "int8", 4096),
        # one query against one prompt: the smallest attention, all latency
        _attention("query_prompt_f16", 1, 1, 5, 5, 64, "f16", 1, 77, 0),
        # cross-attention of eight images that share a prompt pair, 640-wide level
        _attention("cross_640_f16", 16, 4096, 10, 10, 64, "f16", 2, 77, 0),
        # cross-attention at the 1280-wide level over a long prompt shared by four images, and 16 tokens of each image's own
        _attention("cross_1280_int8", 8, 1024, 20, 20, 64, "int8", 2, 231, 16),
        # self-attention of one image pair at the 640-wide level: the largest products
        _attention("self_640_f16", 2, 4096, 10, 10, 64, "f16", 0, 0, 4096),
        # self-attention of a portrait image pair at the 1280-wide level: 38 x 26 tokens
        _attention("self_1280_f16", 2, 988, 20, 20, 64, "f16", 0, 0, 988),
        # one token for each of 64 sequences behind one long prefix, own parts of unlike lengths
        _attention("decode_f16", 64, 1, 20, 20, 64, "f16", 1, 8192, 256, ragged=True),
        # the same with shared key heads, an 8-bit cache and a longer prefix
        _attention("decode_e4m3_shared_heads", 32, 1, 32, 8, 128, "e4m3", 1, 32768, 511, ragged=True),
        # a question of 333 tokens for each of four sequences behind a shared text, causal, heads of 80
        _attention("question_int8", 4, 333, 16, 8, 80, "int8", 1, 2000, 333, causal=True),
    ]


def _log_uniform(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    if rng.random() < 0.3:
        dtype = rng.choice(["int8", "e4m3", "e5m2", "f16"])
        heads, dim = rng.choice([(5, 64), (10, 64), (20, 64), (8, 128), (12, 80), (6, 48)])
        if rng.random() < 0.3:
            slots, tokens = _log_uniform(rng, 1, 128), rng.randint(1, 4)
            capacity = tokens + _log_uniform(rng, 16, 4096)
        else:
            tokens = _log_uniform(rng, 7, 4096)
            slots = _log_uniform(rng, 1, max(1, min(64, 41943040 // (tokens * heads * dim))))
            capacity = tokens + rng.choice([0, 0, 13, 100])
        case = _store("", slots, tokens, heads, dim, dtype, capacity, ragged=capacity > tokens and rng.random() < 0.7)
    else:
        dtype = rng.choice(["f16", "f16", "int8", "e4m3", "e5m2"])
        role = rng.choice(["cross", "cross", "self", "decode", "decode", "question"])
        if role == "cross":
            heads = rng.choice([10, 20])
            prefixes = rng.choice([1, 2, 2])
            batch, queries = prefixes * rng.randint(1, 8), _log_uniform(rng, 64, 4096 if heads == 10 else 1024)
            case = _attention("", batch, queries, heads, heads, 64, dtype, prefixes, rng.choice([77, 77, 154, 231, rng.randint(1, 400)]),
                              rng.choice([0, 0, 4, 16, rng.randint(1, 64)]))
        elif role == "self":
            heads = rng.choice([10, 20])
            tokens = rng.randint(12, 64 if heads == 10 else 32) * rng.randint(12, 64 if heads == 10 else 32)
            case = _attention("", 2, tokens, heads, heads, 64, "f16", 0, 0, tokens)
        else:
            q_heads, kv_heads, dim = rng.choice([(20, 20, 64), (10, 10, 64), (32, 8, 128), (16, 8, 80), (16, 2, 128), (12, 4, 96)])
            prefixes = rng.choice([1, 1, 1, 2, 3])
            if role == "decode":
                case = _attention("", prefixes * _log_uniform(rng, 1, 24), rng.choice([1, 1, 1, 2, 5]), q_heads, kv_heads, dim, dtype,
                                  prefixes, _log_uniform(rng, 60, 16384), _log_uniform(rng, 16, 1024), ragged=True,
                                  causal=rng.random() < 0.5)
            else:
                queries = _log_uniform(rng, 16, 500)
                case = _attention("", prefixes * rng.randint(1, 3), queries, q_heads, kv_heads, dim, dtype, prefixes,
                                  _log_uniform(rng, 60, 4096), queries + rng.choice([0, 0, 50]), causal=True)
    del case["name"]
    return case


# ---- inputs ----------------------------------------------------------------------------------------------
def _cache_values(shape, generator):
    """Keys or values as projections give them, FP16: each vector of a head has a size of its own, and a few of its places
    are larger than the others."""
    x = torch.randn(shape, generator=generator, device="cuda")
    x *= torch.exp(0.3 * torch.randn(shape[:-1] + (1,), generator=generator, device="cuda"))
    x *= 1.0 + 4.0 * (torch.rand(shape[-1:], generator=generator, device="cuda") < 0.03)
    return x.to(torch.float16)


def _encode(x, dtype):
    """FP16 vectors [..., D] in the cache's type: (data, scales [...] or None)."""
    if dtype == "f16":
        return x, None
    largest = x.abs().amax(-1).double()
    if dtype == "int8":
        scales = torch.where(largest > 0, largest / 127.0, torch.ones_like(largest)).float()
        return torch.round(x.double() / scales.double()[..., None]).clamp(-127, 127).to(torch.int8), scales
    exponent = torch.ceil(torch.log2(largest.clamp_min(2.0 ** -24) / FP8_MAX[dtype]))
    exponent = exponent + (largest > FP8_MAX[dtype] * torch.exp2(exponent)).double()          # the logarithm's last bit
    exponent = exponent - (largest <= FP8_MAX[dtype] * torch.exp2(exponent - 1)).double()
    scales = torch.where(largest > 0, torch.exp2(exponent), torch.ones_like(largest)).float()
    return (x.float() / scales[..., None]).clamp(-FP8_MAX[dtype], FP8_MAX[dtype]).to(FP8_TYPE[dtype]), scales


def _decode(data, scales):
    return data.float() if scales is None else data.float() * scales[..., None]


def _inputs(case, seed):
    generator = torch.Generator(device="cuda")
    generator.manual_seed(seed)
    state = {"case": case}

    def integers(low, high, count):
        return torch.randint(low, high + 1, (count,), generator=generator, device="cuda", dtype=torch.int32)

    if case["kind"] == "store":
        shape = (case["slots"], case["tokens"], case["heads"], case["dim"])
        state["key"], state["value"] = _cache_values(shape, generator), _cache_values(shape, generator)
        state["positions"] = integers(0, case["capacity"] - case["tokens"], case["slots"]) if case["ragged"] else None
        return state
    state["query"] = torch.randn((case["batch"], case["queries"], case["q_heads"], case["dim"]), generator=generator,
                                 device="cuda").to(torch.float16)
    for part, rows, tokens in (("prefix", case["prefixes"], case["prefix"]), ("own", case["batch"], case["own_tokens"])):
        state[part] = None
        if rows and tokens:
            # in the cache's own order: sequence, head, token
            shape = (rows, case["kv_heads"], tokens, case["dim"])
            state[part] = _encode(_cache_values(shape, generator), case["dtype"]) + _encode(_cache_values(shape, generator), case["dtype"])
    state["own_lengths"] = None
    if state["own"] is not None and case["ragged"]:
        state["own_lengths"] = integers(min(case["queries"], case["own_tokens"]), case["own_tokens"], case["batch"])
    return state


def _operators(pkg, made=[]):
    """The operators on the current stream. A program has one context for all its calls."""
    if not made:
        made.append(pkg.Ops(pkg.Context(0, workspace_bytes=1 << 20)))
    made[0].ctx.set_stream(torch.cuda.current_stream(0))
    return made[0]


def prepare(case, seed):
    state = _inputs(case, seed)
    if own:
        pkg = importlib.import_module("sdxl-end2end_b200")
        types = {"int8": pkg.ScalarType.Int8, "e4m3": pkg.ScalarType.Float8E4M3, "e5m2": pkg.ScalarType.Float8E5M2,
                 "f16": pkg.ScalarType.Float16}
        state["ops"] = ops = _operators(pkg)
        if case["kind"] == "store":
            state["cache"] = ops.kv_cache(case["slots"], case["capacity"], case["heads"], case["dim"], types[case["dtype"]])
        else:
            for part in ("prefix", "own"):
                if state[part] is not None:
                    k, k_scales, v, v_scales = state[part]
                    state[part] = pkg.KVCache(k.transpose(1, 2), v.transpose(1, 2), types[case["dtype"]], k_scales, v_scales)
    return state


# ---- the plain forms -------------------------------------------------------------------------------------
def _plain_attention(state):
    case = state["case"]
    batch, queries, q_heads, kv_heads = case["batch"], case["queries"], case["q_heads"], case["kv_heads"]
    query = state["query"].float().permute(0, 2, 1, 3) / math.sqrt(case["dim"])
    query = query.reshape(batch, kv_heads, q_heads // kv_heads * queries, case["dim"])
    parts = {}
    for part in ("prefix", "own"):
        if state[part] is not None:
            k, k_scales, v, v_scales = state[part]
            parts[part] = (_decode(k, k_scales), _decode(v, v_scales))
    out = torch.empty((batch, kv_heads, q_heads // kv_heads * queries, case["dim"]), dtype=torch.float16, device=query.device)
    for b in range(batch):
        scores, values = [], []
        if "prefix" in parts:
            row = b // (batch // case["prefixes"])
            scores.append(torch.matmul(query[b], parts["prefix"][0][row].transpose(1, 2)))
            values.append(parts["prefix"][1][row])
        if "own" in parts:
            tokens = torch.arange(case["own_tokens"], device=query.device)
            length = state["own_lengths"][b] if state["own_lengths"] is not None else case["own_tokens"]
            visible = (tokens < length).expand(queries, -1)
            if case["causal"]:
                visible = visible & (tokens[None, :] <= length - queries + torch.arange(queries, device=query.device)[:, None])
            score = torch.matmul(query[b], parts["own"][0][b].transpose(1, 2))
            scores.append(score.masked_fill(~visible.repeat(q_heads // kv_heads, 1), float("-inf")))
            values.append(torch.where((tokens < length)[:, None], parts["own"][1][b], 0.0))
        scores, values = torch.cat(scores, 2), torch.cat(values, 1)
        largest = scores.amax(2, keepdim=True)
        weights = torch.exp(scores - torch.where(largest > float("-inf"), largest, 0.0))
        total = weights.sum(2, keepdim=True)
        out[b] = (torch.matmul(weights, values) / torch.where(total > 0, total, 1.0)).to(torch.float16)
    return out.view(batch, q_heads, queries, case["dim"]).permute(0, 2, 1, 3).contiguous()


def run(state):
    case = state["case"]
    if own:
        ops = state["ops"]
        if case["kind"] == "store":
            ops.kv_cache_write(state["cache"], state["key"], state["value"], positions=state["positions"])
            return ops.kv_cache_read(state["cache"], case["tokens"], positions=state["positions"])
        return ops.shared_prefix_attention(state["query"], state["own"], state["prefix"], own_lengths=state["own_lengths"],
                                           causal=case["causal"])
    if case["kind"] == "attention":
        return _plain_attention(state)
    # what a cache of this type holds of the tokens
    return tuple(_decode(*_encode(state[part], case["dtype"])).to(torch.float16) for part in ("key", "value"))


# ---- what a pass cannot do without -----------------------------------------------------------------------
def work(case):
    width = 2 if case["dtype"] == "f16" else 1
    vector = width * case["dim"] + (0 if case["dtype"] == "f16" else 4)         # one head of one token in the cache
    if case["kind"] == "store":
        vectors = 2 * case["slots"] * case["tokens"] * case["heads"]
        return {"bytes": vectors * 2 * (2 * case["dim"] + vector), "flops": 2 * vectors * case["dim"]}
    rows = case["batch"] * case["queries"] * case["q_heads"]
    # lengths of their own are drawn evenly between one query's worth and all tokens
    own_mean = (min(case["queries"], case["own_tokens"]) + case["own_tokens"]) / 2 if case["ragged"] else case["own_tokens"]
    seen = own_mean
    if case["causal"] and own_mean:
        seen = max(0.0, own_mean - (case["queries"] - 1) / 2)
    tokens = case["prefixes"] * case["prefix"] + case["batch"] * own_mean
    return {"bytes": int(4 * rows * case["dim"] + 2 * vector * case["kv_heads"] * tokens),
            "flops": int(4 * rows * case["dim"] * (case["prefix"] * (case["prefixes"] > 0) + seen))}


# ---- the definition in 64 bits ---------------------------------------------------------------------------
def _exact_store(x, dtype):
    """Nearest representable multiple of the vector's scale, value by value."""
    x = x.double()
    if dtype == "f16":
        return x
    a = x.abs().max(dim=-1, keepdim=True).values
    one = torch.ones_like(a)
    if dtype == "int8":
        s = torch.where(a == 0, one, a / 127).float().double()
        return s * torch.clamp((x / s).round(), min=-127, max=127)
    # frexp: a = m 2^e with m in [0.5, 1); the format's largest value is top * 2^(e_max + 1)
    top, e_max, mantissa, least = {"e4m3": (0.875, 8, 3, -6), "e5m2": (0.875, 15, 2, -14)}[dtype]
    m, e = torch.frexp(a)
    s = torch.where(a == 0, one, torch.ldexp(one, e - (e_max + 1) + (m > top).to(e.dtype)))
    y = x / s
    step = torch.ldexp(torch.ones_like(y), torch.clamp(torch.frexp(y)[1] - 1, min=least) - mantissa)
    return s * torch.clamp((y / step).round() * step, min=-FP8_MAX[dtype], max=FP8_MAX[dtype])


def exact(case, seed):
    state = _inputs(case, seed)
    if case["kind"] == "store":
        return _exact_store(state["key"], case["dtype"]), _exact_store(state["value"], case["dtype"])
    q = state["query"].double()
    group = case["q_heads"] // case["kv_heads"]
    y = torch.zeros_like(q)

    def head(part, row, h):
        k, k_scales, v, v_scales = (None if t is None else t[row, h].double() for t in state[part])
        return (k, v) if k_scales is None else (k * k_scales.unsqueeze(1), v * v_scales.unsqueeze(1))

    for b in range(case["batch"]):
        n = case["own_tokens"] if state["own_lengths"] is None else int(state["own_lengths"][b])
        for h in range(case["kv_heads"]):
            keys, vals, count = [], [], 0
            if state["prefix"] is not None:
                k, v = head("prefix", b * case["prefixes"] // case["batch"], h)
                keys.append(k), vals.append(v)
                count = case["prefix"]
            if state["own"] is not None:
                k, v = head("own", b, h)
                keys.append(k[:n]), vals.append(v[:n])
            keys, vals = torch.cat(keys), torch.cat(vals)
            last = torch.full((case["queries"],), keys.shape[0], device=q.device)
            if case["causal"] and state["own"] is not None:
                last = count + (n - case["queries"] + 1 + torch.arange(case["queries"], device=q.device)).clamp(0, n)
            hidden = torch.arange(keys.shape[0], device=q.device)[None] >= last[:, None]
            for g in range(h * group, (h + 1) * group):
                s = (q[b, :, g] @ keys.t()) * case["dim"] ** -0.5
                s = torch.softmax(s.masked_fill(hidden, -math.inf), dim=1).nan_to_num(0.0)
                y[b, :, g] = s @ vals
    return y
