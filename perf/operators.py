"""What is measured of the operators that take a prompt's tokens chunk by chunk, beside the decode step.

A server that admits a prompt next to running requests needs, for a ragged batch of chunks (a few thousand new
tokens of one or several sequences, some of a single token): the attention of the new tokens over the paged e4m3
cache, the causal convolution and the gates in front of the gated delta rule, the delta rule itself on the slots'
int8 state, and copies of cache pages and state slots for prefixes that several requests share.

Dimensions are those of the framework's model: 24 query heads over 4 KV heads of 256, 16 key heads and 32 or 48 value
heads of 128, four convolution taps, pages of 16 or 64 tokens.  Everything is drawn on the GPU from the seed;
how a batch is divided into sequences follows from the case alone.
"""

import math

import numpy as np
import torch

own = False

QUERY_HEADS, KV_HEADS, GROUP, HEAD_DIM = 24, 4, 6, 256
KEY_HEADS, DIM, TAPS = 16, 128, 4
EPSILON = 1e-6
CHUNK = 64  # tokens that the plain form of the delta rule takes at once


def listed():
    return [
        # a short turn at the end of a long conversation: few rows, and a cache that has to be read whole
        {"name": "attention_t16_of_32k", "kind": "attention", "sequences": 1, "tokens": 16, "past": 32752, "page": 16,
         "gated": True, "scaled": True},
        # the first chunk of one prompt, nothing in the cache before it
        {"name": "attention_prompt_2048", "kind": "attention", "sequences": 1, "tokens": 2048, "past": 0, "page": 16,
         "gated": True, "scaled": True},
        # a mixed batch: chunks of several prompts, odd lengths, single tokens among them
        {"name": "attention_mixed_13", "kind": "attention", "sequences": 13, "tokens": 2039, "past": 8192, "page": 64,
         "gated": True, "scaled": False},
        # the last chunk of a long document
        {"name": "attention_t4096_of_32k", "kind": "attention", "sequences": 1, "tokens": 4096, "past": 28672,
         "page": 16, "gated": False, "scaled": True},
        # a short turn: one sequence, less than a block of tokens
        {"name": "delta_t17_v32", "kind": "delta", "sequences": 1, "tokens": 17, "heads": 32, "normed": False},
        # one prompt: as long as the recurrence is, and as narrow as the heads are few
        {"name": "delta_prompt_2048_v48", "kind": "delta", "sequences": 1, "tokens": 2048, "heads": 48, "normed": True},
        # a mixed batch of odd lengths
        {"name": "delta_mixed_13_v32", "kind": "delta", "sequences": 13, "tokens": 2039, "heads": 32, "normed": True},
        # four long prompts at once
        {"name": "delta_c4_8192_v48", "kind": "delta", "sequences": 4, "tokens": 8192, "heads": 48, "normed": False},
        # in front of the delta rule: a short turn ...
        {"name": "prepare_t17_v32", "kind": "prepare", "sequences": 1, "tokens": 17, "heads": 32},
        # ... and a full batch
        {"name": "prepare_c4_8192_v48", "kind": "prepare", "sequences": 4, "tokens": 8192, "heads": 48},
        # a request continues a shared prefix that ends inside a page: its own copy, K and V of 16 layers
        {"name": "copy_page", "kind": "copy", "arrays": 32, "units": 512, "unit": 16384, "pairs": 1},
        # the pages of long conversations move together: 200 pages of 64 tokens in every layer
        {"name": "copy_200_pages", "kind": "copy", "arrays": 32, "units": 512, "unit": 65536, "pairs": 200},
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["attention", "attention", "delta", "delta", "prepare", "copy"])
    if kind == "attention":
        tokens = _log_int(rng, 1, 4096)
        past = _log_int(rng, 1, 32768) - 1
        while tokens * (tokens + past) > 4096 * 24576:
            past //= 2
        return {"kind": kind, "sequences": _log_int(rng, 1, min(tokens, 32)), "tokens": tokens, "past": past,
                "page": rng.choice([16, 64]), "gated": rng.random() < 0.5, "scaled": rng.random() < 0.5}
    if kind in ("delta", "prepare"):
        tokens = _log_int(rng, 1, 8192)
        case = {"kind": kind, "sequences": _log_int(rng, 1, min(tokens, 32)), "tokens": tokens, "heads": rng.choice([32, 48])}
        if kind == "delta":
            case["normed"] = rng.random() < 0.5
        return case
    units = rng.randint(64, 512)
    return {"kind": kind, "arrays": rng.randint(1, 36), "units": units, "unit": 16 * _log_int(rng, 64, 4096),
            "pairs": _log_int(rng, 1, units * 2 // 5)}


def _lengths(case):
    """Tokens of each sequence (one at least; very different ones) and what its cache held before."""
    sequences, tokens = case["sequences"], case["tokens"]
    rng = np.random.default_rng([tokens, sequences, 5])
    weights = np.exp(rng.uniform(0.0, 4.0, sequences))
    lengths = 1 + np.floor((tokens - sequences) * weights / weights.sum()).astype(np.int64)
    lengths[int(np.argmax(lengths))] += tokens - int(lengths.sum())
    past = np.zeros(sequences, dtype=np.int64)
    if case.get("past"):
        past = np.floor(np.exp(rng.uniform(0.0, math.log(case["past"] + 1), sequences))).astype(np.int64)
        past[int(rng.integers(sequences))] = case["past"]
    return lengths, past


# ---- inputs ----------------------------------------------------------------------------------------------

def _generator(seed):
    generator = torch.Generator(device="cuda")
    generator.manual_seed(seed)
    return generator


def _randn(shape, generator, std=1.0):
    return torch.randn(shape, device="cuda", generator=generator) * std


def _bf16(shape, generator, std=1.0):
    return _randn(shape, generator, std).to(torch.bfloat16)


def _u32(values):
    return torch.from_numpy(np.asarray(values, dtype=np.int32)).cuda()


def _batch(case):
    lengths, past = _lengths(case)
    begins = np.concatenate([[0], np.cumsum(lengths)])
    return {"kind": case["kind"], "tokens": case["tokens"], "sequences": case["sequences"],
            "lengths": [int(n) for n in lengths], "first": [int(b) for b in begins], "begins": _u32(begins),
            "past": [int(p) for p in past]}


def _prepare_attention(case, seed):
    generator = _generator(seed)
    state = _batch(case)
    page = state["page"] = case["page"]
    contexts = np.array(state["lengths"]) + np.array(state["past"])
    blocks = -(-contexts // page)
    pool, widest = int(blocks.sum()) + 3, int(blocks.max())
    tables = np.zeros((case["sequences"], widest), dtype=np.int32)
    pages = np.random.default_rng([seed, 11]).permutation(pool)
    first = 0
    for row, count in enumerate(blocks):
        tables[row, :count] = pages[first:first + count]
        first += int(count)
    # queries after their norm; keys and values fill the codes' range by their scales
    state.update(pool=pool, widest=widest, tables=_u32(tables), contexts=_u32(contexts),
                 query=_bf16((case["tokens"], QUERY_HEADS, HEAD_DIM), generator), gate=None, scales=None,
                 output=torch.zeros((case["tokens"], QUERY_HEADS, HEAD_DIM), dtype=torch.bfloat16, device="cuda"))
    if case["gated"]:
        state["gate"] = _bf16((case["tokens"], QUERY_HEADS, 2 * HEAD_DIM), generator)
    scale = torch.ones(KV_HEADS, device="cuda")
    if case["scaled"]:
        scale = (0.5 + torch.rand(KV_HEADS, device="cuda", generator=generator)) / 64.0
        state["scales"] = scale
    for name in ("keys", "values"):
        values = _randn((pool, KV_HEADS, page, HEAD_DIM), generator) / scale[None, :, None, None]
        state[name] = values.clamp_(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
    return state


def _gates(tokens, heads, generator):
    """Decay and write strength as the model's gates give them: heads that forget in a few tokens beside heads
    that hold for thousands."""
    rate = torch.exp(torch.linspace(math.log(0.002), math.log(2.0), heads, device="cuda"))
    alpha = torch.exp(-rate * torch.nn.functional.softplus(_randn((tokens, heads), generator)))
    return alpha, torch.sigmoid(_randn((tokens, heads), generator))


def _slots(case, seed):
    """Slots of a pool that has three more, and which sequences continue what their slot holds (the others begin)."""
    rng = np.random.default_rng([seed, 13])
    sequences = case["sequences"]
    return _u32(rng.permutation(sequences + 3)[:sequences]), _u32(rng.random(sequences) < 0.7), sequences + 3


def _prepare_delta(case, seed):
    generator = _generator(seed)
    state = _batch(case)
    tokens, heads = case["tokens"], case["heads"]
    state["heads"] = heads
    state["slots"], state["continues"], state["capacity"] = _slots(case, seed)
    unit = [torch.nn.functional.normalize(_randn((tokens, KEY_HEADS, DIM), generator), dim=-1) for _ in range(2)]
    values = torch.nn.functional.silu(_randn((tokens, heads, DIM), generator))
    parts = (unit[0] / math.sqrt(DIM), unit[1], values)
    state["qkv"] = torch.cat([part.reshape(tokens, -1) for part in parts], 1).to(torch.bfloat16)
    state["alpha"], state["beta"] = _gates(tokens, heads, generator)
    held = _randn((state["capacity"], heads, DIM, DIM), generator, 0.1)
    peak = held.abs().amax(-1)
    state["codes"] = (held * (127.0 / peak)[..., None]).round_().to(torch.int8)
    state["scales"] = peak * (1.0 / 127.0)
    state["out"] = torch.zeros((tokens, heads, DIM), dtype=torch.bfloat16, device="cuda")
    state["held"] = torch.zeros((state["capacity"], heads, DIM, DIM), dtype=torch.bfloat16, device="cuda")
    state["gate"] = state["weight"] = None
    if case["normed"]:
        state["gate"] = _bf16((tokens, heads * DIM), generator)
        state["weight"] = (1.0 + _randn((DIM,), generator, 0.1)).to(torch.bfloat16)
    return state


def _prepare_prepare(case, seed):
    generator = _generator(seed)
    state = _batch(case)
    tokens, heads = case["tokens"], case["heads"]
    state["heads"] = heads
    state["slots"], state["continues"], state["capacity"] = _slots(case, seed)
    channels = state["channels"] = (2 * KEY_HEADS + heads) * DIM
    # rows of the fused in-projection: q | k | v | z | b | a
    state["width"] = channels + heads * DIM + 2 * heads
    state["b_column"], state["a_column"] = channels + heads * DIM, channels + heads * DIM + heads
    state["mixed"] = _bf16((tokens, state["width"]), generator)
    state["taps"] = _bf16((channels, TAPS), generator, 0.5)
    state["a_log"] = _bf16((heads,), generator, 0.5)
    state["dt_bias"] = _bf16((heads,), generator, 0.5)
    state["history"] = _bf16((state["capacity"], channels, TAPS - 1), generator).float()
    state["qkv"] = torch.zeros((tokens, channels), dtype=torch.bfloat16, device="cuda")
    state["alpha"] = torch.zeros((tokens, heads), device="cuda")
    state["beta"] = torch.zeros((tokens, heads), device="cuda")
    return state


def _prepare_copy(case, seed):
    arrays, units, unit = case["arrays"], case["units"], case["unit"]
    rng = np.random.default_rng([seed, 17])
    chosen = rng.permutation(units)[:2 * case["pairs"]].reshape(-1, 2)
    memory = torch.randint(0, 256, (arrays, units, unit), dtype=torch.uint8, device="cuda", generator=_generator(seed))
    table = np.array([[memory[i].data_ptr(), unit, units] for i in range(arrays)], dtype=np.uint64)
    return {"kind": "copy", "memory": memory, "table": table, "pairs": _u32(chosen), "count": case["pairs"]}


def prepare(case, seed):
    return {"attention": _prepare_attention, "delta": _prepare_delta, "prepare": _prepare_prepare,
            "copy": _prepare_copy}[case["kind"]](case, seed)


# ---- the plain form --------------------------------------------------------------------------------------

def _plain_attention(state):
    page, output = state["page"], state["output"]
    scales = state["scales"] if state["scales"] is not None else torch.ones(KV_HEADS, device="cuda")
    for s, (begin, length, past) in enumerate(zip(state["first"], state["lengths"], state["past"])):
        context = past + length
        pages = state["tables"][s, :-(-context // page)].long()
        query = state["query"][begin:begin + length].float().reshape(length, KV_HEADS, GROUP, HEAD_DIM)
        at = torch.arange(length, device="cuda") + past
        hidden = (torch.arange(context, device="cuda")[None, :] > at[:, None])[None]
        for head in range(KV_HEADS):
            keys, values = (state[name][pages, head].reshape(-1, HEAD_DIM)[:context].view(torch.float8_e4m3fn).float() *
                            scales[head] for name in ("keys", "values"))
            scores = (query[:, head].transpose(0, 1) @ keys.T) * (1.0 / math.sqrt(HEAD_DIM))
            scores = scores.masked_fill_(hidden, -math.inf)
            weights = scores.sub_(scores.amax(-1, keepdim=True)).exp_()
            result = (weights @ values) / weights.sum(-1, keepdim=True)
            result = result.transpose(0, 1)
            if state["gate"] is not None:
                gate = state["gate"][begin:begin + length, head * GROUP:(head + 1) * GROUP, HEAD_DIM:].float()
                result = result * (1.0 / (1.0 + torch.exp(-gate)))
            output[begin:begin + length, head * GROUP:(head + 1) * GROUP] = result.to(torch.bfloat16)
    return output


def _padded(state, rows, blocks):
    """Rows of a ragged batch [tokens, heads, ...] as [sequences, heads, blocks, CHUNK, ...], zeros behind each sequence."""
    out = torch.zeros((state["sequences"], blocks * CHUNK) + rows.shape[1:], device="cuda")
    out[state["row_sequence"], state["row_place"]] = rows.float()
    return out.reshape((state["sequences"], blocks, CHUNK) + rows.shape[1:]).movedim(3, 1)


def _rows(state):
    lengths = torch.tensor(state["lengths"], device="cuda")
    sequence = torch.repeat_interleave(torch.arange(state["sequences"], device="cuda"), lengths)
    place = torch.arange(state["tokens"], device="cuda") - state["begins"].long()[sequence]
    return sequence, place


def _store_state(state, held):
    """The slots of the batch in eight bits again: a scale for each row of the state."""
    peak = held.abs().amax(-1)
    inverse = torch.where(peak > 0, 127.0 / peak, torch.zeros_like(peak))
    slots = state["slots"].long()
    state["codes"][slots] = (held * inverse[..., None]).round().to(torch.int8)
    state["scales"][slots] = peak * (1.0 / 127.0)


def _state_values(state):
    # eight bits of a state are worth as many as bf16 has
    return torch.mul(state["codes"], state["scales"][..., None], out=state["held"])


def _plain_delta(state):
    heads, sequences = state["heads"], state["sequences"]
    state["row_sequence"], state["row_place"] = _rows(state)
    blocks = -(-max(state["lengths"]) // CHUNK)
    tokens, ratio = state["tokens"], heads // KEY_HEADS
    q, k, v = state["qkv"].split([KEY_HEADS * DIM, KEY_HEADS * DIM, heads * DIM], 1)
    q, k = (_padded(state, x.reshape(tokens, KEY_HEADS, DIM), blocks).repeat_interleave(ratio, 1) for x in (q, k))
    v = _padded(state, v.reshape(tokens, heads, DIM), blocks)
    beta = _padded(state, state["beta"], blocks)
    # decay from the block's start, and between two tokens of it; padding holds everything
    logs = state["alpha"].double().clamp_min(1e-45).log()
    total = torch.zeros((sequences, blocks * CHUNK, heads), dtype=torch.float64, device="cuda")
    total[state["row_sequence"], state["row_place"]] = logs
    total = total.reshape(sequences, blocks, CHUNK, heads).movedim(3, 1).cumsum(-1)
    lower = torch.ones((CHUNK, CHUNK), dtype=torch.bool, device="cuda").tril()
    decay = (total[..., :, None] - total[..., None, :]).masked_fill(~lower, -math.inf).exp().float()
    from_start, to_end = total.exp().float(), (total[..., -1:] - total).exp().float()
    within = (k @ k.transpose(-1, -2)) * decay * beta[..., None]
    mixing = (q @ k.transpose(-1, -2)) * decay
    solved = torch.eye(CHUNK, device="cuda").expand(within.shape).contiguous()
    for i in range(1, CHUNK):  # (1 + strictly lower part)^-1, row by row
        solved[..., i, :i] = -(within[..., i:i + 1, :i] @ solved[..., :i, :i])[..., 0, :]
    slots = state["slots"].long()
    held = state["codes"][slots].float() * state["scales"][slots][..., None]
    held = held * (state["continues"] != 0)[:, None, None, None]
    outputs = []
    for c in range(blocks):
        kc, qc, start = k[:, :, c], q[:, :, c], from_start[:, :, c, :, None]
        fresh = (v[:, :, c] - start * (kc @ held.transpose(-1, -2))) * beta[:, :, c, :, None]
        fresh = solved[:, :, c] @ fresh
        outputs.append(start * (qc @ held.transpose(-1, -2)) + mixing[:, :, c] @ fresh)
        held = held * from_start[:, :, c, -1, None, None] + (fresh * to_end[:, :, c, :, None]).transpose(-1, -2) @ kc
    result = torch.stack(outputs, 2).movedim(1, 3).reshape(sequences, blocks * CHUNK, heads, DIM)
    result = result[state["row_sequence"], state["row_place"]]
    if state["gate"] is not None:
        gate = state["gate"].float().reshape(tokens, heads, DIM)
        result = result / torch.sqrt((result * result).mean(-1, keepdim=True) + EPSILON)
        result = result * state["weight"].float() * (gate / (1.0 + torch.exp(-gate)))
    state["out"].copy_(result)
    _store_state(state, held)
    return {"out": state["out"], "state": _state_values(state)}


def _plain_prepare(state):
    heads, channels, tokens = state["heads"], state["channels"], state["tokens"]
    sequence, _ = _rows(state)
    slots = state["slots"].long()
    history = state["history"][slots] * (state["continues"] != 0)[:, None, None]
    # every sequence's rows behind its three of history
    rows = torch.zeros((tokens + 3 * state["sequences"], channels), device="cuda")
    at = torch.arange(tokens, device="cuda") + 3 * (sequence + 1)
    rows[at] = state["mixed"][:, :channels].float()
    before = state["begins"].long()[:-1] + 3 * torch.arange(state["sequences"], device="cuda")
    places = before[:, None] + torch.arange(3, device="cuda")
    rows[places] = history.transpose(1, 2)
    taps = state["taps"].float()
    sums = rows[at - 3] * taps[:, 0] + rows[at - 2] * taps[:, 1] + rows[at - 1] * taps[:, 2] + rows[at] * taps[:, 3]
    active = sums / (1.0 + torch.exp(-sums))
    q, k, v = active.split([KEY_HEADS * DIM, KEY_HEADS * DIM, heads * DIM], 1)
    q, k = (x.reshape(tokens, KEY_HEADS, DIM) for x in (q, k))
    q, k = (x / torch.sqrt((x * x).sum(-1, keepdim=True) + EPSILON) for x in (q, k))
    q = q * (1.0 / math.sqrt(DIM))
    state["qkv"].copy_(torch.cat([q.reshape(tokens, -1), k.reshape(tokens, -1), v], 1))
    last = state["begins"].long()[1:] + 3 * torch.arange(1, state["sequences"] + 1, device="cuda")
    state["history"][slots] = rows[last[:, None] + torch.arange(-3, 0, device="cuda")].transpose(1, 2)
    a = state["mixed"][:, state["a_column"]:state["a_column"] + heads].double() + state["dt_bias"].double()
    b = state["mixed"][:, state["b_column"]:state["b_column"] + heads].double()
    rate = torch.exp(state["a_log"].double())
    state["alpha"].copy_(torch.exp(-rate * torch.log1p(torch.exp(a))))
    state["beta"].copy_(1.0 / (1.0 + torch.exp(-b)))
    return {name: state[name] for name in ("qkv", "alpha", "beta", "history")}


def _plain_copy(state):
    pairs = state["pairs"].long()
    state["memory"][:, pairs[:, 1]] = state["memory"][:, pairs[:, 0]]
    return state["memory"]


# ---- the framework's operators ---------------------------------------------------------------------------

def _workspace(state, nbytes):
    """A program keeps its workspace from one call to the next."""
    if "workspace" not in state:
        state["workspace"] = torch.zeros(max(16, nbytes), dtype=torch.uint8, device="cuda")
    return state["workspace"]


def _own_attention(state):
    from qwencore_b200 import ops
    workspace = _workspace(state, ops.attention_chunk_workspace_bytes())
    ops.paged_attention_chunk(state["query"], state["gate"], state["keys"], state["values"], state["tables"],
                              state["contexts"], state["begins"], state["widest"], state["output"], state["tokens"],
                              state["sequences"], workspace, state["page"], state["pool"], key_scales=state["scales"],
                              value_scales=state["scales"])
    return state["output"]


def _own_delta(state):
    from qwencore_b200 import abi, ops
    abi.configure(state["heads"], 64)
    workspace = _workspace(state, ops.delta_chunk_workspace_bytes(state["tokens"], state["sequences"]))
    ops.delta_chunk(state["codes"], state["scales"], state["slots"], state["continues"], state["begins"], state["qkv"],
                    state["alpha"], state["beta"], state["out"], state["capacity"], state["tokens"],
                    state["sequences"], workspace, gate=state["gate"], norm_weight=state["weight"], epsilon=EPSILON)
    return {"out": state["out"], "state": _state_values(state)}


def _own_prepare(state):
    from qwencore_b200 import abi, ops
    abi.configure(state["heads"], 64)
    ops.delta_prepare_chunk(state["mixed"], state["a_column"], state["b_column"], state["taps"], state["a_log"],
                            state["dt_bias"], state["history"], state["slots"], state["continues"], state["begins"],
                            state["qkv"], state["alpha"], state["beta"], state["capacity"], state["tokens"],
                            state["sequences"], state["width"])
    return {name: state[name] for name in ("qkv", "alpha", "beta", "history")}


def _own_copy(state):
    from qwencore_b200 import ops
    ops.cache_copy(state["table"], state["pairs"], state["count"])
    return state["memory"]


def run(state):
    if own:
        return {"attention": _own_attention, "delta": _own_delta, "prepare": _own_prepare,
                "copy": _own_copy}[state["kind"]](state)
    return {"attention": _plain_attention, "delta": _plain_delta, "prepare": _plain_prepare,
            "copy": _plain_copy}[state["kind"]](state)


# ---- from the definitions, in 64 bits --------------------------------------------------------------------

def _exact_attention(s):
    result = torch.zeros((s["tokens"], QUERY_HEADS, HEAD_DIM), dtype=torch.float64, device="cuda")
    dequantised = []
    for name in ("keys", "values"):
        cache = s[name].view(torch.float8_e4m3fn).double()
        dequantised.append(cache if s["scales"] is None else cache * s["scales"].double()[None, :, None, None])
    for i in range(s["sequences"]):
        row, context = s["first"][i], s["past"][i] + s["lengths"][i]
        ids = s["tables"][i, :-(-context // s["page"])].long()
        keys, values = (cache[ids].transpose(0, 1).reshape(KV_HEADS, -1, HEAD_DIM)[:, :context] for cache in dequantised)
        for at in range(0, s["lengths"][i], 512):  # rows in slices, all heads of one KV head at once
            count = min(512, s["lengths"][i] - at)
            query = s["query"][row + at:row + at + count].double()
            seen = s["past"][i] + at + 1 + torch.arange(count, device="cuda")
            for head in range(QUERY_HEADS):
                logits = torch.einsum("td,cd->tc", query[:, head], keys[head // GROUP]) / 16.0
                logits[torch.arange(context, device="cuda")[None] >= seen[:, None]] = -math.inf
                result[row + at:row + at + count, head] = torch.softmax(logits, 1) @ values[head // GROUP]
    if s["gate"] is not None:
        result *= torch.sigmoid(s["gate"][..., HEAD_DIM:].double())
    return result


def _exact_delta(s):
    heads, ratio, slots = s["heads"], s["heads"] // KEY_HEADS, s["slots"].long()
    rows = s["qkv"].double()
    q = rows[:, :KEY_HEADS * DIM].reshape(-1, KEY_HEADS, DIM)
    k = rows[:, KEY_HEADS * DIM:2 * KEY_HEADS * DIM].reshape(-1, KEY_HEADS, DIM)
    v = rows[:, 2 * KEY_HEADS * DIM:].reshape(-1, heads, DIM)
    values = s["codes"].double() * s["scales"].double()[..., None]
    state = values[slots]
    state[s["continues"] == 0] = 0.0
    out = torch.zeros((s["tokens"], heads, DIM), dtype=torch.float64, device="cuda")
    order = sorted(range(s["sequences"]), key=lambda i: -s["lengths"][i])
    state = state[order]
    for step in range(max(s["lengths"])):  # one token of every sequence that is long enough
        live = [i for i in order if s["lengths"][i] > step]
        n = len(live)
        at = torch.tensor([s["first"][i] + step for i in live], device="cuda")
        key, query = (x[at].repeat_interleave(ratio, 1) for x in (k, q))
        state[:n] *= s["alpha"][at].double()[..., None, None]
        wrong = v[at] - torch.einsum("nhij,nhj->nhi", state[:n], key)
        state[:n] += torch.einsum("nhi,nhj->nhij", wrong * s["beta"][at].double()[..., None], key)
        out[at] = torch.einsum("nhij,nhj->nhi", state[:n], query)
    if s["gate"] is not None:
        out = out * torch.rsqrt(out.square().mean(-1, keepdim=True) + EPSILON) * s["weight"].double()
        out = out * torch.nn.functional.silu(s["gate"].double().reshape(out.shape))
    largest = state.abs().amax(-1, keepdim=True)
    step = largest / 127.0
    values[slots[order]] = torch.where(largest > 0, torch.round(state / step) * step, state)
    return {"out": out, "state": values}


def _exact_prepare(s):
    heads, channels = s["heads"], s["channels"]
    out, history = [], s["history"].double().clone()
    for i in range(s["sequences"]):
        rows = s["mixed"][s["first"][i]:s["first"][i + 1], :channels].double().T
        slot = int(s["slots"][i])
        before = history[slot] if int(s["continues"][i]) else torch.zeros_like(history[slot])
        line = torch.cat([before, rows], 1)
        out.append(torch.nn.functional.silu((line.unfold(1, TAPS, 1) * s["taps"].double()[:, None]).sum(-1)).T)
        history[slot] = line[:, -3:]
    out = torch.cat(out)
    for part, factor in ((slice(0, KEY_HEADS * DIM), DIM ** -0.5), (slice(KEY_HEADS * DIM, 2 * KEY_HEADS * DIM), 1.0)):
        x = out[:, part].reshape(-1, KEY_HEADS, DIM)
        out[:, part] = (factor * x * torch.rsqrt(x.square().sum(-1, keepdim=True) + EPSILON)).reshape(-1, KEY_HEADS * DIM)
    a = s["mixed"][:, s["a_column"]:s["a_column"] + heads].double()
    rate = torch.nn.functional.softplus(a + s["dt_bias"].double(), threshold=60.0) * s["a_log"].double().exp()
    beta = torch.sigmoid(s["mixed"][:, s["b_column"]:s["b_column"] + heads].double())
    return {"qkv": out, "alpha": (-rate).exp(), "beta": beta, "history": history}


def exact(case, seed):
    if case["kind"] == "copy":
        return None  # bytes: equal or wrong
    state = prepare(case, seed)
    return {"attention": _exact_attention, "delta": _exact_delta, "prepare": _exact_prepare}[case["kind"]](state)


# ---- what a pass cannot do without -----------------------------------------------------------------------

def work(case):
    if case["kind"] == "copy":
        return {"bytes": 2 * case["arrays"] * case["unit"] * case["pairs"], "flops": 0}
    lengths, past = _lengths(case)
    tokens = case["tokens"]
    if case["kind"] == "attention":
        seen = int((lengths * past + lengths * (lengths + 1) // 2).sum())
        rows = tokens * QUERY_HEADS * HEAD_DIM * 2 * (3 if case["gated"] else 2)
        return {"bytes": int((lengths + past).sum()) * 2 * KV_HEADS * HEAD_DIM + rows, "flops": seen * QUERY_HEADS * HEAD_DIM * 4}
    heads, channels = case["heads"], (2 * KEY_HEADS + case["heads"]) * DIM
    if case["kind"] == "prepare":
        history = 2 * case["sequences"] * channels * 12
        return {"bytes": tokens * (channels * 4 + heads * 12) + history + channels * 8, "flops": tokens * channels * 10}
    # the recurrence itself: two products with the state and its update, for each token and head; the state's values
    # leave as bf16 beside the codes
    state = case["sequences"] * heads * 2 * (DIM * DIM + 4 * DIM) + (case["sequences"] + 3) * heads * DIM * DIM * 3
    rows = tokens * (channels * 2 + heads * (8 + 2 * DIM) + (heads * 2 * DIM if case["normed"] else 0))
    return {"bytes": rows + state, "flops": tokens * heads * DIM * DIM * 6}
