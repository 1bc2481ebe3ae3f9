"""What is timed of recurrent layers' state and of beam search: the gated delta rule, the short convolution in front of it, the
selection over beams and vocabulary, and the reordering of caches by what it selects.

The gated delta rule.  A state S [Dv, Dk] in float32 for each sequence and value head; each key head serves Hv / Hk value heads:

    q^ = scale q / sqrt(sum q^2 + eps),  k^ = k / sqrt(sum k^2 + eps)
    g = exp(-exp(a_log) softplus(a + dt_bias)),  beta = sigmoid(b)
    S <- g S;  u = beta (v - S k^);  S <- S + u k^T;  o = S q^

The short convolution.  y_t = silu(sum_w weight[:, w] x_{t - W + 1 + w}) by channel, the W - 1 inputs before the call's first one
taken from the cache, which then holds the last W - 1.  In both, sequence b's tokens are those at left_pad[b] <= t < lengths[b]; the
others are not there (outputs of zero).

The selection.  Beam k of batch row b continued by token t scores  s[b, k] + x[b, k, t] - log sum exp x[b, k, :]; the `count` best of
the beams times the vocabulary, best first; among equals the lower beam, then the lower token.  A beam that is done offers one
candidate, the pad token, at its own score.

Reordering.  Row b of a cache becomes what row order[b] was, from position `shared` on (before it they are the same).
"""
import math
import os
import sys

import torch

own = False  # True: the framework's operators; False: their plain forms

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
EPS = 1e-6
CHUNK = 64    # tokens of a chunk of the plain gated delta rule
WIDTH = 4     # taps of the short convolution
PAD_TOKEN = 0


def _delta(name, **given):
    case = dict(name=name, kind="delta", dtype="bf16", batch=1, new=1, k_heads=16, v_heads=32, k_dim=128, v_dim=128, ragged=False)
    case.update(given)
    return case


def _conv(name, **given):
    case = dict(name=name, kind="conv", dtype="bf16", batch=1, new=1, channels=8192, ragged=False)
    case.update(given)
    return case


def _select(name, **given):
    case = dict(name=name, kind="select", dtype="bf16", batch=1, beams=4, vocabulary=32000, count=4, done=False)
    case.update(given)
    return case


def _beams(name, **given):
    """A decode step of beam search on one attention layer and one recurrent layer.  `vocabulary` 0: the order is given."""
    case = dict(name=name, kind="beams", dtype="bf16", batch=1, beams=4, vocabulary=0, context=1000, shared=500, q_heads=32, kv_heads=8,
                head_dim=128, state_heads=0)
    case.update(given)
    return case


def listed():
    return [
        # One user's token: a layer of a hybrid model.
        _delta("delta_step"),
        # Serving 64 sequences, a token each.
        _delta("delta_serve", batch=64),
        # Five draft tokens of 16 sequences scored at once, in full precision.
        _delta("delta_draft", dtype="f32", batch=16, new=5),
        # A chat turn's prompt.
        _delta("delta_turn", new=333),
        # A chunk of a long document.
        _delta("delta_prompt", new=8192),
        # Prompts of many lengths, padded to one.
        _delta("delta_ragged", dtype="f16", batch=8, new=2000, ragged=True),
        # The convolution of the serving step and of the document above: queries, keys and values in one array.
        _conv("conv_serve", batch=64),
        _conv("conv_prompt", new=8192),
        # One request's four beams over a small vocabulary, logits in full precision.
        _select("select_small", dtype="f32"),
        # Thirty-two requests of eight beams over a large one, some of them done.
        _select("select_serve", batch=32, beams=8, vocabulary=152064, count=8, done=True),
        # Eight hypotheses of one request trade places and take their next token.
        _beams("reorder_step", beams=8, context=2011, shared=700),
        # A whole step of eight requests of four: selection, both layers' caches reordered, attention.
        _beams("beams_serve", dtype="f16", batch=8, vocabulary=128000, context=4100, shared=3500, state_heads=32),
    ]


# (key heads, value heads, key size, value size)
DELTA_LAYOUTS = [(16, 32, 128, 128), (16, 16, 128, 128), (8, 16, 64, 64), (4, 4, 256, 512), (8, 8, 96, 96)]
# (query heads, kv heads, head size)
ATTENTION_LAYOUTS = [(32, 8, 128), (16, 4, 64), (16, 8, 256)]
LARGEST_BYTES, LARGEST_FLOPS, LARGEST_CONTEXT = 2.7e8, 2.6e10, 6.0e8


def _log_uniform(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    while True:
        kind = rng.choice(["delta", "delta", "delta", "conv", "select", "select", "beams"])
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        if kind == "delta":
            hk, hv, dk, dv = rng.choice(DELTA_LAYOUTS)
            case = _delta("", dtype=dtype, batch=_log_uniform(rng, 1, 64), k_heads=hk, v_heads=hv, k_dim=dk, v_dim=dv,
                          new=rng.choice([1, rng.randint(2, 16), _log_uniform(rng, 17, 8192), _log_uniform(rng, 17, 8192)]))
            case["ragged"] = case["batch"] > 1 and case["new"] > 16 and rng.random() < 0.5
        elif kind == "conv":
            case = _conv("", dtype=dtype, batch=_log_uniform(rng, 1, 64), channels=rng.choice([512, 1536, 6144, 8192, 1000]),
                         new=rng.choice([1, rng.randint(2, 16), _log_uniform(rng, 17, 8192)]))
            case["ragged"] = case["batch"] > 1 and case["new"] > 16 and rng.random() < 0.5
        elif kind == "select":
            beams = rng.choice([1, 2, 3, 4, 5, 8, 16])
            case = _select("", dtype=dtype, batch=_log_uniform(rng, 1, 64), beams=beams, vocabulary=_log_uniform(rng, 1000, 262144),
                           count=beams * rng.choice([1, 2]), done=rng.random() < 0.5)
        else:
            hq, hkv, d = rng.choice(ATTENTION_LAYOUTS)
            context = _log_uniform(rng, 100, 8192)
            case = _beams("", dtype=dtype, batch=_log_uniform(rng, 1, 8), beams=rng.choice([2, 3, 4, 5, 8]), context=context,
                          shared=rng.randint(0, context), q_heads=hq, kv_heads=hkv, head_dim=d, state_heads=rng.choice([0, 16, 32]),
                          vocabulary=rng.choice([0, _log_uniform(rng, 1000, 128000)]))
        del case["name"]
        w = work(case)
        if kind == "beams":
            rows = case["batch"] * case["beams"] * case["kv_heads"] * case["context"] * case["head_dim"] * 4.0
            if rows <= LARGEST_CONTEXT:
                return case
        elif w["bytes"] <= LARGEST_BYTES and w["flops"] <= LARGEST_FLOPS:
            return case


# ---- inputs -------------------------------------------------------------------------------------------------------
def _kvhip():
    path = os.path.join(os.getcwd(), "mlx-swift-lm_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import kvhip
    return kvhip


class _Maker:
    def __init__(self, seed):
        self.gen = torch.Generator(device="cuda")
        self.gen.manual_seed(seed)

    def normal(self, *shape):
        return torch.randn(*shape, generator=self.gen, device="cuda")

    def uniform(self, low, high, *shape):
        return low + (high - low) * torch.rand(*shape, generator=self.gen, device="cuda")

    def whole(self, low, high, *shape):
        return torch.randint(low, high, shape, generator=self.gen, device="cuda", dtype=torch.int32)

    def paddings(self, case):
        """Tokens in front of each sequence that are none, and where it ends."""
        if not case["ragged"]:
            return None, None
        n = case["new"]
        pad = self.whole(0, n // 3 + 1, case["batch"])
        return pad, n - self.whole(0, n // 2 + 1, case["batch"])


def _delta_inputs(case, seed):
    m, dt = _Maker(seed), DTYPES[case["dtype"]]
    b, n, hk, hv, dk, dv = (case[x] for x in ("batch", "new", "k_heads", "v_heads", "k_dim", "v_dim"))
    # what the convolution hands on: queries, keys and values side by side, behind a silu; texts dwell on their subjects
    mixed = m.normal(b, n, 2 * hk * dk + hv * dv) + 0.5 * m.normal(b, n // 48 + 2, 2 * hk * dk + hv * dv).repeat_interleave(48, 1)[:, 11:11 + n]
    mixed = (mixed * torch.sigmoid(mixed)).to(dt)
    step = torch.exp(m.uniform(math.log(1e-3), math.log(1e-1), hv))
    pad, lengths = m.paddings(case)
    return {"mixed": mixed, "a": m.normal(b, n, hv).to(dt), "b": m.normal(b, n, hv).to(dt), "a_log": torch.log(m.uniform(1.0, 16.0, hv)),
            "dt_bias": step + torch.log(-torch.expm1(-step)), "delta": 0.1 * m.normal(b, hv, dv, dk), "pad": pad, "lengths": lengths}


def _split(case, mixed):
    b, n, hk, hv, dk, dv = (case[x] for x in ("batch", "new", "k_heads", "v_heads", "k_dim", "v_dim"))
    q, k, v = mixed.split([hk * dk, hk * dk, hv * dv], -1)
    return q.unflatten(-1, (hk, dk)), k.unflatten(-1, (hk, dk)), v.unflatten(-1, (hv, dv))


def _conv_inputs(case, seed):
    m, dt = _Maker(seed), DTYPES[case["dtype"]]
    b, n, c = case["batch"], case["new"], case["channels"]
    pad, lengths = m.paddings(case)
    return {"x": m.normal(b, n, c).to(dt), "weight": (0.4 * m.normal(c, WIDTH)).to(dt), "window": m.normal(b, WIDTH - 1, c).to(dt),
            "pad": pad, "lengths": lengths}


def _logits(m, case):
    b, k, v = case["batch"], case["beams"], case["vocabulary"]
    x = 2.5 * m.normal(b, k, v)
    scores = -torch.sort(m.uniform(1.0, 25.0, b, k), -1).values  # hypotheses, best first
    return x.to(DTYPES[case["dtype"]]), scores


def _select_inputs(case, seed):
    m = _Maker(seed)
    x, scores = _logits(m, case)
    done = m.uniform(0, 1, case["batch"], case["beams"]) < 0.2 if case["done"] else None
    return {"logits": x, "scores": scores, "done": done}


def _beams_inputs(case, seed):
    m, dt = _Maker(seed), DTYPES[case["dtype"]]
    g, n, t, p = case["batch"], case["beams"], case["context"], case["shared"]
    rows, hq, hkv, d = g * n, case["q_heads"], case["kv_heads"], case["head_dim"]

    def context():
        x = torch.empty(rows, hkv, t, d, dtype=dt, device="cuda")
        x[:, :, :p] = m.normal(g, hkv, p, d).to(dt).repeat_interleave(n, 0)  # the hypotheses of one request share its prompt
        x[:, :, p:] = m.normal(rows, hkv, t - p, d).to(dt)
        return x

    state = {"keys": context(), "values": context(), "q": m.normal(rows, hq, 1, d).to(dt), "k": m.normal(rows, hkv, 1, d).to(dt),
             "v": m.normal(rows, hkv, 1, d).to(dt), "delta": None, "window": None, "logits": None, "scores": None, "order": None}
    if case["state_heads"]:
        h = case["state_heads"]
        state["delta"], state["window"] = 0.1 * m.normal(rows, h, 128, 128), m.normal(rows, WIDTH - 1, 2 * h * 128).to(dt)
    if case["vocabulary"]:
        state["logits"], state["scores"] = _logits(m, case)
    else:  # parents, the better hypotheses more often
        parent = (m.uniform(0, 1, g, n).square() * n).to(torch.int32).clamp(max=n - 1)
        state["order"] = (parent + n * torch.arange(g, device="cuda", dtype=torch.int32)[:, None]).flatten()
    return state


INPUTS = {"delta": _delta_inputs, "conv": _conv_inputs, "select": _select_inputs, "beams": _beams_inputs}


def prepare(case, seed):
    state = INPUTS[case["kind"]](case, seed)
    state["case"] = case
    if own and case["kind"] != "select":
        kvhip = _kvhip()
        if case["kind"] == "beams":
            state["cache"] = kvhip.KVCacheSimple()
            state["cache"].reserve(*state["k"].shape[:2], case["head_dim"], case["head_dim"], DTYPES[case["dtype"]], case["context"] + 1)
            state["cache"].update(state.pop("keys"), state.pop("values"), fetch=False)
        state["recurrent"] = kvhip.GatedDeltaCache(conv_width=WIDTH)
        state["recurrent"].window, state["recurrent"].delta_state = state.pop("window", None), state.pop("delta", None)
    return state


# ---- plain forms --------------------------------------------------------------------------------------------------
def _there(state, n):
    """Which of a call's tokens are there: [B, n], or None where all are."""
    if state["pad"] is None:
        return None
    at = torch.arange(n, device="cuda")
    return (at >= state["pad"][:, None]) & (at < state["lengths"][:, None])


def _delta_plain(state):
    """Chunks of 64 tokens: with the decays summed up inside a chunk, G, and A = beta e^(G_i - G_j) k_i k_j below the diagonal,
    the updates of a chunk are  u = (I + A)^-1 beta (v - e^G S k)."""
    case = state["case"]
    b, n, hk, hv = (case[x] for x in ("batch", "new", "k_heads", "v_heads"))
    q, k, v = (x.float() for x in _split(case, state["mixed"]))
    x = state["a"].float() + state["dt_bias"]
    decay = -torch.exp(state["a_log"]) * (x.clamp(min=0) + torch.log1p(torch.exp(-x.abs())))
    beta = 1 / (1 + torch.exp(-state["b"].float()))
    q = q * (case["k_dim"] ** -0.5 / torch.sqrt(q.square().sum(-1, keepdim=True) + EPS))
    k = k / torch.sqrt(k.square().sum(-1, keepdim=True) + EPS)
    there = _there(state, n)
    if there is not None:
        decay, beta = decay.masked_fill(~there[..., None], 0), beta.masked_fill(~there[..., None], 0)
        q, k, v = (x.masked_fill(~there[..., None, None], 0) for x in (q, k, v))
    c = min(CHUNK, n)
    chunks = (n + c - 1) // c

    def by_chunk(x, repeat=1):  # [B, n, H, ...] -> [B, H, chunks, c, ...]
        x = torch.nn.functional.pad(x.flatten(3) if x.dim() == 4 else x[..., None], (0, 0, 0, 0, 0, chunks * c - n))
        return x.unflatten(1, (chunks, c)).permute(0, 3, 1, 2, 4).repeat_interleave(repeat, 1).contiguous()

    q, k, v, beta = by_chunk(q, hv // hk), by_chunk(k, hv // hk), by_chunk(v), by_chunk(beta)
    total = by_chunk(decay.double()).cumsum(3)  # [B, Hv, chunks, c, 1]
    fade = torch.exp((total - total.transpose(-1, -2)).clamp(max=0).float()).tril()
    kt = k.transpose(-1, -2).contiguous()
    a = (torch.matmul(k, kt) * fade * beta).tril(-1)
    inverse = torch.eye(c, device="cuda").expand_as(a).contiguous()
    for i in range(1, c):
        inverse[..., i, :i] = -torch.matmul(a[..., i:i + 1, :i], inverse[..., :i, :i])[..., 0, :]
    scores = torch.matmul(q, kt) * fade
    rise, fall, last = torch.exp(total.float()), torch.exp((total[..., -1:, :] - total).float()), torch.exp(total[..., -1, 0].float())
    s = state["delta"].transpose(-1, -2).contiguous()  # [B, Hv, Dk, Dv]
    out = torch.empty_like(v)
    for i in range(chunks):
        u = torch.matmul(inverse[:, :, i], beta[:, :, i] * (v[:, :, i] - rise[:, :, i] * torch.matmul(k[:, :, i], s)))
        out[:, :, i] = rise[:, :, i] * torch.matmul(q[:, :, i], s) + torch.matmul(scores[:, :, i], u)
        s = last[:, :, i, None, None] * s + torch.matmul(kt[:, :, i], fall[:, :, i] * u)
    out = out.flatten(2, 3)[:, :, :n].transpose(1, 2)
    if there is not None:
        out = out.masked_fill(~there[..., None, None], 0)
    state["delta"] = s.transpose(-1, -2).contiguous()
    return [out.to(state["mixed"].dtype).contiguous(), state["delta"]]


def _conv_plain(state):
    x, n = state["x"], state["case"]["new"]
    there = _there(state, n)
    if there is None:
        every = torch.cat([state["window"], x], 1).float()
        at = torch.arange(n, device="cuda").expand(x.shape[0], n)
        ends = torch.full((x.shape[0],), n, device="cuda")
    else:  # each sequence's tokens move up behind its window
        pad = state["pad"].clamp(max=n)
        ends = (state["lengths"].clamp(max=n) - pad).clamp(min=0)
        at = torch.arange(n, device="cuda") - pad[:, None]
        source = (torch.arange(n, device="cuda") + pad[:, None]).clamp(max=n - 1)
        every = torch.cat([state["window"], x.gather(1, source[..., None].expand_as(x).long())], 1).float()
        at = at.clamp(min=0)
    acc = torch.zeros(x.shape, device="cuda")
    for w in range(WIDTH):
        tap = every[:, w:w + n] if there is None else every.gather(1, (at + w)[..., None].expand(x.shape).long())
        acc += tap * state["weight"][:, w].float()
    y = acc / (1 + torch.exp(-acc))
    if there is not None:
        y = y.masked_fill(~there[..., None], 0)
    keep = (ends[:, None] + torch.arange(WIDTH - 1, device="cuda"))[..., None].expand(-1, -1, x.shape[2])
    state["window"] = every.gather(1, keep.long()).to(x.dtype)
    return [y.to(x.dtype), state["window"]]


def _select_plain(state):
    case, x = state["case"], state["logits"].double()
    b, beams, count = case["batch"], case["beams"], case.get("count", case["beams"])
    top = x.amax(-1, keepdim=True)
    scores = x - top - torch.log(torch.exp(x - top).sum(-1, keepdim=True)) + state["scores"].double()[..., None]
    done = state.get("done")
    if done is not None:
        only = torch.full_like(scores, -math.inf)
        only[..., PAD_TOKEN] = state["scores"].double()
        scores = torch.where(done[..., None], only, scores)
    take = min(count, case["vocabulary"])
    best = torch.sort(scores, dim=-1, descending=True, stable=True)  # the best of each beam, then of all
    merged = torch.sort(best.values[..., :take].flatten(1), dim=-1, descending=True, stable=True)
    pick = merged.indices[:, :count]
    tokens = best.indices[..., :take].flatten(1).gather(1, pick)
    rows = torch.div(pick, take, rounding_mode="floor") + beams * torch.arange(b, device="cuda")[:, None]
    return [rows.to(torch.int32), tokens.to(torch.int32), merged.values[:, :count].float()]


def _beams_plain(state):
    case = state["case"]
    outs = _select_plain(state) if case["vocabulary"] else []
    order = outs[0].flatten().long() if outs else state["order"].long()
    p, hkv = case["shared"], case["kv_heads"]
    for name in ("keys", "values"):
        state[name][:, :, p:] = state[name][order, :, p:]
    for name in ("delta", "window"):
        if state[name] is not None:
            state[name] = state[name][order]
            outs.append(state[name])
    keys, values = torch.cat([state["keys"], state["k"]], 2).float(), torch.cat([state["values"], state["v"]], 2).float()
    q = state["q"].float().unflatten(1, (hkv, -1))[:, :, :, 0]  # [rows, Hkv, groups, D]
    s = torch.matmul(q, keys.transpose(-1, -2).contiguous()) * case["head_dim"] ** -0.5
    e = torch.exp(s - s.amax(-1, keepdim=True))
    out = torch.matmul(e, values) / e.sum(-1, keepdim=True)
    return outs + [out.flatten(1, 2)[:, :, None].to(state["q"].dtype)]


PLAIN = {"delta": _delta_plain, "conv": _conv_plain, "select": _select_plain, "beams": _beams_plain}


# ---- one pass -----------------------------------------------------------------------------------------------------
def run(state):
    case = state["case"]
    if not own:
        return PLAIN[case["kind"]](state)
    kvhip, recurrent = _kvhip(), state.get("recurrent")
    if case["kind"] == "delta":
        q, k, v = _split(case, state["mixed"])
        out = kvhip.gated_delta_update(q, k, v, state["a"], state["b"], state["a_log"], state["dt_bias"], recurrent,
                                       left_pad=state["pad"], lengths=state["lengths"])
        return [out, recurrent.delta_state]
    if case["kind"] == "conv":
        y = kvhip.causal_convolution(state["x"], state["weight"], recurrent, left_pad=state["pad"], lengths=state["lengths"])
        return [y, recurrent.window]
    if case["kind"] == "select":
        return list(kvhip.beam_select(state["logits"], state["scores"], count=case["count"], done=state["done"], pad_token=PAD_TOKEN))
    outs, cache, order = [], state["cache"], state["order"]
    if case["vocabulary"]:
        outs = list(kvhip.beam_select(state["logits"], state["scores"]))
        order = outs[0].flatten()
    cache.reorder(order, shared=case["shared"])
    if case["state_heads"]:
        recurrent.reorder(order)
        outs += [recurrent.delta_state, recurrent.window]
    outs.append(kvhip.attention_with_cache_update(state["q"], state["k"], state["v"], cache, case["head_dim"] ** -0.5))
    cache.trim(1)  # (so that a pass can be repeated)
    return outs


# ---- what a pass cannot do without --------------------------------------------------------------------------------
def work(case):
    size = 4.0 if case["dtype"] == "f32" else 2.0
    b = case["batch"]
    if case["kind"] == "delta":
        n, hk, hv, dk, dv = (case[x] for x in ("new", "k_heads", "v_heads", "k_dim", "v_dim"))
        tokens = b * n * (0.6 if case["ragged"] else 1.0)
        return {"bytes": size * (tokens * (2 * hk * dk + hv * dv + 2 * hv) + b * n * hv * dv) + 8.0 * b * hv * dk * dv,
                "flops": 6.0 * tokens * hv * dk * dv}
    if case["kind"] == "conv":
        n, c = case["new"], case["channels"]
        tokens = b * n * (0.6 if case["ragged"] else 1.0)
        return {"bytes": size * c * (tokens + b * n + 2.0 * b * (WIDTH - 1) + WIDTH), "flops": tokens * c * (2.0 * WIDTH + 4)}
    rows = b * case["beams"]
    choice = {"bytes": size * rows * case["vocabulary"], "flops": 4.0 * rows * case["vocabulary"]}
    if case["kind"] == "select":
        return {"bytes": choice["bytes"] + 4.0 * rows + 12.0 * b * case["count"], "flops": choice["flops"]}
    # of `beams` parents drawn evenly, how many rows change and how many distinct ones they come from
    k, t, p, hkv, d, h = (case[x] for x in ("beams", "context", "shared", "kv_heads", "head_dim", "state_heads"))
    moved = rows * (1 - 1 / k) + rows * (1 - (1 - 1 / k) ** k)
    cells = 2.0 * hkv * (t - p) * d * size + h * 128 * (128 * 4.0 + 2 * (WIDTH - 1) * size)
    attended = rows * (2.0 * hkv * (t + 1) * d + 2.0 * case["q_heads"] * d) * size
    return {"bytes": choice["bytes"] + moved * cells + attended, "flops": choice["flops"] + 4.0 * rows * case["q_heads"] * (t + 1) * d}


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------
def _exact_delta(case, given):
    q, k, v = (x.double() for x in _split(case, given["mixed"]))
    per = case["v_heads"] // case["k_heads"]
    n = case["new"]
    q = (q * case["k_dim"] ** -0.5 / (q * q).sum(-1, keepdim=True).add(EPS).sqrt()).repeat_interleave(per, 2)
    k = (k / (k * k).sum(-1, keepdim=True).add(EPS).sqrt()).repeat_interleave(per, 2)
    x = given["a"].double() + given["dt_bias"].double()
    g = torch.exp(-given["a_log"].double().exp() * torch.logaddexp(x, torch.zeros_like(x)))
    beta = torch.sigmoid(given["b"].double())
    s, out = given["delta"].double(), torch.zeros(v.shape, dtype=torch.float64, device="cuda")
    for t in range(n):
        faded = s * g[:, t, :, None, None]
        u = beta[:, t, :, None] * (v[:, t] - (faded * k[:, t, :, None, :]).sum(-1))
        new = torch.addcmul(faded, u[..., None], k[:, t, :, None, :])
        o = (new * q[:, t, :, None, :]).sum(-1)
        if given["pad"] is not None:
            here = (given["pad"] <= t) & (t < given["lengths"])
            new = torch.where(here[:, None, None, None], new, s)
            o = torch.where(here[:, None, None], o, 0.0)
        s, out[:, t] = new, o
    return [out.cpu().numpy(), s.cpu().numpy()]


def _exact_conv(case, given):
    n, ys, windows = case["new"], [], []
    for i in range(case["batch"]):
        first, end = (0, n) if given["pad"] is None else (int(given["pad"][i]), int(given["lengths"][i]))
        seen = torch.cat([given["window"][i], given["x"][i, first:max(end, first)]]).double()
        m = seen.shape[0] - (WIDTH - 1)
        y = torch.zeros(n, case["channels"], dtype=torch.float64, device="cuda")
        if m:
            z = sum(seen[w:w + m] * given["weight"][:, w].double() for w in range(WIDTH))
            y[first:end] = z * torch.sigmoid(z)
        ys.append(y)
        windows.append(seen[m:])
    return [torch.stack(ys).cpu().numpy(), torch.stack(windows).cpu().numpy()]


def _exact_select(case, given):
    rows, tokens, scores = [], [], []
    for i in range(case["batch"]):
        s = torch.log_softmax(given["logits"][i].double(), -1) + given["scores"][i].double()[:, None]
        if given.get("done") is not None:
            for k in torch.nonzero(given["done"][i]).flatten().tolist():
                s[k] = -math.inf
                s[k, PAD_TOKEN] = given["scores"][i, k].double()
        best = torch.sort(-s.flatten(), stable=True)
        at = best.indices[:case.get("count", case["beams"])]
        rows.append(i * case["beams"] + at // case["vocabulary"])
        tokens.append(at % case["vocabulary"])
        scores.append(-best.values[:len(at)])
    return [torch.stack(x) for x in (rows, tokens, scores)]


def _exact_beams(case, given):
    outs, order = [], given["order"]
    if case["vocabulary"]:
        outs = _exact_select(case, given)
        order = outs[0].flatten()
    outs = [x.cpu().numpy() for x in outs]
    order, p, groups = order.tolist(), case["shared"], case["q_heads"] // case["kv_heads"]
    outs += [torch.stack([given[name][r] for r in order]).double().cpu().numpy() for name in ("delta", "window") if given[name] is not None]
    attended = []
    for b, r in enumerate(order):
        k, v = (torch.cat([given[x][b, :, :p], given[x][r, :, p:], given[x[0]][b]], 1).double() for x in ("keys", "values"))
        q = given["q"][b, :, 0].double().unflatten(0, (-1, groups))
        w = torch.softmax((q[:, :, None, :] * k[:, None]).sum(-1) * case["head_dim"] ** -0.5, -1)
        attended.append((w[..., None] * v[:, None]).sum(2).flatten(0, 1)[:, None])
    return outs + [torch.stack(attended).cpu().numpy()]


def exact(case, seed):
    given = INPUTS[case["kind"]](case, seed)
    if case["kind"] == "delta":
        return _exact_delta(case, given)
    if case["kind"] == "conv":
        return _exact_conv(case, given)
    if case["kind"] == "select":
        return [x.cpu().numpy() for x in _exact_select(case, given)]
    return _exact_beams(case, given)
