"""Workloads of the device-pointer operators: packed prompt attention, attention over a shared prefix, logit adjustment.

Each case is one call as a serving loop makes it.  ``run`` computes it with the library's entry points when ``own`` is
true and in elementary 32-bit torch operations when it is not; ``exact`` computes it from the definition in 64 bits.
"""
import math
import random

import torch

own = False

_DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_ops = None


def _device_ops():
    """The backend and its operators, created once as a user's program does."""
    global _ops
    if _ops is None:
        from funasrnet_b200.backend import CudaFloatBackend
        from funasrnet_b200.device_ops import DeviceOps

        _ops = DeviceOps(CudaFloatBackend(torch.cuda.current_device()))
    return _ops


# ------------------------------------------------------------------------------------------------ cases ----


def listed():
    def prompts(name, dtype, heads, kv_heads, head, seqs, new, past, mix, causal=True):
        return {"name": name, "op": "prompts", "dtype": dtype, "heads": heads, "kv_heads": kv_heads, "head": head,
                "seqs": seqs, "new_lo": new[0], "new_hi": new[1], "past_lo": past[0], "past_hi": past[1],
                "causal": causal, "mix": mix}

    def shared(name, dtype, heads, kv_heads, head, seqs, prefix, suffix, mix):
        return {"name": name, "op": "shared", "dtype": dtype, "heads": heads, "kv_heads": kv_heads, "head": head,
                "seqs": seqs, "prefix": prefix, "suffix_lo": suffix[0], "suffix_hi": suffix[1], "mix": mix}

    def logits(name, dtype, rows, vocab, history, biases, masks, mix):
        return {"name": name, "op": "logits", "dtype": dtype, "rows": rows, "vocab": vocab, "history_lo": history[0],
                "history_hi": history[1], "biases": biases, "masks": masks, "mix": mix}

    return [
        # One short utterance of 37 frames prefilled alone: a single call whose latency the user waits for.
        prompts("prompt_37", "f16", 16, 8, 128, 1, (37, 37), (0, 0), 1),
        # Twenty-four utterances of ragged lengths prefilled in one call, as a server collects them.
        prompts("prompts_mixed", "bf16", 16, 8, 128, 24, (1, 700), (0, 0), 2),
        # Two long transcripts prefilled whole: the compute-bound end.
        prompts("prompts_long", "bf16", 16, 8, 128, 2, (8192, 8192), (0, 0), 3),
        # The next chunk of five sessions with a history each, smaller heads in wide groups.
        prompts("chunks_on_history", "f16", 32, 4, 64, 5, (33, 256), (3001, 20000), 4),
        # Frames that see one another in both directions (an audio prefix), a head size between the usual ones.
        prompts("frames_both_ways", "f16", 12, 12, 80, 9, (100, 1500), (0, 0), 5, causal=False),
        # Two sessions right after a short prompt: latency.
        shared("shared_small", "f16", 16, 8, 128, 2, 61, (0, 7), 6),
        # Sixty-four sessions that share a prompt, each with its own audio frames and text so far.
        shared("shared_64", "f16", 16, 8, 128, 64, 2048, (1, 664), 7),
        # One session on a very long shared document: the prefix is all there is to read.
        shared("shared_one_long", "bf16", 32, 8, 128, 1, 65537, (40, 40), 8),
        # A large batch on a long shared prompt.
        shared("shared_256", "bf16", 16, 8, 128, 256, 16384, (100, 900), 9),
        # One session's next token with a short history: latency.
        logits("logits_one", "f32", 1, 151936, (20, 20), 12, False, 10),
        # A batch of sessions with hot-word biases and grammars on some.
        logits("logits_64", "bf16", 64, 151936, (0, 700), 100, True, 11),
        # A large batch with long histories.
        logits("logits_256", "f32", 256, 151936, (1000, 9000), 40, True, 12),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["prompts", "shared", "logits"])
    if op == "logits":
        rows = _log_int(rng, 1, 256)
        lo = _log_int(rng, 1, 4000) - 1
        return {"op": op, "dtype": rng.choice(["f32", "f16", "bf16"]), "rows": rows, "vocab": _log_int(rng, 997, 151936),
                "history_lo": lo, "history_hi": lo + _log_int(rng, 1, 5000), "biases": _log_int(rng, 1, 200) - 1,
                "masks": rng.random() < 0.6, "mix": rng.randrange(1 << 30)}
    heads, kv_heads = rng.choice([(16, 8), (16, 16), (32, 4), (14, 2), (12, 4), (24, 8), (32, 8), (8, 1), (20, 4)])
    case = {"op": op, "dtype": rng.choice(["f16", "bf16"]), "heads": heads, "kv_heads": kv_heads,
            "head": rng.choice([128, 128, 64, 64, 80, 96, 112, 32]), "mix": rng.randrange(1 << 30)}
    if op == "shared":
        lo = _log_int(rng, 1, 700) - 1
        case.update(seqs=_log_int(rng, 1, 256), prefix=_log_int(rng, 1, 16384), suffix_lo=lo,
                    suffix_hi=lo + _log_int(rng, 1, 900))
        return case
    total = _log_int(rng, 1, 8192)
    seqs = min(_log_int(rng, 1, 64), total)
    longest = max(1, 2 * total // seqs)
    past = _log_int(rng, 1, 8192) - 1 if rng.random() < 0.4 else 0
    case.update(seqs=seqs, new_lo=max(0, 2 * (total // seqs) - longest), new_hi=longest, past_lo=past // 3, past_hi=past,
                causal=rng.random() < 0.8)
    while seqs * case["heads"] * longest * (longest + past) > 2 * 16 * 8192 * 8192:  # at most the long listed case
        longest = case["new_hi"] = longest // 2
        case["new_lo"] = min(case["new_lo"], longest)
    return case


def _prompt_lengths(case):
    """(new tokens, keys) of every sequence; a function of the case alone."""
    rng = random.Random(case["mix"])
    new = [rng.randint(case["new_lo"], case["new_hi"]) for _ in range(case["seqs"])]
    past = [rng.randint(case["past_lo"], case["past_hi"]) for _ in range(case["seqs"])]
    if sum(new) == 0:
        new[0] = 1
    return new, [a + b for a, b in zip(new, past)]


def _suffix_lengths(case):
    rng = random.Random(case["mix"])
    return [rng.randint(case["suffix_lo"], case["suffix_hi"]) for _ in range(case["seqs"])]


def _history_lengths(case):
    """(all tokens, of which prompt) of every row."""
    rng = random.Random(case["mix"])
    every = [rng.randint(case["history_lo"], case["history_hi"]) for _ in range(case["rows"])]
    return every, [rng.randint(0, n) for n in every]


def _mask_choice(case):
    """The mask table's rows, and each logit row's place in it (-1: none)."""
    rng = random.Random(case["mix"] + 1)
    table = max(1, min(8, case["rows"]))
    return table, [rng.randint(-1, table - 1) for _ in range(case["rows"])]


def _sums(lengths):
    total = [0]
    for n in lengths:
        total.append(total[-1] + n)
    return total


# ---------------------------------------------------------------------------------------------- prepare ----


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator(device=dev).manual_seed(seed)
    dtype = _DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=dev)

    def ints(values):
        return torch.tensor(values, dtype=torch.int32, device=dev)

    state = {"op": case["op"]}
    if case["op"] == "logits":
        rows, vocab = case["rows"], case["vocab"]
        every, prompt = _history_lengths(case)
        logits = normal(rows, vocab) * 2.5
        near = torch.randint(0, vocab, (rows, 24), generator=gen, device=dev)
        logits.scatter_add_(1, near, 5.0 + normal(rows, 24))
        off = _sums(every)
        # Spoken text repeats a small set of tokens; most of a history comes from one.
        pool = torch.randint(0, vocab, (300,), generator=gen, device=dev)
        pool[:24] = near[0]
        pick = (torch.rand(off[-1], generator=gen, device=dev) ** 2 * 300).long()
        state.update(logits=logits.to(dtype), out=torch.zeros(rows, vocab, dtype=dtype, device=dev),
                     tokens=torch.zeros(rows, dtype=torch.int32, device=dev), history=pool[pick].to(torch.int32),
                     history_offsets=ints(off), prompt_lens=ints(prompt),
                     repetition=1.0 + 0.3 * torch.rand(rows, generator=gen, device=dev),
                     presence=0.4 * torch.rand(rows, generator=gen, device=dev),
                     frequency=0.2 * torch.rand(rows, generator=gen, device=dev))
        if case["biases"]:
            n = case["biases"]
            state.update(bias_tokens=torch.randint(0, vocab, (rows * n,), generator=gen, device=dev).to(torch.int32),
                         bias_values=normal(rows * n) * 3, bias_offsets=ints([n * i for i in range(rows + 1)]))
        else:
            state.update(bias_tokens=None, bias_values=None, bias_offsets=None)
        if case["masks"]:
            table, place = _mask_choice(case)
            words = torch.randint(-2 ** 31, 2 ** 31, (2, table, (vocab + 31) // 32), generator=gen, device=dev)
            state.update(mask=(words[0] & words[1]).to(torch.int32), mask_rows=ints(place))
        else:
            state.update(mask=None, mask_rows=None)
        return state

    heads, kv_heads, head = case["heads"], case["kv_heads"], case["head"]
    gain = 0.5 + torch.rand(head, generator=gen, device=dev)  # the key norm's weight

    def keys(*shape):
        return (normal(*shape, kv_heads, head) * gain).to(dtype)

    def values(*shape):
        return normal(*shape, kv_heads, head).to(dtype)

    if case["op"] == "prompts":
        new, every = _prompt_lengths(case)
        rows = sum(new)
        state.update(causal=case["causal"], q_offsets=ints(_sums(new)), k_offsets=ints(_sums(every)), most_new=max(new),
                     most_keys=max(every), k=keys(sum(every)), v=values(sum(every)))
    else:
        rows = case["seqs"]
        own_lens = _suffix_lengths(case)
        cap = max(1, max(own_lens))
        # Rows behind a sequence's length hold what an earlier sequence left there.
        state.update(prefix_k=keys(case["prefix"]), prefix_v=values(case["prefix"]), suffix_k=keys(rows, cap),
                     suffix_v=values(rows, cap), suffix_lens=ints(own_lens))
    state.update(q=normal(rows, heads, head).to(dtype), out=torch.zeros(rows, heads, head, dtype=dtype, device=dev),
                 lse=torch.zeros(rows, heads, device=dev), scale=1.0 / math.sqrt(head))
    return state


# -------------------------------------------------------------------------------------------------- run ----


def run(state):
    if own:
        return _run_own(state)
    return {"prompts": _plain_prompts, "shared": _plain_shared, "logits": _plain_logits}[state["op"]](state)


def _run_own(s):
    ops = _device_ops()
    stream = torch.cuda.current_stream().cuda_stream
    if s["op"] == "logits":
        ops.adjust_logits(s["logits"], s["out"], s["tokens"], history=s["history"], history_offsets=s["history_offsets"],
                          prompt_lens=s["prompt_lens"], repetition=s["repetition"], presence=s["presence"],
                          frequency=s["frequency"], bias_tokens=s["bias_tokens"], bias_values=s["bias_values"],
                          bias_offsets=s["bias_offsets"], mask=s["mask"], mask_rows=s["mask_rows"], stream=stream)
        return {"logits": s["out"], "tokens": s["tokens"]}
    packed = s["op"] == "prompts"
    if "workspace" not in s:  # a program allocates it once for its largest call
        size = (ops.attention_packed_workspace(s["q"], s["k"], s["q_offsets"]) if packed else
                ops.attention_shared_workspace(s["q"], s["prefix_k"], s["suffix_k"]))
        s["workspace"] = torch.empty(max(16, size), dtype=torch.uint8, device=s["q"].device)
    if packed:
        ops.attention_packed(s["q"], s["k"], s["v"], s["q_offsets"], s["k_offsets"], s["out"], causal=s["causal"],
                             scale=s["scale"], lse=s["lse"], workspace=s["workspace"], stream=stream)
    else:
        ops.attention_shared(s["q"], s["prefix_k"], s["prefix_v"], s["suffix_k"], s["suffix_v"], s["suffix_lens"],
                             s["out"], scale=s["scale"], lse=s["lse"], workspace=s["workspace"], stream=stream)
    return {"out": s["out"], "lse": s["lse"]}


def _softmax_parts(scores):
    """exp(scores - max) in place, its sum and the log of the sum of exponentials; rows of -inf give zeros and -inf."""
    top = scores.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = scores.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    return p, total, (total.log() + top).squeeze(-1)


def _plain_prompts(s):
    q, heads, head = s["q"], s["q"].shape[1], s["q"].shape[2]
    kv_heads = s["k"].shape[1]
    group = heads // kv_heads
    qo, ko = s["q_offsets"].long(), s["k_offsets"].long()
    new, every = qo.diff(), ko.diff()
    n, mq, mk = new.numel(), s["most_new"], max(1, s["most_keys"])
    i, j = torch.arange(mq, device=q.device), torch.arange(mk, device=q.device)
    has_q, has_k = i < new[:, None], j < every[:, None]
    rows_q = torch.where(has_q, qo[:-1, None] + i, 0)
    rows_k = torch.where(has_k, ko[:-1, None] + j, 0)
    # [n, kv_heads, group * mq, head] and [n, kv_heads, mk, head]
    qp = q[rows_q].float().view(n, mq, kv_heads, group, head).permute(0, 2, 3, 1, 4).reshape(n, kv_heads, group * mq, head)
    zero = ~has_k[:, None, :, None]
    kp = s["k"][rows_k].float().permute(0, 2, 1, 3).masked_fill(zero, 0.0)
    vp = s["v"][rows_k].float().permute(0, 2, 1, 3).masked_fill(zero, 0.0)
    seen = has_k[:, None, :].expand(n, mq, mk)
    if s["causal"]:
        seen = seen & (j <= i[:, None] + (every - new)[:, None, None])
    scores = torch.matmul(qp, kp.transpose(-1, -2)).mul_(s["scale"]).view(n, kv_heads, group, mq, mk)
    scores.masked_fill_(~seen[:, None, None], -math.inf)
    p, total, lse = _softmax_parts(scores)
    out = torch.matmul(p.view(n, kv_heads, group * mq, mk), vp).view(n, kv_heads, group, mq, head)
    out = out / torch.where(total == 0, 1.0, total)
    # Back to packed rows: row t is token t - qo[b] of sequence b.
    t = torch.arange(q.shape[0], device=q.device)
    b = torch.searchsorted(qo[1:].contiguous(), t, right=True)
    at = t - qo[b]
    out = out.permute(0, 3, 1, 2, 4)[b, at].reshape(q.shape)
    lse = lse.permute(0, 3, 1, 2)[b, at].reshape(q.shape[0], heads)
    return {"out": out.to(q.dtype), "lse": lse}


def _plain_shared(s):
    q = s["q"]
    n, heads, head = q.shape
    kv_heads = s["prefix_k"].shape[1]
    group, prefix, cap = heads // kv_heads, s["prefix_k"].shape[0], s["suffix_k"].shape[1]
    qf = q.float().view(n, kv_heads, group, head)
    by_head = qf.permute(1, 0, 2, 3).reshape(kv_heads, n * group, head)
    unused = torch.arange(cap, device=q.device) >= s["suffix_lens"][:, None]
    ks = s["suffix_k"].float().permute(0, 2, 1, 3).masked_fill(unused[:, None, :, None], 0.0)
    vs = s["suffix_v"].float().permute(0, 2, 1, 3).masked_fill(unused[:, None, :, None], 0.0)
    on_prefix = torch.matmul(by_head, s["prefix_k"].float().permute(1, 2, 0))
    on_prefix = on_prefix.view(kv_heads, n, group, prefix).permute(1, 0, 2, 3)
    on_suffix = torch.matmul(qf, ks.transpose(-1, -2)).masked_fill(unused[:, None, None, :], -math.inf)
    p, total, lse = _softmax_parts(torch.cat([on_prefix, on_suffix], -1).mul_(s["scale"]))
    of_prefix = p[..., :prefix].permute(1, 0, 2, 3).reshape(kv_heads, n * group, prefix)
    out = torch.matmul(of_prefix, s["prefix_v"].float().permute(1, 0, 2)).view(kv_heads, n, group, head).permute(1, 0, 2, 3)
    out = (out + torch.matmul(p[..., prefix:], vs)) / torch.where(total == 0, 1.0, total)
    return {"out": out.reshape(n, heads, head).to(q.dtype), "lse": lse.reshape(n, heads)}


def _plain_logits(s):
    x = s["logits"].float()
    rows, vocab = x.shape
    off = s["history_offsets"].long()
    at = torch.arange(s["history"].numel(), device=x.device)
    row = torch.searchsorted(off[1:].contiguous(), at, right=True)
    made = (at - off[row] >= s["prompt_lens"][row]).int()
    place = row * vocab + s["history"].long()
    every = torch.zeros(rows * vocab, dtype=torch.int32, device=x.device).scatter_add_(0, place, torch.ones_like(made))
    count = torch.zeros(rows * vocab, dtype=torch.int32, device=x.device).scatter_add_(0, place, made)
    every, count = every.view(rows, vocab), count.view(rows, vocab)
    r = s["repetition"][:, None]
    x = torch.where(every > 0, torch.where(x > 0, x / r, x * r), x)
    less = s["frequency"][:, None] * count.float() + s["presence"][:, None]
    x = torch.where(count > 0, x - less, x)
    if s["bias_tokens"] is not None:  # of several entries for one token the last counts
        e = torch.arange(s["bias_tokens"].numel(), device=x.device)
        row = torch.searchsorted(s["bias_offsets"].long()[1:].contiguous(), e, right=True)
        last = torch.full((rows * vocab,), -1, dtype=torch.int64, device=x.device)
        last = last.scatter_reduce_(0, row * vocab + s["bias_tokens"].long(), e, "amax").view(rows, vocab)
        x = torch.where(last >= 0, x + s["bias_values"][last.clamp(min=0)], x)
    if s["mask"] is not None:
        v = torch.arange(vocab, device=x.device)
        allowed = (s["mask"][:, v >> 5] >> (v & 31)) & 1
        allowed = (allowed[s["mask_rows"].clamp(min=0).long()] != 0) | (s["mask_rows"] < 0)[:, None]
        x = torch.where(allowed, x, -math.inf)
    top = x.amax(-1, keepdim=True)
    v = torch.arange(vocab, dtype=torch.int32, device=x.device)
    first = torch.where(x == top, v, vocab).amin(-1)
    return {"logits": x.to(s["logits"].dtype),
            "tokens": torch.where(top.squeeze(-1) > -math.inf, first, -1).to(torch.int32)}


# ------------------------------------------------------------------------------------------------- work ----


def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "logits":
        rows, vocab = case["rows"], case["vocab"]
        moved = 2 * rows * vocab * size + 4 * sum(_history_lengths(case)[0]) + 8 * rows * case["biases"] + 28 * rows
        flops = 2 * rows * vocab
        if case["masks"]:
            table, place = _mask_choice(case)
            moved += 4 * len({p for p in place if p >= 0}) * ((vocab + 31) // 32)
        return {"bytes": moved, "flops": flops}
    heads, kv_heads, head = case["heads"], case["kv_heads"], case["head"]
    if case["op"] == "shared":
        mine = _suffix_lengths(case)
        rows, keys = case["seqs"], case["prefix"] + sum(mine)
        pairs = case["seqs"] * case["prefix"] + sum(mine)
    else:
        new, every = _prompt_lengths(case)
        rows, keys = sum(new), sum(every)
        # Causal: row i of L sees (keys - L) + i + 1 of them.
        pairs = sum(a * (b - a) + a * (a + 1) // 2 if case["causal"] else a * b for a, b in zip(new, every))
    return {"bytes": rows * heads * (2 * head * size + 4) + 2 * keys * kv_heads * head * size,
            "flops": 4 * heads * head * pairs}


# ------------------------------------------------------------------------------------------------ exact ----


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "logits":
        return _exact_logits(case, s)
    q = s["q"].double()
    out, lse = torch.zeros_like(q), torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device=q.device)
    group = case["heads"] // case["kv_heads"]

    def attend(rows, k, v, past):
        """rows: slice of queries; k, v [keys, kv_heads, head]; past: None, or how many keys the first query sees less one."""
        for h in range(case["heads"]):
            for a in range(rows.start, rows.stop, 4096):
                part = slice(a, min(rows.stop, a + 4096))
                z = (q[part, h] @ k[:, h // group].double().T) * s["scale"]
                if past is not None:
                    see = torch.arange(part.start - rows.start, part.stop - rows.start, device=q.device) + past
                    z = z.masked_fill(torch.arange(k.shape[0], device=q.device) > see[:, None], -math.inf)
                if k.shape[0]:
                    lse[part, h] = torch.logsumexp(z, -1)
                    out[part, h] = torch.nan_to_num(torch.softmax(z, -1), nan=0.0) @ v[:, h // group].double()

    if case["op"] == "prompts":
        new, every = _prompt_lengths(case)
        qo, ko = _sums(new), _sums(every)
        for b in range(case["seqs"]):
            attend(slice(qo[b], qo[b + 1]), s["k"][ko[b]:ko[b + 1]], s["v"][ko[b]:ko[b + 1]],
                   every[b] - new[b] if case["causal"] else None)
    else:
        for b, n in enumerate(_suffix_lengths(case)):
            k = torch.cat([s["prefix_k"], s["suffix_k"][b, :n]])
            v = torch.cat([s["prefix_v"], s["suffix_v"][b, :n]])
            g = k.double().permute(1, 0, 2)
            z = torch.einsum("hgd,hkd->hgk", q[b].view(case["kv_heads"], group, -1), g) * s["scale"]
            lse[b] = torch.logsumexp(z, -1).reshape(-1)
            out[b] = torch.einsum("hgk,khd->hgd", torch.softmax(z, -1), v.double()).reshape(case["heads"], -1)
    return {"out": out, "lse": lse}


def _exact_logits(case, s):
    x = s["logits"].double()
    every, prompt = _history_lengths(case)
    off = _sums(every)
    for b in range(case["rows"]):
        seen = s["history"][off[b]:off[b + 1]].long()
        token, count = torch.unique(seen[prompt[b]:], return_counts=True)
        any_token = torch.unique(seen)
        r, p, f = (s[k][b].double() for k in ("repetition", "presence", "frequency"))
        old = x[b, any_token]
        x[b, any_token] = torch.where(old > 0, old / r, old * r)
        x[b, token] -= f * count + p
    if case["biases"]:
        n = case["biases"]
        tokens, amounts = s["bias_tokens"].view(-1, n).cpu().tolist(), s["bias_values"].view(-1, n).double().cpu().tolist()
        for b in range(case["rows"]):
            table = dict(zip(tokens[b], amounts[b]))
            at = torch.tensor(list(table), device=x.device)
            x[b, at] += torch.tensor(list(table.values()), dtype=torch.float64, device=x.device)
    if case["masks"]:
        _, place = _mask_choice(case)
        bits = (s["mask"][:, :, None] >> torch.arange(32, dtype=torch.int32, device=x.device)) & 1
        bits = bits.reshape(bits.shape[0], -1)[:, :case["vocab"]].bool()
        for b, p in enumerate(place):
            if p >= 0:
                x[b, ~bits[p]] = -math.inf
    best, token = x.max(-1)
    first = (x == best[:, None]).int().argmax(-1)
    return {"logits": x, "tokens": torch.where(best > -math.inf, first, -1)}
