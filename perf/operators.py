"""What is measured of the operators of a long, shared and pruned paged cache.

  prefix   one step's attention for groups of requests that share the first keys of their contexts
           (a system prompt, a document under many questions): the shared pages are read once a group
  mass     one step's attention that also adds up, for every cached key, the attention weight that
           the step's queries gave it
  evict    the choice of the keys that stay by that weight, and the move of their rows to the front of
           the request's pages

The cache is the engine's: pages [pages, kv heads, page size, head size], block tables of page ids with
-1 behind a request's last page, the fused projection of a step [tokens, (heads + 2 kv heads) * head size],
whose keys and values are in the pages already. Head counts and sizes are those of the benchmark's models (12 over 2, 28 over 4 and
40 over 8 heads of 128) and of the tests' (heads of 64 and 32). Lengths follow from the case
alone, what the tensors hold from the seed.

Fields of a case: op, dtype, heads, kv_heads, dim, page, requests, and

  prefix   groups (of `requests` requests each), prefix_low..prefix_high shared keys, own_low..own_high keys
           behind them (this step's among them), tokens each request brings
  mass     context_low..context_high keys, of which the step's tokens_low..tokens_high are the last
  evict    context_low..context_high keys, budget, keep_first, keep_last
"""

import math
import random

import numpy as np
import torch

own = False

KEY_STD = 0.8        # of cached keys and values, as a projection of normed rows gives them
QUERY_STD = 1.6      # scores then spread by 1.3: some keys of a long context stand out


def _prefix(name, heads, kv_heads, dim, groups, requests, prefix, own_keys, tokens=1, dtype="bfloat16", page=16):
    return dict(name=name, op="prefix", dtype=dtype, heads=heads, kv_heads=kv_heads, dim=dim, page=page, groups=groups, requests=requests,
                prefix_low=prefix[0], prefix_high=prefix[1], own_low=own_keys[0], own_high=own_keys[1], tokens=tokens)


def _mass(name, heads, kv_heads, dim, requests, context, tokens=(1, 1), dtype="bfloat16", page=16, keep_first=0):
    return dict(name=name, op="mass", dtype=dtype, heads=heads, kv_heads=kv_heads, dim=dim, page=page, requests=requests,
                context_low=context[0], context_high=context[1], tokens_low=tokens[0], tokens_high=tokens[1], keep_first=keep_first)


def _evict(name, kv_heads, dim, requests, context, budget, keep_first=4, keep_last=64, dtype="bfloat16", page=16):
    return dict(name=name, op="evict", dtype=dtype, heads=kv_heads, kv_heads=kv_heads, dim=dim, page=page, requests=requests,
                context_low=context[0], context_high=context[1], budget=budget, keep_first=keep_first, keep_last=keep_last)


def listed():
    return [
        # Four short chats under one instruction: a step as small as they come, where latency counts.
        _prefix("prefix_few", 12, 2, 128, 1, 4, (500, 500), (3, 90)),
        # A service's system prompt and examples under 64 conversations of unequal lengths.
        _prefix("prefix_serving", 28, 4, 128, 1, 64, (8000, 8000), (20, 700)),
        # Questions about a long document, each verified with drafted tokens, five a step.
        _prefix("prefix_document", 40, 8, 128, 1, 24, (30011, 30011), (100, 900), tokens=5),
        # Three tenants' prompts beside each other, small heads, larger pages.
        _prefix("prefix_groups", 14, 2, 64, 3, 41, (700, 2500), (1, 300), page=32),
        # The true 32-bit path.
        _prefix("prefix_float32", 12, 2, 64, 2, 8, (900, 1000), (1, 200), dtype="float32"),
        # One request, one token.
        _mass("mass_one", 12, 2, 128, 1, (700, 700)),
        # A decoding batch of unequal contexts; the first four keys are never given up and carry no weight.
        _mass("mass_serving", 28, 4, 128, 48, (300, 6000), keep_first=4),
        # Prompts of unequal lengths, the second and later portions of some.
        _mass("mass_prompt", 28, 4, 128, 3, (1500, 2900), tokens=(700, 1500)),
        # The true 32-bit path, a decoding batch.
        _mass("mass_float32", 12, 2, 64, 8, (100, 2100), dtype="float32"),
        # A small request goes back to its budget.
        _evict("evict_one", 2, 128, 1, (640, 640), 512),
        # A batch goes back to its budget; some requests are still below it.
        _evict("evict_serving", 4, 128, 48, (1900, 3900), 2048),
        # Long prompts cut down to a sixth.
        _evict("evict_long", 8, 128, 6, (50000, 64000), 10000, keep_first=16, keep_last=1000, page=64),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    most = {}
    for c in listed():
        w = work(c)
        most[c["op"]] = max(most.get(c["op"], 0.0), w["bytes"] / 6.5e12 + w["flops"] / 1.6e15)
    while True:
        op = rng.choice(["prefix", "mass", "evict"])
        dtype = "float32" if rng.random() < 0.2 else "bfloat16"
        heads, kv_heads, dim = rng.choice([(12, 2, 128), (28, 4, 128), (40, 8, 128), (14, 2, 64), (3, 1, 32), (8, 8, 64)])
        page = rng.choice([16, 16, 16, 32, 64])
        if op == "prefix":
            low = _log_int(rng, 100, 16000)
            own_low = _log_int(rng, 1, 300)
            tokens = rng.choice([1, 1, 1, 2, 5])
            c = _prefix("", heads, kv_heads, dim, rng.choice([1, 1, 2, 3]), _log_int(rng, 1, 80), (low, low + rng.randrange(max(1, low // 2))),
                        (own_low + tokens, own_low + tokens + _log_int(rng, 1, 600)), tokens, dtype, page)
        elif op == "mass":
            portion = rng.random() < 0.35
            t_low = _log_int(rng, 2, 800) if portion else 1
            t_high = t_low + rng.randrange(1 + t_low // 2) if portion else 1
            low = t_high + _log_int(rng, 1, 4000)
            c = _mass("", heads, kv_heads, dim, _log_int(rng, 1, 4 if portion else 48), (low, low + rng.randrange(1 + low)), (t_low, t_high), dtype, page,
                      rng.choice([0, 4, 33]))
        else:
            budget = _log_int(rng, 128, 8192)
            low = rng.randrange(budget // 2, 3 * budget)
            c = _evict("", kv_heads, dim, _log_int(rng, 1, 48), (low, low + rng.randrange(1, 3 * budget)), budget, rng.choice([0, 1, 4, 16]),
                       rng.randrange(0, budget // 2), dtype, page)
        del c["name"]
        w = work(c)
        floor = w["bytes"] / 6.5e12 + w["flops"] / (1.6e15 if dtype == "bfloat16" else 4e13)
        if floor <= most[op] and (dtype == "bfloat16" or w["flops"] < 2e9):
            return c


def _lengths(count, low, high, salt):
    """`count` lengths between low and high, the ends among them where there are two and more."""
    rng = random.Random(1000003 * salt + count)
    got = [low, high][:count] + [rng.randint(low, high) for _ in range(count - 2)]
    rng.shuffle(got)
    return got


def _shape(case):
    """What a case's lengths are: per request the keys in the cache after the step, the step's tokens, the shared keys."""
    if case["op"] == "prefix":
        shared = [n for n in _lengths(case["groups"], case["prefix_low"], case["prefix_high"], 1) for _ in range(case["requests"])]
        behind = _lengths(len(shared), max(case["own_low"], case["tokens"]), max(case["own_high"], case["tokens"]), 2)
        return [s + o for s, o in zip(shared, behind)], [case["tokens"]] * len(shared), shared
    contexts = _lengths(case["requests"], case["context_low"], case["context_high"], 3)
    if case["op"] == "mass":
        return contexts, _lengths(case["requests"], case["tokens_low"], case["tokens_high"], 4), [0] * len(contexts)
    return contexts, [0] * len(contexts), [0] * len(contexts)


def work(case):
    size = 2 if case["dtype"] == "bfloat16" else 4
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    kv_len, tokens, shared = _shape(case)
    if case["op"] == "evict":
        cut = [n for n in kv_len if n > case["budget"]]
        moved = sum(min(case["budget"], n) - case["keep_first"] for n in cut)
        read = 4 * kv_heads * sum(cut)
        return {"bytes": read + 4 * kv_heads * case["budget"] * len(kv_len) + 2 * kv_heads * moved * (2 * dim * size + 4), "flops": kv_heads * sum(cut)}
    rows = 2 * sum(tokens) * heads * dim * size                                        # queries in, outputs out
    pairs = sum(t * n - t * (t - 1) // 2 for t, n in zip(tokens, kv_len))              # (query, visible key)
    if case["op"] == "prefix":
        keys = sum(n - s for n, s in zip(kv_len, shared)) + sum(shared[:: case["requests"]])
        weights = 0
    else:
        keys = sum(kv_len)
        weights = 4 * kv_heads * sum(2 * (n - case["keep_first"]) - t for n, t in zip(kv_len, tokens))
    return {"bytes": rows + 2 * keys * kv_heads * dim * size + weights, "flops": 4 * dim * heads * pairs}


def _int32(values, device="cuda"):
    return torch.tensor(np.asarray(values, dtype=np.int32), device=device)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    dtype = getattr(torch, case["dtype"])
    heads, kv_heads, dim, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    kv_len, tokens, shared = _shape(case)
    seqs = len(kv_len)
    group = case["requests"] if case["op"] == "prefix" else 1
    # Pages: whole shared pages belong to a group, the rest to a request; a page that the border cuts is copied to each.
    whole = [s // page for s in shared]
    counts = [-(-n // page) for n in kv_len]
    total = sum(c - w for c, w in zip(counts, whole)) + sum(whole[::group]) + 1          # the last page is nobody's
    order = np.random.RandomState(int(seed) % (1 << 32)).permutation(total - 1).astype(np.int32)
    table = np.full((seqs, max(counts)), -1, dtype=np.int32)
    at = 0
    for b in range(seqs):
        if b % group == 0:
            common, at = order[at : at + whole[b]], at + whole[b]
        table[b, : whole[b]] = common
        table[b, whole[b] : counts[b]] = order[at : at + counts[b] - whole[b]]
        at += counts[b] - whole[b]

    def normal(std, *shape):
        return (torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32) * std).to(dtype)

    s = dict(case=case, heads=heads, kv_heads=kv_heads, dim=dim, page=page, max_kv_len=max(kv_len), block_table=_int32(table), kv_len=_int32(kv_len),
             keys=normal(KEY_STD, total, kv_heads, page, dim), values=normal(KEY_STD, total, kv_heads, page, dim))
    if case["op"] == "evict":
        # What a long run leaves: a few keys hold most of the weight; equal sums occur.
        s["mass"] = torch.randn((total, kv_heads, page), generator=gen, device="cuda").mul_(2).exp_().half().float()
        # The weights that move with their keys. The choice reads a copy that stays, so that every pass has the same work.
        s["moving"] = s["mass"].clone()
        return s
    s.update(q_start=_int32(np.concatenate(([0], np.cumsum(tokens)))), q_pos0=_int32([n - t for n, t in zip(kv_len, tokens)]), max_q_len=max(tokens),
             qkv=normal(QUERY_STD, sum(tokens), (heads + 2 * kv_heads) * dim), scale=dim ** -0.5)
    if case["op"] == "prefix":
        for b in range(0, seqs):       # the keys that the group shares in the page that the border cuts
            first, cut = b - b % group, shared[b] % page
            if cut and b != first:
                for pool in (s["keys"], s["values"]):
                    pool[int(table[b, whole[b]]), :, :cut] = pool[int(table[first, whole[b]]), :, :cut]
        s.update(prefix_len=_int32(shared), group_start=_int32(range(0, seqs + 1, group)), max_prefix_len=max(shared), max_group_tokens=sum(tokens[:group]),
                 max_own_len=max(n - p for n, p in zip(kv_len, shared)))
    else:
        # What some steps before gave a key: as much as this one.
        s["mass"] = torch.rand((total, kv_heads, page), generator=gen, device="cuda") * (2.0 * heads / kv_heads / max(kv_len))
    return s


# ----------------------------------------------------------------------------------- #
# the framework's operators

def _own_run(s):
    from paged_attention_engine_b200.kernels import ops

    op, case = s["case"]["op"], s["case"]
    if op == "evict":
        kept = ops.choose_kept(s["mass"], s["block_table"], s["kv_len"], case["budget"], case["keep_first"], case["keep_last"], s["max_kv_len"])
        ops.compact_kept(s["keys"], s["values"], s["moving"], s["block_table"], s["kv_len"], kept)
        return {"kept": kept, "keys": s["keys"], "values": s["values"], "mass": s["moving"]}
    sizes = (s["heads"], s["kv_heads"], s["dim"], s["page"])
    if op == "prefix":
        return {"out": ops.paged_attention_prefix(
            s["qkv"], s["keys"], s["values"], s["block_table"], s["q_start"], s["q_pos0"], s["kv_len"], s["prefix_len"], s["group_start"], *sizes,
            s["max_q_len"], s["max_prefix_len"], s["max_own_len"], s["max_group_tokens"], s["scale"])}
    out = ops.paged_attention_mass(s["qkv"], s["keys"], s["values"], s["mass"], s["block_table"], s["q_start"], s["q_pos0"], s["kv_len"], *sizes,
                                   s["max_q_len"], s["max_kv_len"], s["scale"], keep_first=case["keep_first"])
    return {"out": out, "mass": s["mass"]}


# ----------------------------------------------------------------------------------- #
# the plain forms

def _rows(pool, table):
    """The rows of the pages that `table` [n, width] names, in 32 bits: [n, kv heads, width * page, head size]."""
    got = pool[table.long()].float()
    n, width, kv_heads, page, dim = got.shape
    return got.permute(0, 2, 1, 3, 4).reshape(n, kv_heads, width * page, dim)


def _plain_prefix(s):
    case, heads, kv_heads, dim, page = s["case"], s["heads"], s["kv_heads"], s["dim"], s["page"]
    groups, requests, tokens, share = case["groups"], case["requests"], case["tokens"], heads // kv_heads
    seqs = groups * requests
    q = s["qkv"][:, : heads * dim].float().view(groups, requests * tokens, kv_heads, share, dim).transpose(1, 2)
    first = s["group_start"][:-1].long()
    # the shared keys, once a group
    shared_table = s["block_table"][first, : -(-s["max_prefix_len"] // page)]
    k, v = _rows(s["keys"], shared_table), _rows(s["values"], shared_table)
    q1 = q.reshape(groups, kv_heads, requests * tokens * share, dim)
    s1 = q1 @ k.transpose(2, 3) * s["scale"]
    j = torch.arange(k.shape[2], device="cuda")
    s1 = s1.masked_fill(j >= s["prefix_len"][first].view(-1, 1, 1, 1), -math.inf)
    # each request's own keys
    at = s["prefix_len"].long()[:, None] + torch.arange(s["max_own_len"], device="cuda")
    pages = s["block_table"].long().gather(1, (at // page).clamp(max=s["block_table"].shape[1] - 1))
    k2, v2 = (pool[pages, :, at % page].float().transpose(1, 2) for pool in (s["keys"], s["values"]))
    q2 = q1.view(groups, kv_heads, requests, tokens * share, dim).transpose(1, 2).reshape(seqs, kv_heads, tokens * share, dim)
    s2 = q2 @ k2.transpose(2, 3) * s["scale"]
    stand = (s["q_pos0"].long()[:, None] + torch.arange(tokens, device="cuda")).repeat_interleave(share, 1)
    s2 = s2.masked_fill(at[:, None, None, :] > stand[:, None, :, None], -math.inf)
    # one softmax over both
    s2g = s2.view(groups, requests, kv_heads, tokens * share, -1).transpose(1, 2).reshape(groups, kv_heads, requests * tokens * share, -1)
    top = torch.maximum(s1.amax(-1, keepdim=True), s2g.amax(-1, keepdim=True))
    e1, e2 = (s1 - top).exp(), (s2g - top).exp()
    o2 = e2.view(groups, kv_heads, requests, tokens * share, -1).transpose(1, 2).reshape(seqs, kv_heads, tokens * share, -1) @ v2
    o2 = o2.view(groups, requests, kv_heads, tokens * share, dim).transpose(1, 2).reshape(groups, kv_heads, requests * tokens * share, dim)
    out = (e1 @ v + o2) / (e1.sum(-1, keepdim=True) + e2.sum(-1, keepdim=True))
    out = out.view(groups, kv_heads, requests * tokens, share, dim).transpose(1, 2)
    return {"out": out.reshape(seqs * tokens, heads * dim).to(s["qkv"].dtype)}


def _plain_mass(s):
    case, heads, kv_heads, dim = s["case"], s["heads"], s["kv_heads"], s["dim"]
    share, longest, table = heads // kv_heads, s["max_q_len"], s["block_table"]
    t = torch.arange(longest, device="cuda")
    count = s["q_start"].long().diff()
    row = (s["q_start"].long()[:-1, None] + t).clamp(max=s["qkv"].shape[0] - 1)
    q = s["qkv"][:, : heads * dim].float()[row].view(-1, longest, kv_heads, share, dim).permute(0, 2, 1, 3, 4).flatten(2, 3)
    k, v = _rows(s["keys"], table), _rows(s["values"], table)
    scores = q @ k.transpose(2, 3) * s["scale"]
    j = torch.arange(k.shape[2], device="cuda")
    stand = (s["q_pos0"].long()[:, None] + t).repeat_interleave(share, 1)
    scores = scores.masked_fill(j > stand[:, None, :, None], -math.inf)
    e = (scores - scores.amax(-1, keepdim=True)).exp()
    w = e / e.sum(-1, keepdim=True)
    w = w * (t < count[:, None]).repeat_interleave(share, 1)[:, None, :, None]
    out = (w @ v).view(-1, kv_heads, longest, share, dim).transpose(1, 2).reshape(-1, longest, heads * dim)
    seq = torch.repeat_interleave(torch.arange(len(count), device="cuda"), count, output_size=s["qkv"].shape[0])
    out = out[seq, torch.arange(s["qkv"].shape[0], device="cuda") - s["q_start"].long()[seq]]
    # the weights' sums, added to what the keys had; this step's keys had nothing
    pages = table.long()
    old = s["mass"][pages].transpose(1, 2).flatten(2)                        # [requests, kv heads, keys]
    new = torch.where(j >= s["q_pos0"].view(-1, 1, 1), 0.0, old) + w.sum(2)
    new = torch.where((j >= case["keep_first"]) & (j < s["kv_len"].view(-1, 1, 1)), new, old)
    s["mass"][pages] = new.view(*new.shape[:2], table.shape[1], -1).transpose(1, 2)
    return {"out": out.to(s["qkv"].dtype), "mass": s["mass"]}


def _plain_evict(s):
    case, table, page = s["case"], s["block_table"].long(), s["page"]
    budget = case["budget"]
    mass = s["mass"][table].transpose(1, 2).flatten(2)                       # [requests, kv heads, keys]
    j, n = torch.arange(mass.shape[2], device="cuda"), s["kv_len"].long().view(-1, 1, 1)
    mass = torch.where((j < case["keep_first"]) | (j >= n - case["keep_last"]), math.inf, mass)
    mass = torch.where(j < n, mass, -math.inf)
    best = mass.sort(dim=2, descending=True, stable=True).indices[:, :, :budget]
    place = torch.arange(best.shape[2], device="cuda")
    best = torch.where(place < n, best, mass.shape[2]).sort(2).values
    kept = torch.where(place < n, best, -1)
    if kept.shape[2] < budget:
        kept = torch.cat((kept, kept.new_full((*kept.shape[:2], budget - kept.shape[2]), -1)), 2)
    # row kept[i] goes to place i; where nothing is kept a row is written over itself
    to = torch.arange(budget, device="cuda").expand_as(kept)
    source = torch.where(kept >= 0, kept, to)
    width = table.shape[1]

    def places(i):
        at = (i // page).clamp(max=width - 1)
        return table[:, None].expand(-1, kept.shape[1], -1).gather(2, at), i % page

    head = torch.arange(kept.shape[1], device="cuda").view(1, -1, 1)
    (sp, so), (tp, to_) = places(source), places(to)
    for pool in (s["keys"], s["values"], s["moving"]):
        pool[tp, head, to_] = pool[sp, head, so]
    return {"kept": kept.int(), "keys": s["keys"], "values": s["values"], "mass": s["moving"]}


def run(state):
    if own:
        return _own_run(state)
    return {"prefix": _plain_prefix, "mass": _plain_mass, "evict": _plain_evict}[state["case"]["op"]](state)


# ----------------------------------------------------------------------------------- #
# the definition, request by request, in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    kv_len, tokens, _ = _shape(case)
    heads, kv_heads, dim, page = s["heads"], s["kv_heads"], s["dim"], s["page"]
    if case["op"] == "evict":
        budget = case["budget"]
        kept = np.full((len(kv_len), kv_heads, budget), -1, dtype=np.int32)
        table, mass = s["block_table"].cpu().numpy(), s["mass"].cpu().numpy()
        for b, n in enumerate(kv_len):
            rows = np.concatenate([mass[p] for p in table[b, : -(-n // page)]], axis=1)[:, :n]
            for g in range(kv_heads):
                order = sorted(range(case["keep_first"], n - case["keep_last"]), key=lambda i: (-rows[g, i], i))
                chosen = list(range(n)) if n <= budget else sorted(
                    [*range(case["keep_first"]), *order[: budget - case["keep_first"] - case["keep_last"]], *range(n - case["keep_last"], n)])
                kept[b, g, : len(chosen)] = chosen
        return {"kept": torch.from_numpy(kept), "keys": None, "values": None, "mass": None}
    out = torch.empty(s["qkv"].shape[0], heads, dim, dtype=torch.float64, device="cuda")
    mass = s["mass"].double() if case["op"] == "mass" else None
    start = 0
    for b, (n, t) in enumerate(zip(kv_len, tokens)):
        pages = s["block_table"][b, : -(-n // page)].long()
        for g in range(kv_heads):
            k, v = (pool[pages, g].reshape(-1, dim)[:n].double() for pool in (s["keys"], s["values"]))
            visible = torch.arange(n, device="cuda")[None, :] <= torch.arange(n - t, n, device="cuda")[:, None]
            total = torch.zeros(n, dtype=torch.float64, device="cuda")
            for h in range(g * heads // kv_heads, (g + 1) * heads // kv_heads):
                q = s["qkv"][start : start + t, h * dim : (h + 1) * dim].double()
                w = torch.softmax((q @ k.T * dim ** -0.5).masked_fill(~visible, -math.inf), -1)
                out[start : start + t, h] = w @ v
                total += w.sum(0)
            if mass is not None:
                j = torch.arange(n, device="cuda")
                p, o = pages[j // page], j % page
                old = torch.where(j < n - t, mass[p, g, o], 0.0)
                chosen = j >= case["keep_first"]
                mass[p[chosen], g, o[chosen]] = (old + total)[chosen]
        start += t
    return {"out": out.view(out.shape[0], -1)} if mass is None else {"out": out.view(out.shape[0], -1), "mass": mass}
