"""Cases for the paged key-value cache: storing tokens into pages, attention of one
new token per sequence over the pages, and eviction by accumulated attention weight.

Each case has a plain form in elementary torch operations and the calls a user of the
library makes (`own`).  A sequence's cache is a row of page ids and a length; keys and
values lie in pages [pages][key_heads][page][head size], f32 or bf16; one f32 weight per
cached token and key head, [pages][key_heads][page], sums the attention it has drawn.
"""
import math

import torch

own = False

# What every case has: op, n (sequences), longest (the longest sequence's cached tokens),
# ragged (lengths from idle to longest, or all alike), key_heads, dh, page, bf16 (page type).
# attend: heads, reach (visible last tokens; 0 for all), weights (accumulate attention).
# store: m (tokens per sequence).  evict: keep, sinks, recent.


def _case(op, n, longest, ragged, key_heads, dh, page, bf16, **more):
    return dict(op=op, n=n, longest=longest, ragged=ragged, key_heads=key_heads, dh=dh, page=page, bf16=bf16, **more)


def listed():
    return [
        # One short chat turn on the 12-head model with 4 key heads: the latency of a call.
        dict(_case("attend", 1, 97, False, 4, 64, 16, False, heads=12, reach=0, weights=False), name="attend short"),
        # The same model's global layer after a 16384-token prompt, one user.
        dict(_case("attend", 1, 16389, False, 4, 64, 64, False, heads=12, reach=0, weights=False), name="attend one long"),
        # 64 users of that model, a few thousand tokens each, joined and left at different times.
        dict(_case("attend", 64, 4352, True, 4, 64, 16, False, heads=12, reach=0, weights=False), name="attend batch"),
        # A serving batch of a wider model with bf16 pages: 4 query heads per key head, ragged, idle rows.
        dict(_case("attend", 48, 16000, True, 8, 128, 16, True, heads=32, reach=0, weights=False), name="attend batch bf16"),
        # Eight long documents, bf16 pages: the largest call.
        dict(_case("attend", 8, 65536, False, 8, 128, 64, True, heads=32, reach=0, weights=False), name="attend documents"),
        # A window of 4096 over one shared key head, wide heads, 16 query heads to it, uneven pages.
        dict(_case("attend", 24, 9001, True, 1, 256, 24, True, heads=16, reach=4096, weights=False), name="attend window mqa"),
        # Decode of a cache that will be evicted from: attention that also keeps its weights.
        dict(_case("attend", 16, 4001, True, 8, 128, 32, False, heads=32, reach=0, weights=True), name="attend weights"),
        # One user's cache of a global layer brought down to a quarter.
        dict(_case("evict", 1, 16640, False, 4, 64, 64, False, keep=4096, sinks=4, recent=256), name="evict one"),
        # A batch of long prompts after prefill, brought down to a common budget.
        dict(_case("evict", 16, 32768, True, 8, 128, 16, True, keep=4096, sinks=4, recent=1024), name="evict batch"),
        # A budget overshot by a few decode steps, many short sequences.
        dict(_case("evict", 32, 600, False, 4, 64, 16, False, keep=512, sinks=1, recent=64), name="evict small"),
        # A decode step's store: one token for each of 64 sequences.
        dict(_case("store", 64, 4352, True, 4, 64, 16, False, m=1), name="store step"),
        # Prompts moved into pages after prefill, rounded to bf16.
        dict(_case("store", 8, 8191, False, 8, 128, 16, True, m=8191), name="store prompts"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "evict", "evict", "store"])
    key_heads, dh, bf16 = rng.choice([1, 2, 3, 4, 8]), rng.choice([32, 40, 64, 64, 80, 96, 128, 128, 192, 256]), rng.random() < 0.5
    n, page, ragged = _log(rng, 1, 64), rng.choice([8, 16, 16, 24, 32, 64, 128]), rng.random() < 0.6
    row = key_heads * dh * (2 if bf16 else 4) * 2
    # At most 500 MB of cache in a drawn case, a quarter of the largest listed one.
    longest = min(_log(rng, 1, 60000), max(1, int(5e8 / (row * n))))
    if op == "attend":
        group = rng.choice([1, 2, 3, 4, 5, 8, 16])
        reach = _log(rng, 1, 8192) if rng.random() < 0.25 else 0
        return _case(op, n, longest, ragged, key_heads, dh, page, bf16, heads=key_heads * group, reach=reach,
                     weights=rng.random() < 0.4)
    if op == "evict":
        keep = max(1, int(longest * rng.uniform(0.1, 1.1)))
        sinks = min(keep, rng.choice([0, 1, 4]))
        return _case(op, n, longest, ragged, key_heads, dh, page, bf16, keep=keep, sinks=sinks,
                     recent=int((keep - sinks) * rng.uniform(0.0, 0.6)))
    return _case(op, n, longest, ragged, key_heads, dh, page, bf16, m=1 if rng.random() < 0.5 else longest)


def _lengths(case):
    """Cached tokens of each sequence: all `longest`, or spread below it with every ninth idle."""
    n, longest = case["n"], case["longest"]
    if not case["ragged"]:
        return [longest] * n
    spread = [1 + int((longest - 1) * ((0.6180339887 * i + 0.37) % 1.0) ** 2) for i in range(n)]
    out = [0 if i % 9 == 8 else v for i, v in enumerate(spread)]
    out[0] = longest
    return out


def _per_seq(case):
    return -(-case["longest"] // case["page"])


def work(case):
    kh, dh, size = case["key_heads"], case["dh"], 2 if case["bf16"] else 4
    lens = _lengths(case)
    if case["op"] == "attend":
        seen = sum(min(v, case["reach"]) if case["reach"] else v for v in lens)
        return {"bytes": seen * kh * (2 * dh * size + (8 if case["weights"] else 0)) + 2 * case["n"] * case["heads"] * dh * 4,
                "flops": 4 * seen * case["heads"] * dh}
    if case["op"] == "evict":
        kept = sum(min(v, case["keep"]) for v in lens)
        return {"bytes": kh * (4 * sum(lens) + kept * (2 * 2 * dh * size + 4) + 4 * case["n"] * case["keep"]), "flops": 0}
    new = sum(min(v, case["m"]) for v in lens)
    return {"bytes": 2 * new * kh * dh * (4 + size), "flops": 0}


_library = None


def _slm():
    """The library's Python mirror and one context's operators (the package folder has a dot in its name).
    torch works on the context's stream from then on, so what either queues is in order."""
    global _library
    if _library is None:
        import importlib.util
        import sys
        from pathlib import Path
        at = Path.cwd() / "slm.use_b200"
        spec = importlib.util.spec_from_file_location("slm_b200", at / "__init__.py", submodule_search_locations=[str(at)])
        slm = importlib.util.module_from_spec(spec)
        sys.modules["slm_b200"] = slm
        spec.loader.exec_module(slm)
        ctx = slm.Context(0)
        torch.cuda.synchronize()
        torch.cuda.set_stream(torch.cuda.ExternalStream(ctx.stream))
        _library = slm, ctx, slm.Ops(ctx)
    return _library


class _Memory:
    """A device buffer as torch sees it."""

    def __init__(self, buf):
        self.buf = buf
        self.__cuda_array_interface__ = {"shape": (len(buf),), "typestr": "<f4", "data": (buf.ptr, False), "version": 2}


def _seen(buf, like):
    """The buffer's memory as a tensor of `like`'s shape and type."""
    flat = torch.as_tensor(_Memory(buf), device="cuda").view(like.dtype)
    return flat[: like.numel()].view(like.shape)


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n, kh, dh, page = case["n"], case["key_heads"], case["dh"], case["page"]
    per, dtype = _per_seq(case), torch.bfloat16 if case["bf16"] else torch.float32
    kept_per = -(-case["keep"] // page) if case["op"] == "evict" else 0
    pages = n * (per + kept_per)
    x = {"lens": torch.tensor(_lengths(case), device="cuda")}
    # Pages in the order a running server's free list gives them.
    order = torch.randperm(pages, generator=g, device="cuda")
    x["table"], x["to"] = order[: n * per].view(n, per), order[n * per:].view(n, kept_per)

    def normal(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=g, device="cuda", dtype=dtype)

    # Keys share a direction, as a trained model's do; values have zero mean.
    x["k"] = normal(pages, kh, page, dh, dtype=dtype).add_(normal(1, kh, 1, dh, dtype=dtype), alpha=0.5)
    x["v"] = normal(pages, kh, page, dh, dtype=dtype)
    if case["op"] == "attend":
        x["q"] = normal(n, case["heads"], dh)
    if case["op"] == "evict" or case.get("weights"):
        # Heavy-tailed; the youngest or least regarded tokens have drawn exactly nothing.
        w = torch.empty(pages, kh, page, device="cuda").exponential_(generator=g) * torch.exp(normal(pages, kh, page))
        x["weights"] = torch.where(torch.rand(pages, kh, page, generator=g, device="cuda") < 0.1, 0.0, w)
    if case["op"] == "store":
        x["new_k"], x["new_v"] = normal(n, case["m"], kh * dh), normal(n, case["m"], kh * dh)
    return x


def prepare(case, seed):
    if own:
        slm, ctx, ops = _slm()
    state = dict(case=case, **_inputs(case, seed))
    if own:
        # What a user of the library holds: device buffers with the same contents, and the page tables.
        n, page, per = case["n"], case["page"], state["table"].shape[1]
        pages = state["k"].shape[0]
        for name in ("k", "v", "q", "weights", "new_k", "new_v"):
            if name in state:
                data = state[name]
                buf = ops.zeros(-(-data.numel() * data.element_size() // 4))
                state[name] = _seen(buf, data).copy_(data)
                state[name + "_buf"] = buf
        state["ids"] = slm.Table(ctx, n, per, page, pages)
        for i, row in enumerate(state["table"].tolist()):
            state["ids"].assign(i, row)
        state["ids"].set_lens(_lengths(case))
        if case["op"] == "attend":
            state["scores_buf"] = ops.zeros(1)
            state["y_buf"] = ops.zeros(state["q"].numel())
            state["y"] = _seen(state["y_buf"], state["q"])
        if case["op"] == "evict":
            state["to_ids"] = slm.Table(ctx, n, state["to"].shape[1], page, pages)
            for i, row in enumerate(state["to"].tolist()):
                state["to_ids"].assign(i, row)
            state["kept_buf"] = ops.zeros(n * case["key_heads"] * case["keep"])
            state["kept"] = _seen(state["kept_buf"], torch.empty(n, case["key_heads"], case["keep"], dtype=torch.int32, device="meta"))
        ctx.sync()
        torch.cuda.synchronize()
    return state


def _own_run(s):
    _, _, ops = _slm()
    c = s["case"]
    if c["op"] == "attend":
        ops.paged_attend(s["y_buf"], s["scores_buf"], s["q_buf"], s["k_buf"], s["v_buf"], s["ids"], heads=c["heads"],
                         key_heads=c["key_heads"], dh=c["dh"], scale=c["dh"] ** -0.5, reach=c["reach"] or None,
                         bf16=c["bf16"], weights=s.get("weights_buf"))
        return {"y": s["y"], "weights": s["weights"]} if c["weights"] else {"y": s["y"]}
    if c["op"] == "evict":
        ops.paged_evict(s["kept_buf"], s["k_buf"], s["v_buf"], s["weights_buf"], s["ids"], s["to_ids"], keep=c["keep"],
                        sinks=c["sinks"], recent=c["recent"], key_heads=c["key_heads"], dh=c["dh"], bf16=c["bf16"])
        return {"kept": s["kept"], "k": s["k"], "v": s["v"], "weights": s["weights"]}
    ops.paged_store(s["k_buf"], s["v_buf"], s["ids"], s["new_k_buf"], s["new_v_buf"], m=c["m"], key_heads=c["key_heads"],
                    dh=c["dh"], bf16=c["bf16"])
    return {"k": s["k"], "v": s["v"]}


def _rows(pages, table):
    """Pages of every sequence side by side: [n][key_heads][slots](...)."""
    x = pages[table].transpose(1, 2)
    return x.reshape(x.shape[0], x.shape[1], -1, *x.shape[4:])


def _attend(s):
    c, lens = s["case"], s["lens"]
    n, kh, group = c["n"], c["key_heads"], c["heads"] // c["key_heads"]
    k, v = _rows(s["k"], s["table"]).float(), _rows(s["v"], s["table"]).float()
    slot = torch.arange(k.shape[2], device="cuda")
    seen = (slot < lens[:, None]) & (slot >= (lens[:, None] - c["reach"] if c["reach"] else 0))
    score = (s["q"].view(n, kh, group, -1) @ k.transpose(2, 3)) * c["dh"] ** -0.5
    score = score.masked_fill(~seen[:, None, None], -torch.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(torch.isinf(top), 0.0, top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    y = (p @ torch.where(seen[:, None, :, None], v, 0.0)).view(n, c["heads"], -1)
    if not c["weights"]:
        return {"y": y}
    page, row = s["table"][:, slot // c["page"]], slot % c["page"]
    drawn = p.sum(2).transpose(1, 2)  # [n][slots][key_heads]
    s["weights"][page, :, row.expand_as(page)] += drawn
    return {"y": y, "weights": s["weights"]}


def _evict(s):
    c, lens = s["case"], s["lens"]
    w = _rows(s["weights"][..., None], s["table"])[..., 0]
    slot = torch.arange(w.shape[2], device="cuda")
    held = (slot < c["sinks"]) | (slot >= lens[:, None] - c["recent"])
    rank_by = torch.where((slot < lens[:, None])[:, None], torch.where(held[:, None], torch.inf, w), -torch.inf)
    order = torch.sort(rank_by, dim=-1, descending=True, stable=True).indices[..., : c["keep"]]
    count = lens.clamp(max=c["keep"])
    place = torch.arange(order.shape[-1], device="cuda")
    kept = torch.sort(torch.where(place < count[:, None, None], order, 1 << 30), dim=-1).values
    used = (place < count[:, None])[:, None].expand_as(kept)
    seq, head, to = used.nonzero(as_tuple=True)
    old = kept[used]
    page, row = s["table"][seq, old // c["page"]], old % c["page"]
    new_page, new_row = s["to"][seq, to // c["page"]], to % c["page"]
    for name in ("k", "v", "weights"):
        s[name][new_page, head, new_row] = s[name][page, head, row]
    ids = torch.full((c["n"], c["key_heads"], c["keep"]), -1, dtype=torch.int32, device="cuda")
    ids[..., : kept.shape[-1]] = torch.where(used, kept, -1).int()
    return {"kept": ids, "k": s["k"], "v": s["v"], "weights": s["weights"]}


def _store(s):
    c, lens = s["case"], s["lens"]
    slot = lens[:, None] - c["m"] + torch.arange(c["m"], device="cuda")
    seq, j = (slot >= 0).nonzero(as_tuple=True)
    slot = slot[seq, j]
    page, row = s["table"][seq, slot // c["page"]], slot % c["page"]
    for name in ("k", "v"):
        new = s["new_" + name][seq, j].view(-1, c["key_heads"], c["dh"])
        s[name][page, :, row] = new.to(s[name].dtype)
    return {"k": s["k"], "v": s["v"]}


def run(state):
    if own:
        return _own_run(state)
    return {"attend": _attend, "evict": _evict, "store": _store}[state["case"]["op"]](state)


def exact(case, seed):
    """Sequence by sequence in 64 bits, token by token where tokens are moved."""
    x, c, lens = _inputs(case, seed), case, _lengths(case)
    page, kh = c["page"], c["key_heads"]

    def cached(name, i, count):
        pages = x["table"][i, : -(-count // page)]
        rows = x[name][pages].double()  # [pages][key_heads][page](dh)
        return torch.cat(list(rows), dim=1)[:, :count]

    if c["op"] == "attend":
        y = torch.zeros(c["n"], c["heads"], c["dh"], dtype=torch.float64, device="cuda")
        weights = x["weights"].double() if c["weights"] else None
        for i, count in enumerate(lens):
            if count == 0:
                continue
            first = max(0, count - c["reach"]) if c["reach"] else 0
            k, v = (cached(name, i, count)[:, first:] for name in ("k", "v"))
            q = x["q"][i].double().view(kh, -1, c["dh"])
            p = torch.softmax(torch.einsum("hgd,hsd->hgs", q, k) / math.sqrt(c["dh"]), dim=-1)
            y[i] = torch.einsum("hgs,hsd->hgd", p, v).reshape(c["heads"], c["dh"])
            if weights is not None:
                at = torch.arange(first, count, device="cuda")
                weights[x["table"][i, at // page], :, at % page] += p.sum(1).T
        return {"y": y, "weights": weights} if c["weights"] else {"y": y}
    out = {name: x[name].double() for name in ("k", "v") + (("weights",) if c["op"] == "evict" else ())}
    if c["op"] == "store":
        for i, count in enumerate(lens):
            new = min(count, c["m"])
            at = torch.arange(count - new, count, device="cuda")
            for name in ("k", "v"):
                rows = x["new_" + name][i, c["m"] - new:].view(new, kh, c["dh"])
                out[name][x["table"][i, at // page], :, at % page] = rows.to(x[name].dtype).double()
        return out
    for i, count in enumerate(lens):
        if count == 0:
            continue
        w, keep = cached("weights", i, count), min(count, c["keep"])
        for h in range(kh):
            middle = [] if keep == count else sorted(enumerate(w[h].tolist()), key=lambda e: (-e[1], e[0]))
            held = set(range(count)) if keep == count else set(range(c["sinks"])) | set(range(count - c["recent"], count))
            for s, _ in middle:
                if len(held) == keep:
                    break
                held.add(s)
            old = torch.tensor(sorted(held), device="cuda")
            new = torch.arange(keep, device="cuda")
            for name in ("k", "v", "weights"):
                out[name][x["to"][i, new // page], h, new % page] = \
                    x[name][x["table"][i, old // page], h, old % page].double()
    return {"kept": None, **out}
