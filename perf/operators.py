"""Performance cases of the routing operators: tokens grouped by the expert or adapter that serves
them, their rows moved there and back, and low-rank adapters applied per request.

What a program does with them:

* a mixture-of-experts layer plans its batch once (``route_plan``), sends the rows of its tokens to
  their experts (``route_dispatch``) and sums the experts' answers with the router's weights
  (``route_combine``); in training the gradients of both go the same ways back;
* a server of many fine-tuned variants of one model plans a batch by adapter id and adds every
  request's own low-rank product to each shared projection (``adapter_add``).

A case: ``op``; ``tokens`` x ``choices`` ids out of ``groups``, a share ``dropped`` of which name no
group; ``dim`` (and ``out_dim``, ``rank`` of adapters) and ``elem`` of the rows; ``weighted``;
``key_bits`` of the ids of a plan.
"""
import torch

own = False

_ELEM = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_MOST_ROW_BYTES = 32768 * 4 * 4096 * 2  # rows of the largest listed case
_MOST_CHOICES = 65536 * 8


# ---- cases ---------------------------------------------------------------------------------
def _plan(tokens, choices, groups, dropped, key_bits, **name):
    return {"op": "plan", "tokens": tokens, "choices": choices, "groups": groups, "dropped": dropped, "key_bits": key_bits, **name}


def _rows(op, tokens, choices, groups, dropped, dim, elem, weighted, **name):
    return {"op": op, "tokens": tokens, "choices": choices, "groups": groups, "dropped": dropped, "dim": dim, "elem": elem,
            "weighted": weighted, **name}


def _adapter(tokens, groups, dropped, rank, dim, out_dim, elem, **name):
    return {"op": "adapter", "tokens": tokens, "choices": 1, "groups": groups, "dropped": dropped, "rank": rank, "dim": dim,
            "out_dim": out_dim, "elem": elem, **name}


def listed():
    return [
        # the router's answer for one decoding step of 32 requests
        _plan(32, 8, 128, 0.0, 64, name="plan_step"),
        # a training micro-batch whose experts refuse some tokens for want of capacity
        _plan(65536, 8, 256, 0.02, 32, name="plan_train"),
        # rows of a decoding step to their experts: latency
        _rows("dispatch", 32, 8, 128, 0.0, 4096, "bf16", False, name="dispatch_step"),
        # rows of a training micro-batch to their experts
        _rows("dispatch", 16384, 8, 128, 0.0, 2048, "bf16", False, name="dispatch_train"),
        # backward pass of a dispatch that applied the weights itself, full precision
        _rows("dispatch_grad", 8192, 4, 32, 0.0, 1024, "f32", True, name="dispatch_grad_train"),
        # the experts' answers of a decoding step, summed
        _rows("combine", 32, 8, 128, 0.0, 4096, "bf16", True, name="combine_step"),
        # the same over long prompts, few choices and wide rows
        _rows("combine", 32768, 4, 64, 0.0, 4096, "bf16", True, name="combine_prompts"),
        # odd sizes: rows at odd addresses, a fifth of the choices dropped
        _rows("combine", 4097, 3, 17, 0.2, 1001, "f16", True, name="combine_odd"),
        # backward pass of the sum over a training micro-batch
        _rows("combine_grad", 16384, 6, 64, 0.01, 2048, "bf16", True, name="combine_grad_train"),
        # one decoding step of 48 requests that share 64 adapters between them
        _adapter(48, 64, 0.0, 16, 4096, 4096, "bf16", name="adapter_step"),
        # a batch of prompts over two dozen adapters
        _adapter(16384, 24, 0.0, 64, 4096, 4096, "bf16", name="adapter_prompts"),
        # short prompts and single tokens mixed, a quarter of the tokens without an adapter
        _adapter(1111, 200, 0.25, 8, 2048, 6144, "f16", name="adapter_mixed"),
    ]


def _log_int(rng, low, high):
    return min(high, max(low, round(low * (high / low) ** rng.random())))


def draw(rng):
    op = rng.choice(["plan", "dispatch", "dispatch_grad", "combine", "combine_grad", "adapter", "adapter"])
    dropped = rng.choice([0.0, 0.0, round(0.3 * rng.random(), 3)])
    if op == "adapter":
        return _adapter(_log_int(rng, 1, 16384), _log_int(rng, 1, 256), dropped, rng.choice([8, 16, 24, 32, 64]),
                        8 * _log_int(rng, 16, 512), 8 * _log_int(rng, 16, 512), rng.choice(["bf16", "f16"]))
    choices = rng.randint(1, 8)
    groups = _log_int(rng, choices, 512)
    if op == "plan":
        return _plan(_log_int(rng, 1, _MOST_CHOICES // choices), choices, groups, dropped, rng.choice([32, 64]))
    elem = rng.choice(["bf16", "bf16", "f16", "f32"])
    dim = _log_int(rng, 64, 8192)
    if rng.random() < 0.7:
        dim = -(-dim // 64) * 64
    most = min(32768, _MOST_ROW_BYTES // (4 * choices * dim * _ELEM[elem].itemsize))
    return _rows(op, _log_int(rng, 1, most), choices, groups, dropped, dim, elem, rng.random() < 0.8)


def work(case):
    c = case
    n = c["tokens"] * c["choices"]
    if c["op"] == "plan":
        return {"bytes": n * (c["key_bits"] // 8 + 8) + 4 * (c["groups"] + 1), "flops": 0}
    e = _ELEM[c["elem"]].itemsize
    if c["op"] == "adapter":
        served = c["tokens"] * (1 - c["dropped"])
        used = c["groups"] * (1 - (1 - 1 / c["groups"]) ** served)  # adapters that at least one token names, about
        return {"bytes": int((c["tokens"] * (c["dim"] + 2 * c["out_dim"]) + used * c["rank"] * (c["dim"] + c["out_dim"])) * e),
                "flops": int(2 * served * c["rank"] * (c["dim"] + c["out_dim"]))}
    taken = n * (1 - c["dropped"])
    one, many = c["tokens"] * c["dim"] * e, taken * c["dim"] * e
    index = 4 * n + (4 * n if c["weighted"] else 0)
    if c["op"] == "dispatch":  # every row of the output is written, those that nothing takes with zeros
        return {"bytes": int(one + n * c["dim"] * e + index), "flops": int(taken * c["dim"]) if c["weighted"] else 0}
    if c["op"] == "combine":
        return {"bytes": int(one + many + index), "flops": int(2 * taken * c["dim"])}
    dots = 4 * n if c["weighted"] else 0
    if c["op"] == "dispatch_grad":
        return {"bytes": int(one * (2 if c["weighted"] else 1) + many + index + dots), "flops": int(4 * taken * c["dim"])}
    return {"bytes": int(one + (many if c["weighted"] else 0) + n * c["dim"] * e + index + dots), "flops": int(3 * taken * c["dim"])}


# ---- inputs --------------------------------------------------------------------------------
def _inputs(case, seed):
    """The tensors of a case, from the seed alone."""
    c, dev = case, "cuda"
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    T, k, G = c["tokens"], c["choices"], c["groups"]

    def normal(*size):
        return torch.randn(*size, generator=g, device=dev)

    s = {}
    if c["op"] == "adapter":  # a few adapters take most requests; a request's tokens stand next to one another
        at = torch.rand(T, generator=g, device=dev)
        start = (torch.rand(T, generator=g, device=dev) < 0.05) if T > 256 else torch.ones(T, dtype=torch.bool, device=dev)
        start[0] = True
        request = start.cumsum(0) - 1
        ids = ((G * at * at).long().clamp(max=G - 1))[request].reshape(T, 1)
    else:  # the router's choices: distinct, some groups favoured
        logits = normal(T, G) + normal(G)
        ids = logits.topk(k, dim=1).indices
    if c["dropped"]:
        gone = torch.rand(T, k, generator=g, device=dev) < c["dropped"]
        ids = torch.where(gone, torch.full_like(ids, -1), ids)
    s["ids"] = ids.to(torch.int32 if c.get("key_bits") == 32 else torch.int64).contiguous()
    if c["op"] == "plan":
        return s
    ty = _ELEM[c["elem"]]
    if c["op"] == "adapter":
        r, H, N = c["rank"], c["dim"], c["out_dim"]
        s["base"] = normal(T, N).to(ty)
        s["x"] = normal(T, H).to(ty)
        s["down"] = (normal(G, r, H) / H ** 0.5).to(ty)
        s["up"] = (normal(G, N, r) / r ** 0.5).to(ty)
        s["scale"] = 0.5 + torch.rand(G, generator=g, device=dev)
        return s
    s["weights"] = None
    if c["weighted"]:
        s["weights"] = torch.softmax(normal(T, k), dim=1).contiguous()
    s["tokens"] = normal(T, c["dim"]).to(ty)
    if c["op"] != "dispatch":
        s["rows"] = normal(T * k, c["dim"]).to(ty)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["op"], s["groups"] = case["op"], case["groups"]
    if case["op"] == "plan":
        return s
    # the batch is planned once, its layers use the plan
    if own:
        from ugache_b200 import runtime as rt
        s["plan"] = rt.route_plan(s["ids"], s["groups"])
    else:
        s["plan"] = _plain_plan(s["ids"], s["groups"])
        if case["op"] == "adapter":  # tokens of each adapter in a padded list, so that one batched product serves all
            offsets, order, _ = s["plan"]
            count = (offsets[1:] - offsets[:-1]).long()
            most = max(1, int(count.max()))
            at = torch.arange(most, device=order.device)
            place = offsets[:-1, None].long() + at
            s["held"] = at < count[:, None]
            s["lists"] = order.long()[place.clamp(max=order.numel() - 1)]
    return s


# ---- plain forms ---------------------------------------------------------------------------
def _plain_plan(ids, groups):
    flat = ids.reshape(-1).long()
    n = flat.numel()
    key = torch.where((flat >= 0) & (flat < groups), flat, torch.full_like(flat, groups))
    order = torch.sort(key, stable=True).indices
    ends = torch.bincount(key, minlength=groups + 1).cumsum(0)
    offsets = torch.cat([ends.new_zeros(1), ends[:groups]])
    position = torch.empty_like(order)
    position[order] = torch.arange(n, device=order.device)
    position = torch.where(key < groups, position, torch.full_like(position, -1))
    return offsets.to(torch.int32), order.to(torch.int32), position.to(torch.int32).reshape(ids.shape)


def _spread(src, plan, weights, k):
    """Row t of `src` to the rows that t's choices take, times the weight; zero elsewhere."""
    offsets, order, _ = plan
    at = order.long()
    rows = src[at // k].float()
    if weights is not None:
        rows = rows * weights.reshape(-1)[at][:, None]
    taken = torch.arange(at.numel(), device=at.device) < offsets[-1]
    return torch.where(taken[:, None], rows, rows.new_zeros(())).to(src.dtype)


def _picked(rows, plan):
    """The rows that the choices of every token took, [T, k, dim] in 32 bits; zero for a dropped choice."""
    _, _, position = plan
    got = rows[position.long().clamp(min=0)].float()
    return torch.where((position >= 0)[:, :, None], got, got.new_zeros(()))


def _plain_adapter(s):
    _, _, position = s["plan"]
    x, base = s["x"], s["base"]
    lists, held = s["lists"], s["held"]
    inner = torch.bmm(x[lists].float(), s["down"].float().transpose(1, 2)) * s["scale"][:, None, None]
    delta = torch.bmm(inner, s["up"].float().transpose(1, 2))
    out = base.float()
    out.index_add_(0, lists[held], delta[held])
    return out.to(base.dtype)


def run(state):
    s = state
    op = s["op"]
    if own:
        from ugache_b200 import runtime as rt
        if op == "plan":
            p = rt.route_plan(s["ids"], s["groups"])
            return p.offsets, p.order, p.position
        if op == "dispatch":
            return rt.route_dispatch(s["tokens"], s["plan"], weights=s["weights"])
        if op == "dispatch_grad":
            return rt.route_dispatch_grad(s["rows"], s["plan"], weights=s["weights"],
                                          x=s["tokens"] if s["weights"] is not None else None)
        if op == "combine":
            return rt.route_combine(s["rows"], s["plan"], weights=s["weights"])
        if op == "combine_grad":
            return rt.route_combine_grad(s["tokens"], s["plan"], weights=s["weights"],
                                         rows=s["rows"] if s["weights"] is not None else None)
        return rt.adapter_add(s["base"], s["x"], s["down"], s["up"], s["plan"], scale=s["scale"])
    if op == "plan":
        return _plain_plan(s["ids"], s["groups"])
    if op == "adapter":
        return _plain_adapter(s)
    k, w = s["ids"].shape[1], s["weights"]
    if op == "dispatch":
        return _spread(s["tokens"], s["plan"], w, k)
    if op == "combine_grad":
        dots = None
        if w is not None:
            dots = (_picked(s["rows"], s["plan"]) * s["tokens"].float()[:, None, :]).sum(2)
        return _spread(s["tokens"], s["plan"], w, k), dots
    picked = _picked(s["rows"], s["plan"])
    total = (picked if w is None else picked * w[:, :, None]).sum(1).to(s["rows"].dtype)
    if op == "combine":
        return total
    return total, None if w is None else (picked * s["tokens"].float()[:, None, :]).sum(2)


# ---- definition in 64 bits -----------------------------------------------------------------
def exact(case, seed):
    if case["op"] == "plan":
        return None  # whole numbers
    s = _inputs(case, seed)
    ids, G, op = s["ids"].long(), case["groups"], case["op"]
    T, k = ids.shape
    if op == "adapter":
        out = s["base"].double()
        for a in range(G):
            t = torch.nonzero(ids[:, 0] == a).reshape(-1)
            if t.numel():
                inner = s["x"][t].double() @ s["down"][a].double().t()
                out[t] += float(s["scale"][a].double()) * (inner @ s["up"][a].double().t())
        return out
    # where each choice stands: behind all choices of smaller groups and the earlier ones of its own
    flat, place, at = ids.reshape(-1), torch.full((T * k,), -1, dtype=torch.long, device=ids.device), 0
    for a in range(G):
        i = torch.nonzero(flat == a).reshape(-1)
        place[i] = at + torch.arange(i.numel(), device=ids.device)
        at += i.numel()
    place = place.reshape(T, k)
    w = torch.ones(T, k, dtype=torch.float64, device=ids.device) if s["weights"] is None else s["weights"].double()
    src = s["tokens"].double()
    dots, total = torch.zeros(T, k, dtype=torch.float64, device=ids.device), torch.zeros_like(src)
    spread = torch.zeros(T * k, src.shape[1], dtype=torch.float64, device=ids.device) if op in ("dispatch", "combine_grad") else None
    for j in range(k):
        t = torch.nonzero(place[:, j] >= 0).reshape(-1)
        p = place[t, j]
        if spread is not None:
            spread[p] = src[t] * w[t, j, None]
        if op != "dispatch":
            row = s["rows"][p].double()
            total[t] += row * w[t, j, None]
            dots[t, j] = (row * src[t]).sum(1)
    if s["weights"] is None:
        dots = None
    return {"dispatch": spread, "combine": total, "dispatch_grad": (total, dots), "combine_grad": (spread, dots)}[op]
