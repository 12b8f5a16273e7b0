"""The operators around a LoRA model's projections that keep their weights in bf16 or float32, over the sizes they are used at.

Three of them, which a training step of an unquantized expert or embedding layer calls one after the other:

* ``grouped``  products grouped by expert with ragged sizes, ``out[rows of g] = x[rows of g] @ weight[g]``
  (rows sorted by expert; rows behind the last group give zeros), and with ``backward`` their two gradients;
* ``embed``    rows of an embedding table, scaled, and with ``backward`` the table's dense gradient.  A table of
  ``adapters`` > 0 is the stack of a LoRA embedding's A factors: a row belongs to (adapter, token) and each adapter has
  its own factor;
* ``clip``     the global norm over the gradients of many adapter tensors, one norm per adapter (the leading axis of
  every tensor), and the gradients scaled down to that adapter's limit.

The plain forms are elementary torch operations in float32.
"""

from __future__ import annotations

import math

import torch

own = False

DEVICE = "cuda:0"
_TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def _package():
    import __graft_entry__

    return __graft_entry__.load_package()


def _dims(text):
    """(in, out) features of one layer's projections."""
    return [tuple(int(v) for v in d.split("x")) for d in text.split()]


def listed():
    experts = dict(op="grouped", groups=128, top_k=8, spare=0, backward=False, dw="bf16")
    table = dict(op="embed", vocab=151936, pad=0.0, type="bf16", adapters=0, backward=False)
    return [
        # eight users decode together: eight of 128 experts each, the gate/up weights of the ones that are hit
        dict(experts, name="grouped-decode-t8", rows=64, k=2048, n=1536),
        # the same layer over a prefill of 2048 tokens
        dict(experts, name="grouped-prefill-t2048", rows=16384, k=2048, n=1536),
        # a micro-batch of 4096 tokens trains the down projection: gradients of the rows and of the experts
        dict(experts, name="grouped-train-t4096", rows=32768, k=768, n=2048, backward=True),
        # few large experts over a long batch: the product itself
        dict(experts, name="grouped-large-e8", rows=32768, groups=8, top_k=2, k=4096, n=12288),
        # rows of a short ragged batch in thirteen groups, some empty, with spare rows behind them; float32 weight gradients
        dict(experts, name="grouped-ragged-m1003", rows=1003, groups=13, top_k=0, k=712, n=1096, spare=19, backward=True, dw="f32"),
        # sixteen users decode together: their tokens' rows of the embedding
        dict(table, name="embed-decode-m16", tokens=16, width=4096),
        # LoRA embedding: the A rows of a batch of eight adapters
        dict(table, name="embed-adapters-m8192", tokens=8192, width=32, adapters=8),
        # training the embedding itself on padded sequences
        dict(table, name="embed-train-m16384", tokens=16384, width=2560, pad=0.08, backward=True),
        # training eight adapters' embeddings
        dict(table, name="embed-train-adapters-m32768", tokens=32768, width=32, adapters=8, pad=0.08, backward=True),
        # gradients of the four attention projections of one layer, four adapters
        dict(op="clip", name="clip-layer-a4", dims="4096x4096 4096x1024 4096x1024 4096x4096", layers=1, adapters=4, rank=16, type="bf16"),
        # float32 gradients of expert layers, whose adapters hold every expert's factors
        dict(op="clip", name="clip-experts-f32-a4", dims="262144x196608 98304x262144", layers=2, adapters=4, rank=16, type="f32"),
        # every gradient of a 36-layer model with eight adapters
        dict(op="clip", name="clip-model-a8", dims="4096x6144 4096x4096 4096x24576 12288x4096", layers=36, adapters=8, rank=32, type="bf16"),
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["grouped", "grouped", "embed", "clip"])
    if op == "grouped":
        while True:
            groups, rows = log(4, 128), log(1, 32768)
            top_k = rng.choice([0, 1, 2, 4, 8])
            rows -= rows % max(1, top_k)
            k, n = 8 * log(8, 512), 8 * log(8, 1536)
            if top_k <= groups and rows >= max(1, top_k) and rows * k * n <= 1.6e12 and groups * k * n <= 1.6e9:
                break
        return dict(op=op, rows=rows, groups=groups, top_k=top_k, k=k, n=n, spare=rng.choice([0, 0, rows // 50]) if top_k == 0 else 0,
                    backward=rng.random() < 0.5, dw=rng.choice(["bf16", "f32"]))
    if op == "embed":
        adapters = rng.choice([0, 0, rng.randint(1, 16)])
        width = rng.choice([8, 16, 32, 64, rng.randint(1, 64)]) if adapters else rng.choice([8 * log(16, 512), rng.randint(65, 4096)])
        vocab = log(1000, 200000)
        while (adapters or 1) * vocab * width > 4e8:
            vocab //= 2
        return dict(op=op, vocab=vocab, tokens=log(1, 32768), width=width, adapters=adapters, pad=rng.choice([0.0, 0.1, 0.5]),
                    type=rng.choice(["bf16", "bf16", "f32"]), backward=rng.random() < 0.5)
    while True:
        dims = " ".join("%dx%d" % (log(64, 16384), log(64, 32768)) for _ in range(rng.randint(1, 6)))
        layers, adapters, rank = log(1, 48), rng.choice([1, 1, rng.randint(2, 16)]), rng.choice([1, 4, 8, 16, 32, 64, rng.randint(1, 64)])
        if 1000 <= layers * adapters * rank * sum(k + n for k, n in _dims(dims)) <= 6e8:
            break
    return dict(op=op, dims=dims, layers=layers, adapters=adapters, rank=rank, type=rng.choice(["bf16", "bf16", "f32"]))


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)

    def normal(*shape, std=1.0, dtype=torch.bfloat16):
        return (torch.randn(*shape, generator=g, device=DEVICE) * std).to(dtype)

    def uniform(*shape):
        return torch.rand(*shape, generator=g, device=DEVICE)

    state = dict(case)
    if case["op"] == "grouped":
        rows, groups, k, n = case["rows"], case["groups"], case["k"], case["n"]
        if case["top_k"]:  # a router's choice: some experts are liked more than others
            scores = normal(rows // case["top_k"], groups, dtype=torch.float32) + normal(groups, std=0.5, dtype=torch.float32)
            sizes = torch.bincount(scores.topk(case["top_k"], dim=1).indices.reshape(-1), minlength=groups)
        else:  # uneven parts, a quarter of them empty, and the spare rows behind the last one
            share = uniform(groups) ** 2 * (uniform(groups) > 0.25)
            share[0] += 0.01
            ends = (torch.cumsum(share, 0) / share.sum() * (rows - case["spare"])).round().long().clamp(max=rows - case["spare"])
            sizes = torch.diff(ends, prepend=ends.new_zeros(1))
        state["sizes"] = sizes.to(torch.int32)
        state["longest"] = int(sizes.max())
        state["x"] = normal(rows, k)
        state["weight"] = torch.empty(groups, k, n, dtype=torch.bfloat16, device=DEVICE)
        state["weight"].normal_(std=k ** -0.5, generator=g)
        if case["backward"]:
            state["dy"] = normal(rows, n, std=0.1)
    elif case["op"] == "embed":
        tokens, vocab, adapters, width = case["tokens"], case["vocab"], case["adapters"], case["width"]
        # words of a text: the r-th most frequent one about 1 / r of the time, anywhere in the table; padding is word 0
        rank = torch.exp(uniform(tokens).double() * math.log(vocab)).long().clamp(max=vocab) - 1
        ids = rank * 48271 % vocab
        state["ids"] = torch.where(uniform(tokens) < case["pad"], 0, ids).to(torch.int32)
        if adapters:
            state["adapter"] = torch.randint(0, adapters, (tokens,), generator=g, device=DEVICE, dtype=torch.int32)
            state["scale"] = uniform(adapters) * 2 + 0.5
        else:
            state["scale"] = math.sqrt(width)
        if case["backward"]:
            state["dy"] = normal(tokens, width, std=0.1, dtype=_TYPES[case["type"]])
        else:
            state["table"] = normal(*([adapters] if adapters else []), vocab, width, std=0.05, dtype=_TYPES[case["type"]])
    else:
        adapters, rank = case["adapters"], case["rank"]
        shapes = [s for _ in range(case["layers"]) for k, n in _dims(case["dims"]) for s in ((adapters, k, rank), (adapters, rank, n))]
        state["grads"] = [normal(*s, std=1e-3, dtype=_TYPES[case["type"]]) for s in shapes]
        # limits on both sides of the norms: every other adapter's gradients are scaled down
        norm = 1e-3 * math.sqrt(sum(math.prod(s[1:]) for s in shapes))
        state["limits"] = norm * torch.where(torch.arange(adapters, device=DEVICE) % 2 == 0, 0.5, 2.0) * (1 + 0.1 * uniform(adapters))
        # the scaled gradients go to one bucket, a view of it for each, where the optimizer reads them
        state["bucket"] = torch.empty(sum(math.prod(s) for s in shapes), dtype=_TYPES[case["type"]], device=DEVICE)
        state["views"] = [b.view(s) for b, s in zip(state["bucket"].split([math.prod(s) for s in shapes]), shapes)]
        if own:  # (as a training loop keeps it: the gradients' buffers stay where they are from step to step)
            state["plan"] = _package().grad_clip.GradClipPlan(state["grads"], state["limits"], per_adapter=True, out=state["views"])
    return state


# -- the plain forms -------------------------------------------------------------------------------------------------


def _place(state):
    """Group of every row and its place among the rows of that group (rows behind the last group: none)."""
    ends = torch.cumsum(state["sizes"], 0)
    row = torch.arange(state["rows"], device=DEVICE)
    group = torch.searchsorted(ends, row, right=True)
    held = group < state["groups"]
    group = group.clamp(max=state["groups"] - 1)
    return group, (row - (ends - state["sizes"])[group]).clamp(0, max(0, state["longest"] - 1)), held


def _padded(state, t, place):
    group, at, held = place
    out = torch.zeros(state["groups"], max(1, state["longest"]), t.shape[1], device=DEVICE)
    # (the rows of no group are added as zeros)
    out.index_put_((group, at), t.float() * held[:, None], accumulate=True)
    return out


def _grouped(state):
    place = _place(state)
    group, at, held = place
    weight = state["weight"].float()
    if not state["backward"]:
        return (torch.bmm(_padded(state, state["x"], place), weight)[group, at] * held[:, None]).bfloat16()
    dy = _padded(state, state["dy"], place)
    dx = (torch.bmm(dy, weight.transpose(1, 2).contiguous())[group, at] * held[:, None]).bfloat16()
    dw = torch.bmm(_padded(state, state["x"], place).transpose(1, 2).contiguous(), dy)
    return dx, dw.to(_TYPES[state["dw"]])


def _embed(state):
    ids = state["ids"].long()
    scale = state["scale"]
    if state["adapters"]:
        ids, scale = ids + state["adapter"].long() * state["vocab"], scale[state["adapter"].long()][:, None]
    if not state["backward"]:
        return (state["table"].view(-1, state["width"])[ids].float() * scale).to(_TYPES[state["type"]])
    count = max(1, state["adapters"]) * state["vocab"]
    grad = torch.zeros(count, state["width"], device=DEVICE).index_add_(0, ids, state["dy"].float() * scale).to(_TYPES[state["type"]])
    return grad.view(state["adapters"], state["vocab"], -1) if state["adapters"] else grad


def _clip(state):
    norms = torch.stack([g.float().flatten(1).square().sum(1) for g in state["grads"]]).sum(0).sqrt()
    factor = torch.where(norms > state["limits"], state["limits"] / norms, 1.0)
    torch.cat([(g.float() * factor[:, None, None]).to(g.dtype).view(-1) for g in state["grads"]], out=state["bucket"])
    return state["bucket"], norms


# -- one pass ---------------------------------------------------------------------------------------------------------


def run(state):
    if not own:
        return {"grouped": _grouped, "embed": _embed, "clip": _clip}[state["op"]](state)
    if state["op"] == "grouped":
        grouped = _package().bf16_grouped_linear
        if not state["backward"]:
            return grouped.grouped_matmul(state["x"], state["weight"], state["sizes"])
        return grouped.grouped_matmul_backward(state["x"], state["dy"], state["weight"], state["sizes"], dw_dtype=_TYPES[state["dw"]])
    if state["op"] == "embed":
        embedding = _package().embedding
        if not state["backward"]:
            return embedding.lookup(state["table"], state["ids"], state["scale"], adapter_indices=state.get("adapter"))
        shape = (state["adapters"], state["vocab"], state["width"]) if state["adapters"] else (state["vocab"], state["width"])
        return embedding.lookup_backward(state["dy"], state["ids"], shape, state["scale"], adapter_indices=state.get("adapter"))
    _, norms = state["plan"].run()
    return state["bucket"], norms


def work(case):
    if case["op"] == "grouped":
        rows, k, n, groups = case["rows"], case["k"], case["n"], case["groups"]
        hit = groups * (1 - (1 - 1 / groups) ** rows)  # groups that a router's choice reaches
        if not case["backward"]:
            return {"bytes": 2 * (rows * k + hit * k * n + rows * n), "flops": 2 * rows * k * n}
        dw = 2 if case["dw"] == "bf16" else 4
        return {"bytes": 2 * (2 * rows * k + rows * n + hit * k * n) + dw * groups * k * n, "flops": 4 * rows * k * n}
    if case["op"] == "embed":
        size = 2 if case["type"] == "bf16" else 4
        moved, index = case["tokens"] * case["width"] * size, case["tokens"] * (8 if case["adapters"] else 4)
        if not case["backward"]:
            return {"bytes": 2 * moved + index, "flops": case["tokens"] * case["width"]}
        return {"bytes": moved + index + max(1, case["adapters"]) * case["vocab"] * case["width"] * size, "flops": 2 * case["tokens"] * case["width"]}
    count = case["layers"] * case["adapters"] * case["rank"] * sum(k + n for k, n in _dims(case["dims"]))
    return {"bytes": 2 * count * (2 if case["type"] == "bf16" else 4), "flops": 3 * count}


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "grouped":
        return _exact_grouped(case, state)
    if case["op"] == "embed":
        return _exact_embed(case, state)
    total = sum(torch.linalg.vector_norm(g.double(), dim=(1, 2)) ** 2 for g in state["grads"])
    norms = total.sqrt()
    limits = state["limits"].double()
    scaled = []
    for g in state["grads"]:
        out = g.double()
        for a in range(case["adapters"]):
            if norms[a] > limits[a]:
                out[a] *= limits[a] / norms[a]
        scaled.append(out.view(-1))
    return torch.cat(scaled), norms


def _exact_grouped(case, state):
    x, first = state["x"].double(), 0
    out = torch.zeros(case["rows"], case["k" if case["backward"] else "n"], dtype=torch.float64, device=DEVICE)
    dw = torch.zeros_like(state["weight"], dtype=torch.float64) if case["backward"] else None
    for g, size in enumerate(state["sizes"].tolist()):
        rows = slice(first, first + size)
        first += size
        if case["backward"]:
            out[rows] = state["dy"][rows].double() @ state["weight"][g].double().T
            dw[g] = x[rows].T @ state["dy"][rows].double()
        else:
            out[rows] = x[rows] @ state["weight"][g].double()
    return (out, dw) if case["backward"] else out


def _exact_embed(case, state):
    adapter = state["adapter"].long() if case["adapters"] else torch.zeros(case["tokens"], dtype=torch.long, device=DEVICE)
    scale = state["scale"].double() if case["adapters"] else torch.tensor([state["scale"]], dtype=torch.float64, device=DEVICE)
    if not case["backward"]:
        table = state["table"] if case["adapters"] else state["table"][None]
        return table[adapter, state["ids"].long()].double() * scale[adapter, None]
    # the words that occur, in order, and the gradient rows of each added up between the ends of its run
    word = adapter * case["vocab"] + state["ids"].long()
    order = torch.argsort(word, stable=True)
    words, counts = torch.unique_consecutive(word[order], return_counts=True)
    sums = torch.cat([torch.zeros(1, case["width"], dtype=torch.float64, device=DEVICE),
                      torch.cumsum(state["dy"][order].double() * scale[adapter[order], None], 0)])
    last = torch.cumsum(counts, 0)
    grad = torch.zeros(max(1, case["adapters"]) * case["vocab"], case["width"], dtype=torch.float64, device=DEVICE)
    grad[words] = sums[last] - sums[last - counts]
    return grad.view(case["adapters"], case["vocab"], -1) if case["adapters"] else grad
