"""The operators of a speculative serving step over the paged cache, as cases to be timed and compared.

A step that verifies a tree of drafted tokens runs five operators: the plan of the step (row starts, positions, slots,
block tables and ancestor masks from the lengths of the requests), the norm and rotation of queries and keys with the
append of keys and values to the pages, the attention of the tree's rows over cache and tree, and the acceptance of the
drafted tokens; training takes the gradient of the norm and rotation as well.  Every case runs either as the plain form
(elementary torch operations) or, with `own` set, as the calls a program makes of pagedattentionmetal_b200.
"""
import math
import random

import torch

own = False

_TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "fp8": torch.float16}


# ---------------------------------------------------------------- cases

def listed():
    return [
        # plan of one decode step of a full continuous batch: one new token per request, tables of up to 512 blocks
        {"name": "plan_decode_b256", "op": "plan", "batch": 256, "lo": 512, "hi": 8192, "new_lo": 1, "new_hi": 1,
         "tree": False, "block": 16, "layout": 11},
        # plan of a verification step: 64 requests with trees of up to 64 drafted tokens, masks included
        {"name": "plan_tree_b64", "op": "plan", "batch": 64, "lo": 512, "hi": 8192, "new_lo": 17, "new_hi": 64,
         "tree": True, "block": 16, "layout": 12},
        # acceptance for a handful of requests with small trees: latency only
        {"name": "accept_b8", "op": "accept", "batch": 8, "lo": 1, "hi": 512, "new_lo": 1, "new_hi": 16, "block": 16,
         "layout": 13},
        # acceptance for a full batch with trees of 64 nodes
        {"name": "accept_b256", "op": "accept", "batch": 256, "lo": 512, "hi": 8192, "new_lo": 33, "new_hi": 64,
         "block": 16, "layout": 14},
        # one layer of a decode step of 64 requests: norm, rotation, append of one token each
        {"name": "norm_decode_bf16", "op": "norm", "rows": 64, "heads": 32, "kv_heads": 8, "dim": 128, "rotary": 128,
         "interleaved": False, "dtype": "bf16", "block": 16, "far": 8192},
        # one layer of a prefill of 16 prompts of 2048 tokens
        {"name": "norm_prefill_f16", "op": "norm", "rows": 32768, "heads": 32, "kv_heads": 8, "dim": 128,
         "rotary": 128, "interleaved": False, "dtype": "f16", "block": 16, "far": 131072},
        # gradient of the norm and rotation of a training step of 8192 tokens; key gradients as rows
        {"name": "norm_backward_bf16", "op": "norm_backward", "rows": 8192, "heads": 32, "kv_heads": 8, "dim": 128,
         "rotary": 128, "interleaved": False, "dtype": "bf16", "block": 16, "far": 8192, "pages": False},
        # the same in float32 with key and value gradients gathered from the pages, partial interleaved rotation, odd rows
        {"name": "norm_backward_f32", "op": "norm_backward", "rows": 777, "heads": 8, "kv_heads": 2, "dim": 80,
         "rotary": 40, "interleaved": True, "dtype": "f32", "block": 16, "far": 2048, "pages": True},
        # one user: a small tree over one long context
        {"name": "tree_b1_bf16", "op": "tree", "batch": 1, "lo": 8192, "hi": 8192, "new_lo": 16, "new_hi": 16,
         "heads": 32, "kv_heads": 8, "dim": 128, "dtype": "bf16", "block": 16, "window": 0, "layout": 15},
        # a full batch with trees of up to 64 nodes over contexts of 512 to 8192 tokens
        {"name": "tree_b32_f16", "op": "tree", "batch": 32, "lo": 512, "hi": 8192, "new_lo": 32, "new_hi": 64,
         "heads": 32, "kv_heads": 8, "dim": 128, "dtype": "f16", "block": 16, "window": 0, "layout": 16},
        # long contexts in an 8-bit cache under a sliding window, 8 query heads per key head, small trees
        {"name": "tree_b16_fp8_window", "op": "tree", "batch": 16, "lo": 8192, "hi": 32768, "new_lo": 5, "new_hi": 8,
         "heads": 64, "kv_heads": 8, "dim": 128, "dtype": "fp8", "block": 16, "window": 4096, "layout": 17},
        # ragged float32: short contexts (some empty), odd tree sizes, an odd head dimension
        {"name": "tree_b7_f32", "op": "tree", "batch": 7, "lo": 0, "hi": 700, "new_lo": 1, "new_hi": 33,
         "heads": 6, "kv_heads": 2, "dim": 80, "dtype": "f32", "block": 8, "window": 0, "layout": 18},
    ]


def _spread(rng, lo, hi):
    """A whole number in [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["plan", "accept", "norm", "norm_backward", "tree", "tree"])
    layout = rng.randrange(1 << 30)
    if op in ("plan", "accept"):
        hi = _spread(rng, 16, 8192)
        tree = op == "accept" or rng.random() < 0.5
        new_hi = _spread(rng, 1, 128 if tree else 512)
        batch = min(_spread(rng, 1, 512), max(1, 65536 // new_hi))
        case = {"op": op, "batch": batch, "lo": rng.randrange(0, hi), "hi": hi, "new_lo": rng.randint(1, new_hi),
                "new_hi": new_hi, "block": rng.choice([8, 16, 16, 32, 24]), "layout": layout}
        return {**case, "tree": tree} if op == "plan" else case
    if op in ("norm", "norm_backward"):
        dim = rng.choice([64, 80, 96, 128, 128, 256])
        kv_heads = rng.choice([1, 2, 4, 8])
        heads = kv_heads * rng.choice([1, 2, 4, 8])
        rows = _spread(rng, 1, 8192 if op == "norm_backward" else 16384)
        case = {"op": op, "rows": rows, "heads": heads, "kv_heads": kv_heads, "dim": dim,
                "rotary": rng.choice([dim, dim, dim // 2]), "interleaved": rng.random() < 0.5,
                "dtype": rng.choice(["f32", "f16", "bf16"]), "block": rng.choice([8, 16, 32]),
                "far": rng.choice([2048, 8192, 131072])}
        return {**case, "pages": rng.random() < 0.5} if op == "norm_backward" else case
    dim = rng.choice([64, 128, 128, 128, 96, 80])
    kv_heads = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 2, 4, 7, 8])
    hi = _spread(rng, 16, 8192)
    new_hi = _spread(rng, 1, 64)
    batch = _spread(rng, 1, max(1, min(32, 131072 // hi)))
    return {"op": "tree", "batch": batch, "lo": rng.randrange(0, hi), "hi": hi, "new_lo": rng.randint(1, new_hi),
            "new_hi": new_hi, "heads": kv_heads * group, "kv_heads": kv_heads, "dim": dim,
            "dtype": rng.choice(["f16", "bf16", "bf16", "f32", "fp8"]), "block": rng.choice([16, 16, 32, 8]),
            "window": rng.choice([0, 0, 0, 256, 4096]), "layout": layout}


def _shape(case):
    """Tokens in the cache and new tokens of every request of a case: part of the case, not of the inputs."""
    rng = random.Random(case["layout"])
    lens = [rng.randint(case["lo"], case["hi"]) for _ in range(case["batch"])]
    new = [rng.randint(case["new_lo"], case["new_hi"]) for _ in range(case["batch"])]
    return lens, new


def work(case):
    op = case["op"]
    if op in ("norm", "norm_backward"):
        es = 4 if case["dtype"] == "f32" else 2
        rows, dim = case["rows"], case["dim"]
        q, kv = rows * case["heads"] * dim, rows * case["kv_heads"] * dim
        if op == "norm":
            return {"bytes": 2 * es * (q + 2 * kv) + rows * 12, "flops": 9 * (q + kv)}
        moved = 3 * (q + kv) + (2 * kv if case["pages"] else 0)
        return {"bytes": es * moved + rows * (12 if case["pages"] else 4), "flops": 18 * (q + kv)}
    lens, new = _shape(case)
    rows, batch, block = sum(new), case["batch"], case["block"]
    if op == "plan":
        used = sum(-(-(l + n) // block) for l, n in zip(lens, new))
        width = max(-(-(l + n) // block) for l, n in zip(lens, new))
        per_row = 4 + (4 + 4 * _words(case) if case["tree"] else 8)
        return {"bytes": 4 * (used + batch * width) + rows * per_row + batch * 16, "flops": rows}
    if op == "accept":
        return {"bytes": rows * 20 + batch * (20 + 4 * case["new_hi"]), "flops": rows}
    es = {"f32": 4, "f16": 2, "bf16": 2, "fp8": 1}[case["dtype"]]
    io = 4 if case["dtype"] == "f32" else 2
    seen = [min(l, case["window"]) if case["window"] else l for l in lens]
    pages = sum(-(-s // block) for s in seen)
    wide = case["kv_heads"] * case["dim"]
    return {"bytes": 2 * es * sum(seen) * wide + 2 * io * rows * wide + 2 * io * rows * case["heads"] * case["dim"]
                     + 4 * pages + rows * 4 * _words(case),
            "flops": 4 * case["dim"] * case["heads"] * sum(n * (s + 1) for n, s in zip(new, seen))}


def _words(case):
    return -(-case["new_hi"] // 32)


# ---------------------------------------------------------------- inputs

def _normal(gen, dtype, *shape, scale=1.0):
    return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(dtype)


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _parents(new, gen):
    """Draft trees: node 0 is the root, every other node hangs on one of the few nodes before it."""
    counts = torch.tensor(new)
    i = torch.arange(int(counts.sum())) - torch.repeat_interleave(counts.cumsum(0) - counts, counts)
    back = (torch.rand(i.numel(), generator=gen) * i.clamp(max=6)).floor().long()
    return torch.where(i > 0, i - 1 - back, torch.full_like(i, -1)), i


def _starts(new):
    total, out = 0, [0]
    for n in new:
        total += n
        out.append(total)
    return out


def _block_lists(lens, new, block, gen):
    """Every request's own blocks, scattered over the pool, as rows of one array."""
    need = [max(1, -(-(l + n) // block)) for l, n in zip(lens, new)]
    order = torch.randperm(sum(need) + 3, generator=gen).to(torch.int32)
    lists = torch.zeros(len(need), max(need), dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        lists[b, :n] = order[at:at + n]
        at += n
    return lists.cuda(), sum(need) + 3


def _quantise(x):
    """8-bit codes and one float16 scale for each (block, key head)."""
    scale = (x.float().abs().amax(dim=(2, 3)) / 448).to(torch.float16)
    codes = (x.float() / scale.float()[:, :, None, None]).clamp(-448, 448).to(torch.float8_e4m3fn)
    return codes, scale


def prepare(case, seed):
    host = torch.Generator().manual_seed(seed)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    state = {"case": case}
    {"plan": _prepare_plan, "accept": _prepare_accept, "norm": _prepare_norm, "norm_backward": _prepare_norm,
     "tree": _prepare_tree}[case["op"]](case, state, host, gen)
    if own:
        # what a serving loop keeps from step to step: the engine, and a request naming its static buffers
        _request(case, state)
    return state


def _prepare_plan(case, state, host, gen):
    lens, new = _shape(case)
    rows, batch, block = sum(new), case["batch"], case["block"]
    lists, _ = _block_lists(lens, new, block, host)
    pick = torch.randperm(batch, generator=host)          # the batch takes the lists in its own order
    state.update(lists=lists[torch.argsort(pick).cuda()].contiguous(), index=pick.to(torch.int32).cuda(),
                 lengths=_int32(lens), new=_int32(new), rows=rows, width=lists.shape[1])
    empty = lambda dtype, *shape: torch.empty(*shape, dtype=dtype, device="cuda")
    state.update(tables=empty(torch.int32, batch, lists.shape[1]), totals=empty(torch.int32, batch),
                 starts=empty(torch.int32, batch + 1), positions=empty(torch.int32, rows))
    if case["tree"]:
        state.update(parents=_parents(new, host)[0].to(torch.int32).cuda(),
                     masks=empty(torch.int32, rows, _words(case)))
    else:
        state.update(slots=empty(torch.int64, rows))


def _prepare_accept(case, state, host, gen):
    lens, new = _shape(case)
    rows, batch, block = sum(new), case["batch"], case["block"]
    lists, _ = _block_lists(lens, new, block, host)
    parents, i = _parents(new, host)
    starts = torch.tensor(_starts(new))
    up = torch.where(parents >= 0, parents + torch.repeat_interleave(starts[:-1], torch.tensor(new)), parents)
    draft = torch.randint(0, 128256, (rows,), generator=host)
    child = torch.full((rows + 1,), -1).scatter_reduce(0, torch.where(up >= 0, up, rows), torch.arange(rows), "amax")[:rows]
    agree = (torch.rand(rows, generator=host) < 0.8) & (child >= 0)
    target = torch.where(agree, draft[child.clamp(min=0)], torch.randint(0, 128256, (rows,), generator=host))
    dev = lambda t: t.to(torch.int32).cuda()
    empty = lambda dtype, *shape: torch.empty(*shape, dtype=dtype, device="cuda")
    state.update(starts=dev(starts), parents=dev(parents), draft=dev(draft), target=dev(target), lengths=_int32(lens),
                 tables=lists, rows=rows, slots=empty(torch.int64, rows), counts=empty(torch.int32, batch),
                 path=empty(torch.int32, batch, case["new_hi"]), next=empty(torch.int32, batch),
                 totals=empty(torch.int32, batch))


def _prepare_norm(case, state, host, gen):
    dtype, rows, dim = _TORCH[case["dtype"]], case["rows"], case["dim"]
    heads, kv, block = case["heads"], case["kv_heads"], case["block"]
    qkv = _normal(gen, dtype, rows, (heads + 2 * kv) * dim)            # the projection's output, rows of q | k | v
    blocks = -(-rows // block) + 2
    slots = torch.randperm(blocks * block, generator=gen, device="cuda")[:rows]
    state.update(
        qkv=qkv, q=qkv[:, :heads * dim], k=qkv[:, heads * dim:(heads + kv) * dim], v=qkv[:, (heads + kv) * dim:],
        q_weight=_normal(gen, dtype, dim, scale=0.2) + 1, k_weight=_normal(gen, dtype, dim, scale=0.2) + 1,
        inv_freq=(500000.0 ** (-torch.arange(0, case["rotary"], 2, device="cuda").double() / case["rotary"])).float(),
        positions=torch.randint(0, case["far"], (rows,), generator=gen, device="cuda", dtype=torch.int32), slots=slots,
        eps=1e-6)
    if case["op"] == "norm":
        pool = lambda: torch.zeros(blocks, kv, block, dim, dtype=dtype, device="cuda")
        state.update(q_out=torch.empty(rows, heads, dim, dtype=dtype, device="cuda"), k_pool=pool(), v_pool=pool())
        return
    state.update(dq_out=_normal(gen, dtype, rows, heads, dim, scale=0.5),
                 d_qkv=torch.zeros_like(qkv), dw_q=torch.empty(dim, device="cuda"), dw_k=torch.empty(dim, device="cuda"))
    d = state["d_qkv"]
    state.update(dq=d[:, :heads * dim], dk=d[:, heads * dim:(heads + kv) * dim], dv=d[:, (heads + kv) * dim:])
    if case["pages"]:
        state.update(dk_pool=_normal(gen, dtype, blocks, kv, block, dim, scale=0.5),
                     dv_pool=_normal(gen, dtype, blocks, kv, block, dim, scale=0.5))
    else:
        state.update(dk_out=_normal(gen, dtype, rows, kv, dim, scale=0.5))


def _prepare_tree(case, state, host, gen):
    lens, new = _shape(case)
    rows, block, dim, kv = sum(new), case["block"], case["dim"], case["kv_heads"]
    dtype = _TORCH[case["dtype"]]
    lists, blocks = _block_lists(lens, [0] * len(lens), block, host)
    parents, i = _parents(new, host)
    n, most = torch.tensor(new), case["new_hi"]
    starts = torch.tensor(_starts(new))
    up = torch.where(parents >= 0, parents + torch.repeat_interleave(starts[:-1], n), parents).cuda()
    sees = _ancestors(up, i.cuda(), most)
    k_pool, v_pool = _normal(gen, dtype, blocks, kv, block, dim), _normal(gen, dtype, blocks, kv, block, dim)
    if case["dtype"] == "fp8":
        k_pool, state["k_scale"] = _quantise(k_pool)
        v_pool, state["v_scale"] = _quantise(v_pool)
    state.update(
        q=_normal(gen, dtype, rows, case["heads"], dim), k=_normal(gen, dtype, rows, kv, dim),
        v=_normal(gen, dtype, rows, kv, dim), k_pool=k_pool, v_pool=v_pool, tables=lists, lengths=_int32(lens),
        starts=starts.to(torch.int32).cuda(), masks=_pack(sees, _words(case)),
        positions=(torch.repeat_interleave(torch.tensor(lens), n).cuda() + sees.sum(1) - 1).to(torch.int32),
        out=torch.empty(rows, case["heads"], dim, dtype=dtype, device="cuda"), rows=rows,
        longest=max(min(l, case["window"]) if case["window"] else l for l in lens))


# ---------------------------------------------------------------- one pass

def run(state):
    if own:
        return _run_own(state)
    return {"plan": _plain_plan, "accept": _plain_accept, "norm": _plain_norm, "norm_backward": _plain_norm_backward,
            "tree": _plain_tree}[state["case"]["op"]](state)


def _ancestors(up, i, width):
    """[rows][width]: whether node j of a row's tree is the row itself or one of its ancestors (up: the parent's row)."""
    sees = torch.arange(width, device=i.device)[None] == i[:, None]
    jump = up
    for _ in range(max(1, (width - 1).bit_length())):
        live = jump >= 0
        at = jump.clamp(min=0)
        sees = sees | (sees[at] & live[:, None])
        jump = torch.where(live, jump[at], jump)
    return sees


def _pack(bits, words):
    wide = torch.zeros(bits.shape[0], words * 32, dtype=torch.int64, device=bits.device)
    wide[:, :bits.shape[1]] = bits
    return (wide.view(-1, words, 32) << torch.arange(32, device=bits.device)).sum(2).to(torch.int32)


def _rows_of(starts, rows):
    """Sequence and place within it of every row."""
    r = torch.arange(rows, device=starts.device)
    seq = torch.searchsorted(starts[1:].contiguous(), r, right=True)
    return seq, r - starts[seq]


def _plain_plan(s):
    case = s["case"]
    block, rows = case["block"], s["rows"]
    n = s["new"].long().clamp(0, case["new_hi"])
    starts = torch.cat([n.new_zeros(1), n.cumsum(0)]).clamp(max=rows)
    n = starts[1:] - starts[:-1]
    totals = s["lengths"] + n
    lists = s["lists"][s["index"].long()]
    used = torch.arange(s["width"], device="cuda")[None] < ((totals + block - 1) // block)[:, None]
    tables = torch.where(used, lists, 0)
    seq, i = _rows_of(starts, rows)
    common = {"tables": tables, "totals": totals.to(torch.int32), "starts": starts.to(torch.int32)}
    if case["tree"]:
        parents = s["parents"].long()
        sees = _ancestors(torch.where(parents >= 0, parents + starts[seq], parents), i, case["new_hi"])
        positions = s["lengths"][seq] + sees.sum(1) - 1
        return {**common, "positions": positions.to(torch.int32), "masks": _pack(sees, _words(case))}
    positions = s["lengths"][seq] + i
    slots = lists[seq, positions // block].long() * block + positions % block
    return {**common, "positions": positions.to(torch.int32), "slots": slots}


def _plain_accept(s):
    case = s["case"]
    block, rows, most = case["block"], s["rows"], case["new_hi"]
    starts, parents, target = s["starts"].long(), s["parents"].long(), s["target"]
    seq, i = _rows_of(starts, rows)
    up = torch.where(parents >= 0, parents + starts[seq], parents)
    agrees = (parents < 0) | (s["draft"] == target[up.clamp(min=0)])
    sees = _ancestors(up, i, most)
    # a node is accepted when no node on its way to the root disagrees
    table = torch.zeros(case["batch"], most, dtype=torch.bool, device="cuda")
    table[seq, i] = ~agrees
    accepted = ~(sees & table[seq]).any(1)
    depth = sees.sum(1) - 1
    rank = torch.where(accepted, (depth + 1) * 4096 - i, 0)
    best_rank = torch.zeros(case["batch"], dtype=rank.dtype, device="cuda").scatter_reduce(0, seq, rank, "amax")
    count = (best_rank + 4095) // 4096
    best = starts[:-1] + count * 4096 - best_rank
    on_path = sees[best][seq, i]
    at = s["lengths"][seq] + depth
    slots = torch.where(on_path, s["tables"][seq, at // block].long() * block + at % block, -1)
    path = torch.full((case["batch"], most + 1), -1, dtype=torch.int64, device="cuda")
    path[seq, torch.where(on_path, depth, most)] = torch.where(on_path, torch.arange(rows, device="cuda"), -1)
    return {"slots": slots, "counts": count.to(torch.int32), "path": path[:, :most].to(torch.int32),
            "next": target[best], "totals": (s["lengths"] + count).to(torch.int32)}


def _rotation(s):
    angle = s["positions"].double()[:, None] * s["inv_freq"].double()
    return angle.cos().float()[:, None], angle.sin().float()[:, None]


def _pairs(x, case):
    """The two halves of every rotated pair of a row."""
    r = x[..., :case["rotary"]]
    if case["interleaved"]:
        return r[..., 0::2], r[..., 1::2]
    return r[..., :case["rotary"] // 2], r[..., case["rotary"] // 2:]


def _joined(a, b, x, case):
    r = torch.stack([a, b], -1).flatten(-2) if case["interleaved"] else torch.cat([a, b], -1)
    return torch.cat([r, x[..., case["rotary"]:]], -1)


def _plain_norm(s):
    case = s["case"]
    rows, dim, dtype = case["rows"], case["dim"], s["qkv"].dtype
    cos, sin = _rotation(s)

    def turned(x, weight):
        x = x.reshape(rows, -1, dim).float()
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + s["eps"]) * weight.float()
        a, b = _pairs(x, case)
        return _joined(a * cos - b * sin, b * cos + a * sin, x, case).to(dtype)

    blk, off = s["slots"] // case["block"], s["slots"] % case["block"]
    s["k_pool"][blk, :, off] = turned(s["k"], s["k_weight"])
    s["v_pool"][blk, :, off] = s["v"].reshape(rows, -1, dim)
    return {"q": turned(s["q"], s["q_weight"]), "k_pool": s["k_pool"], "v_pool": s["v_pool"]}


def _plain_norm_backward(s):
    case = s["case"]
    rows, dim, dtype = case["rows"], case["dim"], s["qkv"].dtype
    cos, sin = _rotation(s)

    def back(x, weight, dy):
        x, dy = x.reshape(rows, -1, dim).float(), dy.float()
        a, b = _pairs(dy, case)
        dn = _joined(a * cos + b * sin, b * cos - a * sin, dy, case)
        r = torch.rsqrt((x * x).mean(-1, keepdim=True) + s["eps"])
        xhat, g = x * r, dn * weight.float()
        dx = r * (g - xhat * (g * xhat).mean(-1, keepdim=True))
        return dx.to(dtype), (dn * xhat).double().sum((0, 1)).float()

    if case["pages"]:
        blk, off = s["slots"] // case["block"], s["slots"] % case["block"]
        dk_out = s["dk_pool"][blk, :, off]
    else:
        dk_out = s["dk_out"]
    dq, dw_q = back(s["q"], s["q_weight"], s["dq_out"])
    dk, dw_k = back(s["k"], s["k_weight"], dk_out)
    out = {"dq": dq.view(rows, -1), "dk": dk.view(rows, -1), "dw_q": dw_q, "dw_k": dw_k}
    return {**out, "dv": s["dv_pool"][blk, :, off].reshape(rows, -1)} if case["pages"] else out


def _plain_tree(s):
    case = s["case"]
    batch, heads, kv, dim, block = case["batch"], case["heads"], case["kv_heads"], case["dim"], case["block"]
    most, rows, group = case["new_hi"], s["rows"], case["heads"] // case["kv_heads"]
    starts, lens = s["starts"].long(), s["lengths"].long()
    seq, i = _rows_of(starts, rows)
    # the visible tail of every context, token by token through the block table
    first = (lens - case["window"]).clamp(min=0) if case["window"] else torch.zeros_like(lens)
    token = first[:, None] + torch.arange(max(s["longest"], 1), device="cuda")
    held = token < lens[:, None]
    token = torch.where(held, token, 0)
    blk = s["tables"].long().gather(1, token // block)

    def cached(pool, scale, fresh):
        x = pool.float() if scale is None else pool.float() * scale.float()[:, :, None, None]
        x = torch.where(held[:, :, None, None], x[blk, :, token % block], 0)                # [batch][token][kv][dim]
        mine = torch.zeros(batch, most, kv, dim, device="cuda")
        mine[seq, i] = fresh.float()
        return torch.cat([x, mine], 1).transpose(1, 2)                                      # [batch][kv][key][dim]

    keys = cached(s["k_pool"], s.get("k_scale"), s["k"])
    values = cached(s["v_pool"], s.get("v_scale"), s["v"])
    q = torch.zeros(batch, most, heads, dim, device="cuda")
    q[seq, i] = s["q"].float()
    q = q.view(batch, most, kv, group, dim).permute(0, 2, 3, 1, 4).reshape(batch, kv, group * most, dim)
    sees = ((s["masks"][:, :, None] >> torch.arange(32, device="cuda")) & 1).bool().flatten(1)[:, :most]
    mask = torch.zeros(batch, most, token.shape[1] + most, dtype=torch.bool, device="cuda")
    position = s["positions"].long()
    near = token[seq] > (position - case["window"])[:, None] if case["window"] else True
    in_tree = sees
    if case["window"]:
        place = torch.zeros(batch, most, dtype=torch.int64, device="cuda")
        place[seq, i] = position
        in_tree = sees & (place[seq] > (position - case["window"])[:, None])
    mask[seq, i] = torch.cat([held[seq] & near, in_tree], 1)
    mask = mask[:, None].expand(batch, group, most, -1).reshape(batch, 1, group * most, -1)
    scores = (q @ keys.transpose(2, 3)) * (1.0 / math.sqrt(dim))
    scores = scores.masked_fill(~mask, -torch.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -torch.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    o = (p @ values) / torch.where(total == 0, 1.0, total)
    o = o.view(batch, kv, group, most, dim).permute(0, 3, 1, 2, 4).reshape(batch, most, heads, dim)
    return {"out": o[seq, i].to(s["q"].dtype)}


# ---------------------------------------------------------------- the framework's calls

_ENGINE = None


def _engine(pam):
    """The program's engine: asynchronous, on torch's current stream (1 names the legacy default stream)."""
    global _ENGINE
    if _ENGINE is None:
        _ENGINE = pam.PagedAttentionEngine(torch.cuda.current_device())
        _ENGINE.setAsync(True)
        _ENGINE.enableGracefulDegradation = False
        _ENGINE.setStream(torch.cuda.current_stream().cuda_stream or 1)
    return _ENGINE


def _request(case, s):
    import pagedattentionmetal_b200 as pam

    kind = pam.PagedAttentionDataType
    s["engine"] = _engine(pam)
    op = case["op"]
    if op == "plan":
        s["request"] = pam.PagedStepPlanRequest(
            blockLists=s["lists"], lengths=s["lengths"], newTokens=s["new"], batchSize=case["batch"],
            numLists=s["lists"].shape[0], listStride=s["lists"].shape[1], blockSize=case["block"], numRows=s["rows"],
            maxNewTokens=case["new_hi"], listIndex=s["index"], parents=s.get("parents"), tables=s["tables"],
            maxNumBlocks=s["width"], totalLengths=s["totals"], rowStarts=s["starts"], positions=s["positions"],
            slots=s.get("slots"), masks=s.get("masks"), maskWords=_words(case) if case["tree"] else 0)
        return
    if op == "accept":
        s["request"] = pam.PagedAcceptRequest(
            rowStarts=s["starts"], parents=s["parents"], draftTokens=s["draft"], targetTokens=s["target"],
            lengths=s["lengths"], batchSize=case["batch"], numRows=s["rows"], maxTree=case["new_hi"],
            blockTables=s["tables"], maxNumBlocks=s["tables"].shape[1], blockSize=case["block"], slots=s["slots"],
            acceptedCounts=s["counts"], acceptedRows=s["path"], maxPath=case["new_hi"], nextTokens=s["next"],
            newLengths=s["totals"])
        return
    data = {"f32": kind.float32, "f16": kind.float16, "bf16": kind.bfloat16, "fp8": kind.float8}[case["dtype"]]
    layer = pam.PagedLayerSpec(case["dim"], case["heads"], case["kv_heads"], case["block"], data, case.get("window", 0))
    if op == "tree":
        s["request"] = pam.PagedTreeAttentionRequest(
            q=s["q"], k=s["k"], v=s["v"], kPool=s["k_pool"], vPool=s["v_pool"], blockTables=s["tables"],
            cacheLengths=s["lengths"], rowStarts=s["starts"], masks=s["masks"], positions=s["positions"],
            output=s["out"], batchSize=case["batch"], maxNumBlocks=s["tables"].shape[1], numRows=s["rows"],
            maxNewTokens=case["new_hi"], maskWords=_words(case), layer=layer, kScaleBuffer=s.get("k_scale"),
            vScaleBuffer=s.get("v_scale"))
        return
    wide = s["qkv"].shape[1]
    common = dict(q=s["q"], k=s["k"], qWeight=s["q_weight"], kWeight=s["k_weight"], invFreq=s["inv_freq"],
                  positions=s["positions"], numRows=case["rows"], layer=layer, rotaryDim=case["rotary"],
                  interleaved=case["interleaved"], epsilon=s["eps"], qStride=wide, kStride=wide)
    if op == "norm":
        s["request"] = pam.PagedNormRotateRequest(v=s["v"], vStride=wide, qOut=s["q_out"], kPool=s["k_pool"],
                                                  vPool=s["v_pool"], slots=s["slots"], **common)
        return
    pages = dict(dKPool=s["dk_pool"], dVPool=s["dv_pool"], slots=s["slots"], dV=s["dv"], dVStride=wide) if case["pages"] \
        else dict(dKOut=s["dk_out"])
    s["request"] = pam.PagedNormRotateBackwardRequest(dQOut=s["dq_out"], dQ=s["dq"], dK=s["dk"], dQStride=wide,
                                                      dKStride=wide, dQWeight=s["dw_q"], dKWeight=s["dw_k"], **pages,
                                                      **common)


def _run_own(s):
    op, engine, request = s["case"]["op"], s["engine"], s["request"]
    if op == "plan":
        engine.planStep(request)
        common = {x: s[x] for x in ("tables", "totals", "starts", "positions")}
        return {**common, "masks": s["masks"]} if s["case"]["tree"] else {**common, "slots": s["slots"]}
    if op == "accept":
        engine.acceptTree(request)
        return {x: s[x] for x in ("slots", "counts", "path", "next", "totals")}
    if op == "norm":
        engine.normRotate(request)
        return {"q": s["q_out"], "k_pool": s["k_pool"], "v_pool": s["v_pool"]}
    if op == "norm_backward":
        engine.normRotateBackward(request)
        out = {x: s[x] for x in ("dq", "dk", "dw_q", "dw_k")}
        return {**out, "dv": s["dv"]} if s["case"]["pages"] else out
    engine.treeAttention(request)
    return {"out": s["out"]}


# ---------------------------------------------------------------- the definitions in 64 bits

def exact(case, seed):
    global own
    kept, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = kept
    if case["op"] in ("plan", "accept"):
        return None                          # whole numbers
    return {"norm": _exact_norm, "norm_backward": _exact_norm_backward, "tree": _exact_tree}[case["op"]](s)


def _exact_turn(s, x, weight):
    """Norm and rotation of rows [rows][heads][dim] in float64, pair by pair as complex numbers."""
    case = s["case"]
    half = case["rotary"] // 2
    x = x * (x.pow(2).mean(-1, keepdim=True) + s["eps"]).pow(-0.5) * weight
    head, tail = x[..., :case["rotary"]], x[..., case["rotary"]:]
    pairs = head.unflatten(-1, (half, 2)) if case["interleaved"] else head.unflatten(-1, (2, half)).transpose(-1, -2)
    angle = (s["positions"].double()[:, None] * s["inv_freq"].double())[:, None]
    turned = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * torch.polar(torch.ones_like(angle), angle))
    turned = turned if case["interleaved"] else turned.transpose(-1, -2)
    return torch.cat([turned.flatten(-2), tail], -1)


def _exact_norm(s):
    case = s["case"]
    rows, dim = case["rows"], case["dim"]
    split = lambda x: x.double().reshape(rows, -1, dim)
    k_pool, v_pool = s["k_pool"].double(), s["v_pool"].double()
    flat = lambda pool: pool.transpose(1, 2).reshape(-1, case["kv_heads"], dim)
    unflat = lambda x: x.view(-1, case["block"], case["kv_heads"], dim).transpose(1, 2)
    k_rows, v_rows = flat(k_pool).clone(), flat(v_pool).clone()
    k_rows[s["slots"]] = _exact_turn(s, split(s["k"]), s["k_weight"].double())
    v_rows[s["slots"]] = split(s["v"])
    return {"q": _exact_turn(s, split(s["q"]), s["q_weight"].double()), "k_pool": unflat(k_rows), "v_pool": unflat(v_rows)}


def _exact_norm_backward(s):
    case = s["case"]
    rows, dim = case["rows"], case["dim"]
    flat = lambda pool: pool.double().transpose(1, 2).reshape(-1, case["kv_heads"], dim)[s["slots"]]
    leaf = lambda x: x.double().contiguous().requires_grad_(True)
    out = {}
    for name, dy in (("q", s["dq_out"].double()),
                     ("k", flat(s["dk_pool"]) if case["pages"] else s["dk_out"].double())):
        x, weight = leaf(s[name].reshape(rows, -1, dim)), leaf(s[name + "_weight"])
        dx, dw = torch.autograd.grad(_exact_turn(s, x, weight), (x, weight), dy)
        out["d" + name], out["dw_" + name] = dx.reshape(rows, -1), dw
    answer = {x: out[x] for x in ("dq", "dk", "dw_q", "dw_k")}
    return {**answer, "dv": flat(s["dv_pool"]).reshape(rows, -1)} if case["pages"] else answer


def _exact_tree(s):
    """Sequence by sequence, over the tokens that its rows may see."""
    case = s["case"]
    block, dim, kv = case["block"], case["dim"], case["kv_heads"]
    lens, new = _shape(case)
    out = torch.zeros(s["rows"], case["heads"], dim, dtype=torch.float64, device="cuda")
    at = 0
    for b, (length, n) in enumerate(zip(lens, new)):
        first = max(0, length - case["window"]) if case["window"] else 0
        token = torch.arange(first, length, device="cuda")
        page = s["tables"][b].long()[token // block]

        def joined(pool, scale, fresh):
            x = pool[page, :, token % block].double()
            if scale is not None:
                x = x * scale[page].double()[:, :, None]
            return torch.cat([x, fresh[at:at + n].double()])

        keys = joined(s["k_pool"], s.get("k_scale"), s["k"])
        values = joined(s["v_pool"], s.get("v_scale"), s["v"])
        words = s["masks"][at:at + n].long() & 0xFFFFFFFF
        node = torch.arange(n, device="cuda")
        sees = (words[:, node // 32] >> (node % 32)) & 1 == 1
        position = s["positions"][at:at + n].long()
        place = torch.cat([token, position])
        mask = torch.cat([torch.ones(n, token.numel(), dtype=torch.bool, device="cuda"), sees], 1)
        if case["window"]:
            mask &= place[None] > position[:, None] - case["window"]
        q = s["q"][at:at + n].double().view(n, kv, -1, dim)
        scores = torch.einsum("nkgd,tkd->nkgt", q, keys) / math.sqrt(dim)
        weights = torch.softmax(scores.masked_fill(~mask[:, None, None], -torch.inf), -1)
        out[at:at + n] = torch.einsum("nkgt,tkd->nkgd", weights, values).reshape(n, -1, dim)
        at += n
    return {"out": out}
