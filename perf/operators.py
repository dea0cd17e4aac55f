"""The operators of a step over drafted tokens on the ragged paged cache, as cases to measure: the step's block
tables and slot map (`rpa_plan`), the norm and rotation of its queries and keys with the cache write
(`qk_norm_rope`, `rpa_norm_rope_write`), the attention of a tree of drafted tokens (`rpa_tree_attention`) and the
accepted path's rows moved together (`rpa_commit`).

`run` computes a case in elementary torch operations (`own` false) or through `tilejax_b200.ops` (`own` true).
"""

import math

import numpy as np
import torch

own = False
D = 128  # the head dimension of the ragged paged cache


# ------------------------------------------------------------------------------------------ cases


def listed():
    return [
        # One conversation, a small tree: what a single user waits for, one launch long.
        dict(name="tree one sequence", op="tree", seqs=1, nodes=8, nodes_low=8, ctx_low=500, ctx=500, heads=32,
             kv_heads=8, page=16),
        # An ordinary serving batch with trees of sixteen tokens on pages of 128.
        dict(name="tree batch", op="tree", seqs=32, nodes=16, nodes_low=16, ctx_low=256, ctx=4096, heads=32, kv_heads=8,
             page=128),
        # Seven query heads to a KV head, odd tree sizes and lengths, pages that end inside every block.
        dict(name="tree odd", op="tree", seqs=13, nodes=25, nodes_low=3, ctx_low=7, ctx=2749, heads=28, kv_heads=4,
             page=48),
        # Two long documents, the largest trees: few sequences, each cache split over the whole GPU.
        dict(name="tree long", op="tree", seqs=2, nodes=64, nodes_low=61, ctx_low=120001, ctx=131007, heads=32,
             kv_heads=8, page=128),
        # The largest batch: ragged trees of up to 64 tokens over caches of up to 8192 positions on pages of 16.
        dict(name="tree large", op="tree", seqs=64, nodes=64, nodes_low=17, ctx_low=1000, ctx=8100, heads=32, kv_heads=8,
             page=16),
        # The new tokens of one small tree: latency.
        dict(name="write one sequence", op="write", tokens=8, heads=32, kv_heads=8, page=16, pool=256, rot=128,
             interleaved=False, packed=True, norm=True),
        # The drafted tokens of the large batch, as views of one projection's output.
        dict(name="write large", op="write", tokens=4096, heads=32, kv_heads=8, page=16, pool=2048, rot=128,
             interleaved=False, packed=True, norm=True),
        # A prompt's queries and keys without a cache, neighbouring elements rotated, half of the head only.
        dict(name="norm rope prompt", op="norm", tokens=16384, heads=32, kv_heads=8, rot=64, interleaved=True,
             packed=False, norm=True),
        # Tables of an ordinary batch of trees.
        dict(name="plan batch", op="plan", seqs=32, new=16, new_low=16, ctx=4096, page=128, pages_per_seq=64,
             depths=True),
        # Tables of a large mixed step: one-token sequences and chunks of prompts on small pages.
        dict(name="plan large", op="plan", seqs=1024, new=511, new_low=1, ctx=8000, page=16, pages_per_seq=640,
             depths=False),
        # Accepted paths of one tree, and of a large batch.
        dict(name="commit one sequence", op="commit", seqs=1, nodes=16, path=5, ctx=500, kv_heads=8, page=16),
        dict(name="commit large", op="commit", seqs=256, nodes=64, path=16, ctx=500, kv_heads=8, page=16),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["tree", "tree", "tree", "write", "norm", "plan", "commit"])
    kv_heads = rng.choice([1, 2, 4, 8])
    if op == "tree":
        while True:
            heads = kv_heads * rng.choice([1, 2, 3, 4, 5, 7, 8])
            case = dict(op="tree", seqs=_log(rng, 1, 64), nodes=_log(rng, 1, 64), ctx=_log(rng, 1, 131072), heads=heads,
                        kv_heads=kv_heads, page=rng.choice([16, 32, 48, 64, 128, 256]))
            case["nodes_low"] = rng.randint(max(1, case["nodes"] // 4), case["nodes"])
            case["ctx_low"] = rng.randint(1, case["ctx"])
            if case["seqs"] * case["ctx"] * kv_heads <= 64 * 8100 * 4 and case["seqs"] * case["ctx"] * heads * case["nodes"] <= 64 * 8100 * 32 * 32:
                return case
    if op in ("write", "norm"):
        case = dict(op=op, tokens=_log(rng, 1, 4096), heads=kv_heads * rng.choice([1, 2, 3, 4, 5, 8]), kv_heads=kv_heads,
                    rot=rng.choice([32, 64, 96, 128]), interleaved=rng.random() < 0.5, packed=rng.random() < 0.5,
                    norm=rng.random() < 0.8)
        if op == "write":
            case["page"] = rng.choice([16, 32, 48, 64, 128])
            case["pool"] = -(-2 * case["tokens"] // case["page"]) + rng.randint(1, 64)
        return case
    if op == "plan":
        new = _log(rng, 1, 511)
        page = rng.choice([16, 32, 64, 128])
        ctx = _log(rng, 1, 8000)
        return dict(op="plan", seqs=_log(rng, 1, 1024), new=new, new_low=rng.randint(1, new), ctx=ctx, page=page,
                    pages_per_seq=-(-(ctx + new) // page) + rng.randint(0, 16), depths=rng.random() < 0.5)
    path = rng.randint(1, 16)
    return dict(op="commit", seqs=_log(rng, 1, 256), nodes=rng.randint(2 * path, 2 * path + 32), path=path,
                ctx=_log(rng, 1, 500), kv_heads=kv_heads, page=rng.choice([16, 32, 48, 128]))


def _spread(low, high, n):
    """n whole numbers from low to high: the same for every seed, so that the work is the case's."""
    return np.rint(np.linspace(high, low, n)).astype(np.int64)


# ------------------------------------------------------------------------------------------ inputs


def _random(shape, gen, scale=1.0):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.bfloat16).mul_(scale)


def _int32(values):
    return torch.as_tensor(np.ascontiguousarray(values), dtype=torch.int32).cuda()


def _page_table(lens, page, rng, spare=0):
    """Block tables (seqs, pages_per_seq) over a pool just large enough, every page somewhere else."""
    pages = -(-lens // page)
    pages_per_seq = int(max(1, pages.max())) + spare
    pool = int(pages.sum()) + 3
    order = rng.permutation(pool)[: int(pages.sum())]
    table = np.zeros((len(lens), pages_per_seq), np.int64)
    at = 0
    for s, n in enumerate(pages):
        table[s, :n] = order[at : at + n]
        at += n
    return table, pool


def _ancestors(nodes, rng):
    """A drafted tree in level order: each node sees itself and its ancestors."""
    sees = np.zeros((nodes, nodes), bool)
    for i in range(nodes):
        if i:
            sees[i] = sees[rng.integers(max(0, i // 2 - 2), i)]
        sees[i, i] = True
    return sees


def _pack(sees, words):
    bits = np.zeros((sees.shape[0], words * 32), bool)
    bits[:, : sees.shape[1]] = sees
    packed = np.packbits(bits.reshape(-1, words, 32), axis=-1, bitorder="little")
    return np.ascontiguousarray(packed).view("<i4").reshape(-1, words)


def _table_of_angles(positions, rot):
    """cos and sin of every position's angles, (positions, rot) f32: cosines first, then sines."""
    rates = 10000.0 ** (-torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / rot)
    angles = torch.arange(positions, device="cuda", dtype=torch.float64)[:, None] * rates
    return torch.cat([angles.cos(), angles.sin()], 1).float()


def prepare(case, seed):
    rng = np.random.default_rng(seed)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    state = {"case": case}
    if case["op"] == "tree":
        seqs, hkv, page = case["seqs"], case["kv_heads"], case["page"]
        q_lens = _spread(case["nodes_low"], case["nodes"], seqs)
        ctx = rng.permutation(_spread(case["ctx_low"], case["ctx"], seqs))
        lens = ctx + q_lens
        table, pool = _page_table(lens, page, rng)
        words = -(-case["nodes"] // 32)
        tokens = int(q_lens.sum())
        state.update(
            q=_random((tokens, case["heads"], D), gen), kv_cache=_random((pool, page, hkv, 2, D), gen),
            kv_lens=_int32(lens), page_indices=_int32(table.reshape(-1)),
            cu_q_lens=_int32(np.concatenate([[0], np.cumsum(q_lens)])),
            tree_mask=_int32(np.concatenate([_pack(_ancestors(int(n), rng), words) for n in q_lens])),
            distribution=_int32([seqs, seqs, seqs]), sm_scale=D**-0.5, q_host=[int(n) for n in q_lens],
            lens_host=[int(n) for n in lens])
    elif case["op"] in ("write", "norm"):
        T, H, hkv = case["tokens"], case["heads"], case["kv_heads"]
        if case["packed"]:  # the projection's output, queries, keys and values side by side
            qkv = _random((T, H + 2 * hkv, D), gen)
            q, k, v = qkv[:, :H], qkv[:, H : H + hkv], qkv[:, H + hkv :]
        else:
            q, k, v = (_random((T, h, D), gen) for h in (H, hkv, hkv))
        state.update(q=q, k=k, v=v, positions=_int32(rng.integers(0, 32768, T)),
                     cos_sin=_table_of_angles(32768, case["rot"]), eps=1e-6, interleaved=case["interleaved"],
                     q_gamma=None, k_gamma=None)
        if case["norm"]:
            state.update(q_gamma=(1 + _random((D,), gen, 0.1)), k_gamma=(1 + _random((D,), gen, 0.1)))
        if case["op"] == "write":
            state.update(kv_cache=_random((case["pool"], case["page"], hkv, 2, D), gen),
                         slots=_int32(rng.permutation(case["pool"] * case["page"])[:T]))
    elif case["op"] == "plan":
        seqs, page, pps = case["seqs"], case["page"], case["pages_per_seq"]
        q_lens = rng.permutation(_spread(case["new_low"], case["new"], seqs))
        ctx = rng.permutation(_spread(0, case["ctx"], seqs))
        ctx[ctx < case["ctx"] // 10] = 0  # requests that have just come in
        held = -(-ctx // page)
        order = rng.permutation(int(held.sum() + (-(-(ctx + q_lens) // page)).sum()) + 8)
        table = np.full((seqs, pps), -1, np.int64)
        at = 0
        for s, n in enumerate(held):
            table[s, :n] = order[at : at + n]
            at += n
        tokens = int(q_lens.sum())
        state.update(ctx_lens=_int32(ctx), q_lens=_int32(q_lens), page_indices=_int32(table.reshape(-1)),
                     free_pages=_int32(order[at:]), n_free=_int32([len(order) - at]), page_size=page, tokens=tokens,
                     pages_held=_int32(held), depths=None)
        if case["depths"]:
            state["depths"] = _int32(np.concatenate([np.sort(rng.integers(0, 6, n)) for n in q_lens]))
    else:
        seqs, n, page = case["seqs"], case["nodes"], case["page"]
        lens = rng.permutation(_spread(0, case["ctx"], seqs)) + n
        table, pool = _page_table(lens, page, rng)
        accepted = _spread(1, case["path"], seqs)
        paths = np.zeros((seqs, case["path"]), np.int64)
        for s, a in enumerate(accepted):
            # The root, then nodes of deeper levels, which in a tree wider than deep lie behind the accepted count.
            paths[s, 1:a] = np.sort(rng.permutation(np.arange(a, n))[: a - 1])
        state.update(kv_cache=_random((pool, page, case["kv_heads"], 2, D), gen), kv_lens=_int32(lens),
                     page_indices=_int32(table.reshape(-1)), cu_q_lens=_int32(np.arange(seqs + 1) * n),
                     paths=_int32(paths), n_accepted=_int32(accepted))
    return state


# ------------------------------------------------------------------------------------------ one pass


def run(state):
    return (_own if own else _plain)[state["case"]["op"]](state)


def _own_tree(st):
    from tilejax_b200 import ops

    return ops.rpa_tree_attention(st["q"], st["kv_cache"], st["kv_lens"], st["page_indices"], st["cu_q_lens"],
                                  st["tree_mask"], st["distribution"], st["sm_scale"])


def _own_write(st):
    from tilejax_b200 import ops

    return ops.rpa_norm_rope_write(st["q"], st["k"], st["v"], st["q_gamma"], st["k_gamma"], st["positions"],
                                   st["cos_sin"], st["kv_cache"], st["slots"], eps=st["eps"],
                                   interleaved=st["interleaved"])


def _own_norm(st):
    from tilejax_b200 import ops

    return ops.qk_norm_rope(st["q"], st["k"], st["q_gamma"], st["k_gamma"], st["positions"], st["cos_sin"],
                            eps=st["eps"], interleaved=st["interleaved"])


def _own_plan(st):
    from tilejax_b200 import ops

    step = ops.rpa_plan(st["ctx_lens"], st["q_lens"], st["page_indices"], st["free_pages"], st["n_free"],
                        st["page_size"], st["tokens"], pages_held=st["pages_held"], depths=st["depths"])
    return (step.kv_lens, step.cu_q_lens, step.positions, step.slots, step.pages_held, step.n_free, st["page_indices"])


def _own_commit(st):
    from tilejax_b200 import ops

    lens = ops.rpa_commit(st["kv_cache"], st["kv_lens"], st["page_indices"], st["cu_q_lens"], st["paths"],
                          st["n_accepted"])
    return lens, st["kv_cache"]


_own = dict(tree=_own_tree, write=_own_write, norm=_own_norm, plan=_own_plan, commit=_own_commit)


def _unpack(mask, nodes):
    bits = (mask[:, :, None] >> torch.arange(32, device=mask.device, dtype=torch.int32)) & 1
    return bits.reshape(mask.shape[0], -1)[:, :nodes].bool()


def _plain_tree(st):
    """softmax(sm_scale q K^T over the cached prefix and the node's ancestors) V, a sequence at a time."""
    q, cache = st["q"], st["kv_cache"]
    pages, page, hkv, _, d = cache.shape
    H = q.shape[1]
    table = st["page_indices"].view(st["kv_lens"].shape[0], -1)
    out = torch.empty_like(q)
    first = 0
    for s, (n, length) in enumerate(zip(st["q_host"], st["lens_host"])):
        used = table[s, : -(-length // page)].long()
        kv = cache[used].view(-1, hkv, 2, d)[:length].float()
        k, v = kv[:, :, 0].permute(1, 2, 0), kv[:, :, 1].permute(1, 0, 2)
        rows = q[first : first + n].float().view(n, hkv, H // hkv, d).permute(1, 0, 2, 3).reshape(hkv, -1, d)
        scores = ((rows @ k) * st["sm_scale"]).view(hkv, n, H // hkv, length)
        hidden = ~_unpack(st["tree_mask"][first : first + n], n)
        scores[..., length - n :].masked_fill_(hidden[None, :, None], -math.inf)
        p = (scores - scores.amax(-1, keepdim=True)).exp()
        p = (p / p.sum(-1, keepdim=True)).view(hkv, -1, length)
        o = (p @ v).view(hkv, n, H // hkv, d).permute(1, 0, 2, 3)
        out[first : first + n] = o.reshape(n, H, d).to(q.dtype)
        first += n
    return out


def _norm_rotate(x, gamma, st):
    y = x.float()
    if gamma is not None:
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + st["eps"]) * gamma.float()
    cs = st["cos_sin"][st["positions"].long()]
    half = cs.shape[1] // 2
    cos, sin = cs[:, None, :half], cs[:, None, half:]
    if st["interleaved"]:
        a, b = y[..., 0 : 2 * half : 2], y[..., 1 : 2 * half : 2]
        turned = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    else:
        a, b = y[..., :half], y[..., half : 2 * half]
        turned = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    return torch.cat([turned, y[..., 2 * half :]], -1).to(x.dtype)


def _plain_norm(st):
    return _norm_rotate(st["q"], st["q_gamma"], st), _norm_rotate(st["k"], st["k_gamma"], st)


def _plain_write(st):
    q, k = _plain_norm(st)
    rows = st["kv_cache"].view(-1, *st["kv_cache"].shape[2:])
    rows[st["slots"].long()] = torch.stack([k, st["v"]], 2)
    return q, st["kv_cache"]


def _plain_plan(st):
    page, T = st["page_size"], st["tokens"]
    ctx, new = st["ctx_lens"].long(), st["q_lens"].long()
    S = ctx.shape[0]
    table = st["page_indices"].view(S, -1)
    pps = table.shape[1]
    lens = ctx + new
    cu = torch.cat([torch.zeros(1, device="cuda", dtype=torch.long), new.cumsum(0)])
    held = st["pages_held"].long()
    need = (((lens + page - 1) // page).clamp(max=pps) - held).clamp(min=0)
    before = need.cumsum(0) - need
    free = st["n_free"].long()[0]
    column = torch.arange(pps, device="cuda")
    fresh = (column >= held[:, None]) & (column < (held + need)[:, None])
    k = before[:, None] + column - held[:, None]
    taken = st["free_pages"].long()[(free - 1 - k).clamp(0, st["free_pages"].shape[0] - 1)]
    taken = torch.where(k < free, taken, -1)
    table.copy_(torch.where(fresh, taken, table.long()))
    token = torch.arange(T, device="cuda")
    seq = torch.searchsorted(cu, token, right=True) - 1
    index = token - cu[seq]
    place = ctx[seq] + index
    entry = table[seq, (place // page).clamp(max=pps - 1)].long()
    slots = torch.where((entry >= 0) & (place // page < pps), entry * page + place % page, -1)
    positions = place if st["depths"] is None else ctx[seq] + st["depths"]
    served = (free - before).clamp(min=0).minimum(need)
    left = torch.stack([(free - need.sum()).clamp(min=0), (need.sum() - free).clamp(min=0)])
    return tuple(t.int() for t in (lens, cu, positions, slots, held + served, left)) + (st["page_indices"],)


def _plain_commit(st):
    cache, page = st["kv_cache"], st["kv_cache"].shape[1]
    rows = cache.view(-1, *cache.shape[2:])
    table = st["page_indices"].view(st["kv_lens"].shape[0], -1).long()
    ctx = st["kv_lens"].long() - (st["cu_q_lens"][1:] - st["cu_q_lens"][:-1]).long()
    depth = torch.arange(st["paths"].shape[1], device="cuda")
    kept = depth < st["n_accepted"][:, None]

    def row(place):
        return torch.gather(table, 1, place // page) * page + place % page

    source = ctx[:, None] + torch.where(kept, st["paths"].long(), 0)
    target = torch.where(kept, ctx[:, None] + depth, source)
    rows[row(target)] = rows[row(source)]
    return (ctx + st["n_accepted"]).int(), cache


_plain = dict(tree=_plain_tree, write=_plain_write, norm=_plain_norm, plan=_plain_plan, commit=_plain_commit)


# ------------------------------------------------------------------------------------------ from the definition


def exact(case, seed):
    if case["op"] in ("plan", "commit"):
        return None  # whole numbers, and rows moved as they are
    st = prepare(case, seed)
    if case["op"] == "tree":
        return _exact_tree(st)
    q = _exact_turn(st["q"], st["q_gamma"], st)
    k = _exact_turn(st["k"], st["k_gamma"], st)
    if case["op"] == "norm":
        return q, k
    cache = st["kv_cache"].double()
    page = case["page"]
    at = st["slots"].long()
    cache[at // page, at % page, :, 0] = k
    cache[at // page, at % page, :, 1] = st["v"].double()
    return q, cache


def _exact_tree(st):
    """Every sequence and KV head by itself: exponentials over the visible positions only, in float64."""
    q, cache, mask = st["q"], st["kv_cache"], st["tree_mask"].cpu().numpy()
    S = st["kv_lens"].shape[0]
    table = st["page_indices"].cpu().numpy().reshape(S, -1)
    group = q.shape[1] // cache.shape[2]
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    t = 0
    for s, (n, length) in enumerate(zip(st["q_host"], st["lens_host"])):
        spot = np.arange(length)
        pages = torch.as_tensor(table[s, spot // cache.shape[1]].astype(np.int64)).cuda()
        offsets = torch.as_tensor(spot % cache.shape[1]).cuda()
        visible = np.ones((n, length), bool)
        for i in range(n):
            for j in range(n):
                visible[i, length - n + j] = bool((int(mask[t + i, j // 32]) >> (j % 32)) & 1)
        visible = torch.as_tensor(visible).cuda().repeat_interleave(group, 0)
        for h in range(cache.shape[2]):
            kv = cache[:, :, h][pages, offsets].double()
            heads = q[t : t + n, h * group : (h + 1) * group].double().reshape(n * group, -1)
            z = torch.einsum("rd,pd->rp", heads, kv[:, 0]) * st["sm_scale"]
            z = torch.where(visible, z, torch.full_like(z, -math.inf))
            w = torch.exp(z - z.max(1, keepdim=True).values)
            o = torch.einsum("rp,pd->rd", w, kv[:, 1]) / w.sum(1, keepdim=True)
            out[t : t + n, h * group : (h + 1) * group] = o.reshape(n, group, -1)
        t += n
    return out


def _exact_turn(x, gamma, st):
    """The norm, then each pair turned as a complex number by its position's angle."""
    y = x.double()
    if gamma is not None:
        y = y / torch.sqrt(y.pow(2).sum(-1, keepdim=True) / y.shape[-1] + st["eps"]) * gamma.double()
    rot = st["case"]["rot"]
    table = st["cos_sin"].double()[st["positions"].long()]
    turn = torch.complex(table[:, : rot // 2], table[:, rot // 2 :])[:, None]
    pairs = y[..., :rot].unflatten(-1, (rot // 2, 2) if st["interleaved"] else (2, rot // 2))
    if not st["interleaved"]:
        pairs = pairs.transpose(-1, -2)
    turned = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
    if not st["interleaved"]:
        turned = turned.transpose(-1, -2)
    return torch.cat([turned.flatten(-2), y[..., rot:]], -1)


# ------------------------------------------------------------------------------------------ what a pass cannot do without


def work(case):
    op = case["op"]
    if op == "tree":
        q_lens = _spread(case["nodes_low"], case["nodes"], case["seqs"])
        ctx = _spread(case["ctx_low"], case["ctx"], case["seqs"])
        positions, tokens = int((q_lens + ctx).sum()), int(q_lens.sum())
        pairs = tokens * float(ctx.mean()) + tokens  # which context meets which tree is the seed's; the mean is not
        cache = positions * case["kv_heads"] * 2 * D * 2
        return {"bytes": cache + 2 * tokens * case["heads"] * D * 2 + tokens * 4 * -(-case["nodes"] // 32)
                + 4 * positions // case["page"], "flops": 4 * D * case["heads"] * pairs}
    if op in ("write", "norm"):
        T, heads = case["tokens"], case["heads"] + case["kv_heads"]
        moved = heads + (case["kv_heads"] if op == "write" else 0)
        return {"bytes": T * (2 * moved * D * 2 + 4 * case["rot"] + 4 * (2 if op == "write" else 1)),
                "flops": T * heads * (D * (4 if case["norm"] else 0) + 3 * case["rot"])}
    if op == "plan":
        tokens, S = int(_spread(case["new_low"], case["new"], case["seqs"]).sum()), case["seqs"]
        pages = tokens // case["page"] + S
        return {"bytes": 4 * (5 * S + 2 * tokens + (tokens if case["depths"] else 0) + 2 * pages),
                "flops": 8 * tokens}
    moved = int((_spread(1, case["path"], case["seqs"]) - 1).sum())
    return {"bytes": 2 * moved * case["kv_heads"] * 2 * D * 2 + 4 * case["seqs"] * (5 + case["path"]), "flops": 0}
