"""A step over drafted tokens on the GPU: tables, norm and rotation with the cache write, tree attention, commit, each
against plain NumPy in 64 bits, and a run of them together.

Tolerances. Rounding to bf16 is off by at most 2^-8 of the value. Norm and rotation round once; before that f32 holds
x, 1 / rms and the products to a few 2^-24 of what is added up (`size`): 2^-20 of it bounds them. Attention rounds the
output once and each weight once, the latter relative to the weighted mean of |v| (`size`): 2^-8 of each; the weights'
exponentials, the scores' f32 sums (128 products of |q k| up to about 60 before the scale, 1e-5 after it) and the joins
of partial sums stay below 2^-11 of it together."""

import numpy as np
import pytest
import torch
from helpers import BF16, f64, rand_bf16, to_device, to_host

import oracle
from tilejax_b200 import ops
from tilejax_b200._lib import NativeError

pytestmark = pytest.mark.gpu


def dev32(*values):
    return torch.tensor(np.asarray(values[0] if len(values) == 1 else values), dtype=torch.int32, device="cuda")


# ------------------------------------------------------------------------------------------ tables


PLANS = [  # (ctx, new, page_size, pages_per_seq, tokens - sum(new), pages short, held or None, depths)
    ([3], [1], 4, 2, 0, 0, None, False),
    ([3, 0, 4, 8], [2, 5, 0, 1], 4, 3, 3, 0, None, True),
    ([0, 0], [0, 0], 16, 1, 2, 0, None, False),                       # nothing to do, padding rows
    ([5, 40, 17], [30, 9, 100], 16, 8, 0, 4, None, False),            # the stack runs out on the way
    ([5, 40, 17], [30, 9, 100], 16, 8, 0, 99, None, False),           # an empty stack
    ([30, 60], [10, 10], 16, 4, 0, 0, None, False),                   # the second sequence passes its table's end
    ([16, 20], [3, 3], 16, 4, 1, 0, [3, 1], True),                    # pages held ahead, and fewer than used
    ([2, 3, 4], [4, 4, 4], 16, 2, -5, 0, None, False),                # fewer rows than new tokens
    (list(range(0, 1500, 7)), [1 + 13 * (i % 5) for i in range(215)], 16, 100, 7, 0, None, True),
    (list(range(2500)), [i % 3 for i in range(2500)], 48, 60, 0, 1, None, False),  # more than a round of the scan
]


@pytest.mark.parametrize("case", PLANS)
def test_plan_is_exact(case):
    ctx, new, page, pps, extra, short, held, with_depths = case
    rng = np.random.default_rng(len(ctx))
    S, T = len(ctx), sum(new) + extra
    have = [min(-(-c // page), pps) for c in ctx] if held is None else held
    order = rng.permutation(sum(have) + sum(-(-n // page) + 1 for n in new) + 5)
    table = np.full((S, pps), -1, np.int32)
    at = 0
    for s, n in enumerate(have):
        table[s, :n] = order[at : at + n]
        at += n
    need = sum(max(min(-(-(c + n) // page), pps) - h, 0) for c, n, h in zip(ctx, new, have))
    free = order[at:]
    n_free = [max(need - short, 0)] if short else [len(free)]
    depths = rng.integers(0, 6, T).astype(np.int32) if with_depths else None
    want = oracle.rpa_plan_ref(ctx, new, table.reshape(-1), free, n_free, page, T, held, depths)
    pages = dev32(table.reshape(-1))
    args = (dev32(ctx), dev32(new), pages, dev32(free), dev32(n_free), page, T)
    kw = dict(pages_held=None if held is None else dev32(held), depths=None if depths is None else dev32(depths))
    got = ops.rpa_plan(*args, **kw)
    for name, g, w in zip((*got._fields, "page_indices"), (*got, pages), want):
        np.testing.assert_array_equal(to_host(g), w, err_msg=name)
    # Again, into the same step: the table holds the pages already, the inputs say what was held.
    again = ops.rpa_plan(*args, **kw, out=got)
    for g, w in zip((*again, pages), want):
        np.testing.assert_array_equal(to_host(g), w)


def test_plan_refuses_an_output_among_its_inputs():
    ctx = dev32([3, 4])
    args = (ctx, dev32([1, 1]), dev32([0, -1, 1, -1]), dev32([2, 3]), dev32([2]), 4, 2)
    step = ops.rpa_plan(*args)
    with pytest.raises(ValueError, match="overlaps an input"):
        ops.rpa_plan(*args, out=step._replace(kv_lens=ctx))
    with pytest.raises(ValueError, match="other sizes"):
        ops.rpa_plan(*args, out=step._replace(slots=step.slots[:1]))
    S = 8193
    with pytest.raises(NativeError, match="more than 8192 sequences"):
        ops.rpa_plan(dev32([0] * S), dev32([1] * S), dev32([0] * S), dev32([0]), dev32([1]), 4, S)


def test_plan_refuses_a_table_among_its_other_inputs_and_outputs_in_one_place():
    both = dev32([0, -1, 1, -1, 2, 3])
    args = (dev32([3, 4]), dev32([1, 1]), both[:4], both[3:], dev32([2]), 4, 2)
    with pytest.raises(ValueError, match="page_indices overlaps"):
        ops.rpa_plan(*args)
    args = (*args[:3], both[4:], *args[4:])
    step = ops.rpa_plan(*args)
    with pytest.raises(ValueError, match="out's tensors overlap"):
        ops.rpa_plan(*args, out=step._replace(slots=step.positions))


def test_a_table_entry_past_the_last_slot_has_none():
    # 2^31 - 1 and 2^29 are no pages of a cache whose rows fit int32; their slots must not wrap round to some that are.
    step = ops.rpa_plan(dev32([3, 3, 3]), dev32([1, 1, 1]), dev32([2**31 - 1, 2**29, 2**29 - 1]), dev32([0]), dev32([0]), 4, 3)
    assert to_host(step.slots).tolist() == [-1, -1, 2**31 - 1]


# ------------------------------------------------------------------------------------------ norm, rotation, write


def angles(positions, rot):
    a = np.arange(positions)[:, None] * 10000.0 ** (-np.arange(rot // 2) * 2 / max(rot, 1))
    return np.concatenate([np.cos(a), np.sin(a)], 1).astype(np.float32)


def close(got, want, size, slack=2.0**-20):
    got = f64(got)
    assert np.isfinite(got).all()
    over = np.abs(got - want) - (2.0**-8 * np.abs(want) + slack * size)
    assert over.max(initial=-1.0) <= 1e-30, over.max()


@pytest.mark.parametrize(("T", "H", "Hkv", "D", "rot", "interleaved", "norm"), [
    (1, 32, 8, 128, 128, False, True),
    (7, 32, 8, 128, 128, True, True),
    (5, 3, 1, 128, 64, False, True),       # half of the head, an odd number of rows
    (3, 28, 4, 128, 96, True, False),
    (33, 5, 5, 64, 64, False, True),
    (9, 8, 2, 256, 128, False, True),
    (2, 1, 1, 256, 8, True, True),
    (700, 7, 3, 64, 32, True, False),
    (4, 4, 4, 128, 0, False, True),        # the norm alone
    (6, 5, 2, 128, 24, False, True),       # a rotated part that is not two halves of whole lanes
])
def test_norm_and_rotation(T, H, Hkv, D, rot, interleaved, norm):
    rng = np.random.default_rng(T)
    qkv = rand_bf16((T, H + 2 * Hkv, D), T, 3.0)
    gq, gk = (rand_bf16((D,), 5 + i) for i in range(2)) if norm else (None, None)
    table = angles(100, rot)
    positions = rng.integers(-5, 130, T).astype(np.int32)  # some past the table: clamped
    q, k, v = qkv[:, :H], qkv[:, H : H + Hkv], qkv[:, H + Hkv :]
    want_q, size_q = oracle.norm_rope_f64(q, gq, positions, table, 1e-5, interleaved)
    want_k, size_k = oracle.norm_rope_f64(k, gk, positions, table, 1e-5, interleaved)
    packed = to_device(qkv)
    dq, dk, dv = packed[:, :H], packed[:, H : H + Hkv], packed[:, H + Hkv :]  # views: strides of the packed rows
    gammas = [None if g is None else to_device(g) for g in (gq, gk)]
    args = (*gammas, to_device(positions), to_device(table))
    got = ops.qk_norm_rope(dq, dk, *args, eps=1e-5, interleaved=interleaved)
    close(to_host(got[0]), want_q, size_q)
    close(to_host(got[1]), want_k, size_k)
    # To the cache, some tokens without a slot: the same keys, the values as they are, and nothing else.
    page = 16
    pages = -(-2 * T // page) + 1
    cache = rand_bf16((pages, page, Hkv, 2, D), 9)
    slots = rng.permutation(pages * page)[:T].astype(np.int32)
    slots[::5] = -1
    slots[3::7] = pages * page
    dcache = to_device(cache)
    got_q, same = ops.rpa_norm_rope_write(dq, dk, dv, *args, dcache, to_device(slots), eps=1e-5, interleaved=interleaved)
    assert same is dcache and torch.equal(got_q, got[0])
    rows = cache.reshape(-1, Hkv, 2, D)
    for t in range(T):
        if 0 <= slots[t] < pages * page:
            rows[slots[t], :, 0], rows[slots[t], :, 1] = to_host(got[1][t]), v[t]
    np.testing.assert_array_equal(to_host(dcache).view(np.uint16), cache.view(np.uint16))
    np.testing.assert_array_equal(to_host(packed).view(np.uint16), qkv.view(np.uint16))  # the operands are left alone
    # In place, inside the packed rows.
    ops.qk_norm_rope(dq, dk, *args, eps=1e-5, interleaved=interleaved, out=(dq, dk))
    assert torch.equal(dq, got[0]) and torch.equal(dk, got[1])
    np.testing.assert_array_equal(to_host(dv).view(np.uint16), v.view(np.uint16))


@pytest.mark.parametrize("interleaved", [False, True])
def test_norm_and_rotation_of_rows_eight_bytes_apart_from_sixteen(interleaved):
    # Token and head strides that are multiples of 4 elements but not of 8, and a base in between.
    rng = np.random.default_rng(3)
    T, H, Hkv, D = 9, 6, 2, 128
    table, gammas = angles(64, 64), [rand_bf16((D,), i) for i in (1, 2)]
    positions = rng.integers(0, 64, T).astype(np.int32)
    wide = rand_bf16((T, H + Hkv, D + 12), 4)
    q, k = wide[:, :H, 4 : 4 + D], wide[:, H:, 4 : 4 + D]
    want = [oracle.norm_rope_f64(x, g, positions, table, 1e-6, interleaved) for x, g in zip((q, k), gammas)]
    dev = to_device(wide)
    got = ops.qk_norm_rope(dev[:, :H, 4 : 4 + D], dev[:, H:, 4 : 4 + D], *map(to_device, gammas), to_device(positions),
                           to_device(table), interleaved=interleaved)
    for g, (w, size) in zip(got, want):
        close(to_host(g), w, size)


def test_an_infinity_stays_where_it_is():
    # Without the norm an infinite element turns its pair and nothing else; elements past the rotated part stay as they are.
    for rot, interleaved in ((64, False), (64, True), (24, False)):
        x = rand_bf16((2, 1, 128), 5)
        x[0, 0, 100] = np.inf
        got = to_host(ops.qk_norm_rope(to_device(x), to_device(x), None, None, dev32([3, 4]), to_device(angles(8, rot)),
                                       interleaved=interleaved)[0])
        assert np.isinf(f64(got[0, 0, 100])) and np.isfinite(np.delete(f64(got[0, 0]), 100)).all()
        np.testing.assert_array_equal(got[..., rot:].view(np.uint16), x[..., rot:].view(np.uint16))


def test_norm_and_rotation_refuse_overlapping_outputs_and_unknown_heads():
    q, k = (torch.zeros(4, h, 128, dtype=torch.bfloat16, device="cuda") for h in (8, 2))
    args = (None, None, dev32([0] * 4), torch.zeros(4, 128, device="cuda"))
    with pytest.raises(ValueError, match="memory of its own"):
        ops.qk_norm_rope(q[:2], k[:2], None, None, dev32([0] * 2), args[3], out=(q[1:3], k[:2]))
    with pytest.raises(ValueError, match="memory of its own"):
        ops.qk_norm_rope(q, k, *args, out=(q, q[:, :2]))
    with pytest.raises(NativeError, match="64, 128 or 256"):
        ops.qk_norm_rope(q[:, :, :32].contiguous(), k[:, :, :32].contiguous(), None, None, args[2],
                         torch.zeros(4, 32, device="cuda"))
    with pytest.raises(NativeError, match="eps"):
        ops.qk_norm_rope(q, k, *args, eps=float("nan"))


def test_norm_and_rotation_into_views_of_one_tensor():
    # Outputs side by side within a token, and head by head, are apart; in place they are what separate ones are.
    rng = np.random.default_rng(3)
    T, D = 37, 64
    table, where = torch.from_numpy(angles(50, D)).cuda(), dev32(rng.integers(0, 50, T))
    gammas = [torch.from_numpy(rng.normal(1, 0.1, D)).to("cuda", torch.bfloat16) for _ in range(2)]
    packed = torch.from_numpy(rng.normal(size=(T, 14, D))).to("cuda", torch.bfloat16)
    for cut in (lambda x: (x[:, :9], x[:, 9:13]), lambda x: (x[:, ::2], x[:, 1::2])):
        q, k = cut(packed)
        want = ops.qk_norm_rope(q.contiguous(), k.contiguous(), *gammas, where, table)
        into = torch.full_like(packed, 7)
        got = ops.qk_norm_rope(q, k, *gammas, where, table, out=cut(into))
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and (into[:, 13:] == 7).all() == (q.shape[1] == 9)
        place = packed.clone()
        got = ops.qk_norm_rope(*cut(place), *gammas, where, table, out=cut(place))
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_norm_and_rotation_refuse_operands_that_share_elements():
    x = torch.zeros(4, 8, 128, dtype=torch.bfloat16, device="cuda")
    rest = (None, None, dev32([0] * 4), torch.zeros(4, 128, device="cuda"))
    one = x[:1].expand(4, 8, 128)
    for q, k, out in [(x, x, (x, x)), (x[:, :5], x[:, 4:], (x[:, :5], x[:, 4:])),  # in place, a head of both
                      (x, x[:, :2].clone(), (one, x[:, :2].clone())), (one, x[:, :2].clone(), (one, x[:, :2].clone())),
                      (x[:, :2], x[:, 2:4], (x[:, 4:6], x[:, 5:7])), (x[:, ::2], x[:, 1::2], (x[:, ::2], x[:, :4]))]:
        with pytest.raises(ValueError, match="memory of its own"):
            ops.qk_norm_rope(q, k, *rest, out=out)


# ------------------------------------------------------------------------------------------ tree attention


def tree(n, rng, empty=False):
    sees = np.zeros((n, n), bool)
    for i in range(n):
        if i:
            sees[i] = sees[rng.integers(0, i)]
        sees[i, i] = True
    if empty:
        sees[n // 2] = False
    return sees


def tree_case(q_lens, kv_lens, heads, kv_heads, page_size, *, words=None, max_seqs=None, extra=0, empty=False, seed=0,
              poison=True, scale=1.0):
    """Inputs of a step of trees; with `poison`, NaN and infinities wherever no row looks: rows behind a sequence's last
    position, pages of nobody."""
    rng = np.random.default_rng(seed)
    S = len(q_lens) if max_seqs is None else max_seqs
    T = sum(q_lens)
    used = [-(-n // page_size) for n in kv_lens]
    pps = max(1, *used) + 1
    pool = sum(used) + 2
    order = rng.permutation(pool)
    table = rng.integers(-3, pool + 3, (S, pps)).astype(np.int32)  # entries past a sequence's pages: anything
    cache = (rng.standard_normal((pool, page_size, kv_heads, 2, 128), np.float32)).astype(BF16)
    at = 0
    if poison:
        cache[order[sum(used):]] = np.nan
    for s, n in enumerate(used):
        table[s, :n] = order[at : at + n]
        at += n
        if poison and n:
            tail = kv_lens[s] - (n - 1) * page_size
            cache[table[s, n - 1], tail:] = np.array([np.nan, np.inf, -np.inf])[rng.integers(0, 3, cache[0, tail:].shape)].astype(BF16)
    cu = np.full(S + 1, T, np.int32)
    cu[: len(q_lens) + 1] = np.concatenate([[0], np.cumsum(q_lens)])
    lens = np.zeros(S, np.int32)
    lens[: len(kv_lens)] = kv_lens
    words = max(1, -(-max(q_lens) // 32)) if words is None else words
    masks = [oracle.pack_tree_mask(tree(n, rng, empty), words) for n in q_lens] + [np.zeros((extra, words), np.int32)]
    q = (scale * rng.standard_normal((T + extra, heads, 128), np.float32)).astype(BF16)
    return dict(q=q, kv_cache=cache, kv_lens=lens, page_indices=table.reshape(-1), cu_q_lens=cu,
                tree_mask=np.concatenate(masks), distribution=np.array([len(q_lens)] * 3, np.int32))


def check_tree(inp, sm_scale=128**-0.5, slack=2.0**-8 + 2.0**-11):
    dev = {k: to_device(v) for k, v in inp.items()}
    got = ops.rpa_tree_attention(**dev, sm_scale=sm_scale)
    assert ops.device_status() == 0
    want, size = oracle.tree_attention_f64(*inp.values(), sm_scale)
    close(to_host(got), want, size, slack)
    np.testing.assert_array_equal(to_host(dev["q"]).view(np.uint16), inp["q"].view(np.uint16))
    rest = int(inp["cu_q_lens"][inp["distribution"][0]])
    np.testing.assert_array_equal(to_host(got)[rest:].view(np.uint16), inp["q"][rest:].view(np.uint16))
    in_place = dev["q"].clone()
    same = ops.rpa_tree_attention(**{**dev, "q": in_place}, sm_scale=sm_scale, out=in_place)
    assert same is in_place and torch.equal(in_place.view(torch.int16), got.view(torch.int16))
    return got


TREES = {
    "one token": ([1], [1], 8, 2, 16),
    "one token, long": ([1], [1000], 8, 2, 16),
    "no prefix": ([9], [9], 4, 4, 32),
    "a block exactly": ([16], [128], 16, 2, 64),
    "a block and one": ([16], [129], 16, 2, 64),
    "a page inside": ([5, 3, 8], [63, 64, 65], 8, 2, 48),
    "ragged": ([8, 1, 17, 30], [700, 3, 17, 333], 32, 8, 16),
    "seven to a head": ([25, 3, 19], [200, 61, 129], 28, 4, 48),
    "three to a head": ([43, 44], [300, 90], 3, 1, 16),
    "five to a head": ([26], [77], 20, 4, 16),
    "one to a head": ([64, 2], [190, 66], 2, 2, 128),
    "two row tiles": ([32], [500], 8, 1, 32),
    "many rows": ([70, 33], [400, 100], 8, 1, 256),
    "wide group": ([3, 9], [260, 40], 128, 1, 16),
    "uneven group": ([2, 5], [70, 20], 100, 1, 16),
    "split": ([12], [9000], 8, 2, 16),
}


@pytest.mark.parametrize("name", TREES)
def test_tree_attention_matches_float64(name):
    check_tree(tree_case(*TREES[name], seed=len(name)))


@pytest.mark.parametrize(("kw", "case"), [
    (dict(empty=True), ([6, 5], [6, 70], 8, 2, 16)),           # a row that sees nothing (no prefix), one that sees only it
    (dict(max_seqs=7, extra=5), ([4, 9], [40, 9], 8, 2, 16)),  # a padded batch: empty sequences, rows behind the last
    (dict(words=1), ([40], [300], 4, 2, 16)),                  # nodes past the mask's words: seen by none
    (dict(words=5), ([3], [30], 4, 2, 16)),
    (dict(scale=30.0), ([8, 16], [500, 90], 8, 2, 16)),        # scores far apart: the running maximum moves often
])
def test_tree_attention_at_its_edges(kw, case):
    check_tree(tree_case(*case, **kw))


def tree_attention_on_the_gpu(inp, sm_scale):
    """oracle.tree_attention_f64 in torch's float64, for sizes NumPy takes long over (no hidden NaN)."""
    q, cache = inp["q"].double(), inp["kv_cache"]
    pages, page, hkv, _, D = cache.shape
    S = inp["kv_lens"].shape[0]
    table = inp["page_indices"].view(S, -1)
    cu, lens = inp["cu_q_lens"].tolist(), inp["kv_lens"].tolist()
    out, size = q.clone(), torch.zeros_like(q)
    for s in range(S):
        n, length = cu[s + 1] - cu[s], lens[s]
        kv = cache[table[s, : -(-length // page)].long()].reshape(-1, hkv, 2, D)[:length].double()
        bits = (inp["tree_mask"][cu[s] : cu[s + 1], :, None] >> torch.arange(32, device="cuda", dtype=torch.int32)) & 1
        sees = torch.cat([torch.ones(n, length - n, device="cuda", dtype=torch.bool), bits.reshape(n, -1)[:, :n].bool()], 1)
        rows = q[cu[s] : cu[s + 1]].view(n, hkv, -1, D)
        z = torch.einsum("nhgd,phd->nhgp", rows, kv[:, :, 0]) * sm_scale
        w = z.masked_fill(~sees[:, None, None], -float("inf")).softmax(-1)
        out[cu[s] : cu[s + 1]] = torch.einsum("nhgp,phd->nhgd", w, kv[:, :, 1]).reshape(n, -1, D)
        size[cu[s] : cu[s + 1]] = torch.einsum("nhgp,phd->nhgd", w, kv[:, :, 1].abs()).reshape(n, -1, D)
    return out.cpu().numpy(), size.cpu().numpy()


@pytest.mark.parametrize("seed", range(4))
@pytest.mark.parametrize(("heads", "kv_heads", "page", "seqs", "nodes", "ctx"), [
    (28, 4, 48, 13, 25, 2749),   # units of one and of two row tiles, many in one CTA's run, others over many CTAs
    (8, 2, 16, 40, 9, 600),      # small units: several in every run
    (16, 2, 128, 3, 64, 20000),  # every unit over many CTAs
])
def test_runs_of_many_units_and_units_of_many_runs(heads, kv_heads, page, seqs, nodes, ctx, seed):
    rng = np.random.default_rng(seed)
    q_lens = [int(n) for n in rng.integers(1, nodes + 1, seqs)]
    kv_lens = [n + int(c) for n, c in zip(q_lens, rng.integers(0, ctx, seqs))]
    dev = {k: to_device(v) for k, v in tree_case(q_lens, kv_lens, heads, kv_heads, page, seed=seed, scale=2.0, poison=False).items()}
    want, size = tree_attention_on_the_gpu(dev, 128**-0.5)
    first = ops.rpa_tree_attention(**dev, sm_scale=128**-0.5)
    close(to_host(first), want, size, 2.0**-8 + 2.0**-11)
    for _ in range(20):  # the same bits every time
        assert torch.equal(ops.rpa_tree_attention(**dev, sm_scale=128**-0.5).view(torch.int16), first.view(torch.int16))
    assert ops.device_status() == 0


@pytest.mark.parametrize("rising", [False, True])
def test_scores_hundreds_apart(rising):
    # Scores whose exponentials leave f32's range unless the running maximum follows. f32's error in a score is at most
    # 128 * 2^-24 of the sum of |q k| (about 128 * 200 * 0.64) times the scale: 0.011, the weights' relative error: 2^-5
    # is well above twice that and the roundings to bf16.
    inp = tree_case([9, 16, 40], [700, 90, 333], 8, 2, 16, scale=200.0, seed=7)
    if rising:  # later positions have larger keys
        for s, n in enumerate(inp["kv_lens"]):
            pages = inp["page_indices"].reshape(3, -1)[s, : -(-n // 16)]
            growth = np.linspace(0.01, 1.0, len(pages), dtype=np.float32)[:, None, None, None]
            inp["kv_cache"][pages, :, :, 0] = (inp["kv_cache"][pages, :, :, 0].astype(np.float32) * growth).astype(BF16)
    check_tree(inp, slack=2.0**-5)


def test_the_next_sequences_queries_do_not_change_a_bit():
    # They fill the rest of a row tile, and a raised maximum is raised for a whole warp. Large ones raise it in most blocks.
    inp = tree_case([9, 13, 3], [1500, 1500, 700], 16, 2, 16, poison=False)
    dev = {k: to_device(v) for k, v in inp.items()}
    want = ops.rpa_tree_attention(**dev, sm_scale=128**-0.5)
    for first in (9, 22):
        louder = dev["q"].clone()
        louder[first:] *= 32
        got = ops.rpa_tree_attention(**{**dev, "q": louder}, sm_scale=128**-0.5)
        assert torch.equal(got[:first], want[:first]) and not torch.equal(got[first:], want[first:])


def test_a_longer_tree_than_its_cache_and_lengths_past_the_table():
    inp = tree_case([6, 4], [20, 30], 8, 2, 16)
    inp["kv_lens"][0] = 4          # four positions for six nodes: the first two are in no cache row
    check_tree(inp)
    inp["kv_lens"][:] = [0, 30]    # an empty sequence that brings tokens: its rows are zero
    assert not check_tree(inp)[:6].any()
    # A length past the table: what the table holds is attended to.
    inp = tree_case([2], [60], 4, 2, 16, poison=False)
    inp["page_indices"][-1] = 0
    inp["kv_lens"][0] = 100
    check_tree(inp)


def test_nan_in_a_hidden_node_stays_there():
    # Node 2 of the tree holds NaN and infinity: rows that see it are NaN, those that do not are as without it.
    for nodes, group, ctx in ((6, 4, 50), (40, 8, 200), (40, 8, 24)):
        inp = tree_case([nodes], [ctx + nodes], group, 1, 16, seed=nodes)
        sees = np.zeros((nodes, nodes), bool)
        for i in range(nodes):
            sees[i, i] = True
            sees[i, i % 3] = True
        inp["tree_mask"][:] = oracle.pack_tree_mask(sees, inp["tree_mask"].shape[1])
        spot = ctx + 2
        row = inp["kv_cache"][inp["page_indices"][spot // 16], spot % 16]
        row[0, 1, :64], row[0, 1, 64:] = np.nan, np.inf
        dev = {k: to_device(v) for k, v in inp.items()}
        got = f64(to_host(ops.rpa_tree_attention(**dev, sm_scale=128**-0.5)))
        with np.errstate(invalid="ignore"):
            want, size = oracle.tree_attention_f64(*inp.values(), 128**-0.5)
        blind = ~sees[:, 2]
        close(got[blind], want[blind], size[blind], 2.0**-8 + 2.0**-11)
        assert np.isnan(got[~blind][..., :64]).all() and np.isposinf(got[~blind][..., 64:]).all()


def check_tree_not_finite(inp, sm_scale=128**-0.5):
    """As check_tree, where some elements are NaN by the formula: the same ones, and the others as close as ever."""
    got = f64(to_host(ops.rpa_tree_attention(**{k: to_device(v) for k, v in inp.items()}, sm_scale=sm_scale)))
    with np.errstate(invalid="ignore"):
        want, size = oracle.tree_attention_f64(*inp.values(), sm_scale)
    np.testing.assert_array_equal(np.isnan(got), np.isnan(want))
    fine = ~np.isnan(want)
    close(got[fine], want[fine], size[fine], 2.0**-8 + 2.0**-11)
    return want


SCORE_CASES = {  # (nodes, ctx, heads): every head has KV head 0, pages of 16
    "one masked block": (5, 20, 4),
    "whole blocks before": (6, 300, 4),
    "two row tiles": (40, 330, 8),
    "split": (4, 9000, 4),
}


@pytest.mark.parametrize("kind", ["all minus", "all minus but one", "all minus at first", "plus", "nan", "one key minus", "hidden"])
@pytest.mark.parametrize("name", SCORE_CASES)
def test_scores_that_are_not_finite(name, kind):
    # An infinite query element meets keys of one sign: a row whose scores are all minus infinity is NaN (0 / 0), not a mean
    # of some values; one that sees a single finite score is that position's value.
    nodes, ctx, heads = SCORE_CASES[name]
    inp = tree_case([nodes], [ctx + nodes], heads, 1, 16, seed=ctx)
    table = inp["page_indices"]
    keys = [inp["kv_cache"][table[p // 16], p % 16, 0, 0] for p in range(ctx + nodes)]  # views, (128,) each
    q, node = inp["q"], min(2, nodes - 1)
    if kind.startswith("all minus"):
        q[node, :2, 7] = np.inf
        for k in keys:
            k[7] = -abs(k[7].astype(np.float32)) - 1
        if kind.endswith("one"):
            keys[ctx // 2][7] = 0          # 0 * inf: NaN
            q[node, 1] = -np.inf           # and a row whose every element is infinite
        if kind.endswith("first"):         # finite scores from the middle on
            q[..., 7], q[node, :2, 7] = -1.0, -3e38
            for k in keys[: ctx // 2]:
                k[:] = 0
                k[7] = np.inf
            for k in keys[ctx // 2 :]:
                k[7] = 0
    elif kind == "plus":
        keys[ctx // 2][5], q[node, 1, 5] = np.inf, 1.0
        q[node, 2, 5] = -1.0
    elif kind == "nan":
        q[node, 3, 9] = np.nan
    elif kind == "one key minus":          # a position of weight zero for every row
        keys[ctx - 3][5], q[:, :, 5] = -np.inf, 1.0
    else:                                  # a hidden node's key: rows that do not see it are as without it
        keys[ctx + 1][:] = np.nan
    want = check_tree_not_finite(inp)
    assert np.isnan(want).any() == (kind not in ("all minus at first", "one key minus"))
    assert np.isfinite(want).any()


@pytest.mark.parametrize("sm_scale", [1e4, 1e10, 1e30])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("name", SCORE_CASES)
def test_scores_near_the_ends_of_the_range(name, sign, sm_scale):
    # One channel makes the scores, so f32 has them exactly, and they are whole: two of them are the same or so far apart that
    # the smaller has no weight. The row is the mean of V over its largest scores, whatever their size.
    nodes, ctx, heads = SCORE_CASES[name]
    inp = tree_case([nodes], [ctx + nodes], heads, 1, 16, seed=ctx)
    rng = np.random.default_rng(ctx)
    inp["q"][:] = 0
    inp["q"][..., 3] = sign
    for p in range(ctx + nodes):
        inp["kv_cache"][inp["page_indices"][p // 16], p % 16, 0, 0, 3] = 1 + rng.integers(0, 200)
    check_tree(inp, sm_scale)


@pytest.mark.parametrize("where", ["end", "middle", "first", "all"])
@pytest.mark.parametrize("name", ["ragged", "a page inside", "two row tiles", "many rows", "split", "one token, long"])
def test_positions_without_a_page_are_seen_by_none(name, where):
    # Entries that are no page of the pool, as rpa_plan leaves them where the stack ran out: neither a stand-in page nor NaN
    # in one reaches the result, and a row that sees nothing else is zero.
    q_lens, kv_lens, heads, kv_heads, page = TREES[name]
    inp = tree_case(q_lens, kv_lens, heads, kv_heads, page, seed=5)
    pool = len(inp["kv_cache"])
    table = inp["page_indices"].reshape(len(q_lens), -1)
    for s, n in enumerate(kv_lens):
        used = -(-n // page)
        gone = {"end": range(used - (used + 2) // 3, used), "middle": range(used // 3, used // 2 + 1), "first": [0],
                "all": range(used)}[where]
        for i, entry in enumerate(gone):
            table[s, entry] = [-1, pool, 2**31 - 1, -(2**31)][i % 4]
    for stand_in in (0, pool - 1):
        if stand_in not in table:
            inp["kv_cache"][stand_in] = np.nan
    got = check_tree(inp)
    assert where != "all" or not got.any()


def test_tree_attention_refuses_what_it_cannot_do():
    dev = {k: to_device(v) for k, v in tree_case([4], [40], 8, 2, 16).items()}
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        with pytest.raises(NativeError, match="sm_scale"):
            ops.rpa_tree_attention(**dev, sm_scale=scale)
    with pytest.raises(NativeError, match="multiple of the KV heads"):
        ops.rpa_tree_attention(**{**dev, "q": torch.zeros(4, 7, 128, dtype=torch.bfloat16, device="cuda")})
    with pytest.raises(NativeError, match="multiple of 16"):
        ops.rpa_tree_attention(**{**dev, "kv_cache": torch.zeros(4, 24, 2, 2, 128, dtype=torch.bfloat16, device="cuda")})
    with pytest.raises(NativeError, match="at most 128"):
        ops.rpa_tree_attention(**{**dev, "q": torch.zeros(4, 258, 128, dtype=torch.bfloat16, device="cuda")})
    with pytest.raises(ValueError, match="memory of its own"):
        wide = torch.zeros(6, 8, 128, dtype=torch.bfloat16, device="cuda")
        ops.rpa_tree_attention(**{**dev, "q": wide[:4]}, out=wide[2:])
    with pytest.raises(ValueError, match="overlaps an input"):
        ops.rpa_tree_attention(**dev, out=dev["kv_cache"].view(-1)[: 4 * 8 * 128].view(4, 8, 128))


def test_a_captured_step_follows_its_inputs():
    # Captured once, replayed with other lengths, tables, masks and data in the same tensors; an eager call in between.
    def case(seed, q_lens, kv_lens):
        return tree_case(q_lens, kv_lens, 8, 2, 16, seed=seed, max_seqs=3, extra=40 - sum(q_lens), words=1, poison=False)

    cases = [case(1, [20, 9, 3], [300, 1500, 77]), case(2, [4, 30], [4000, 31]), case(3, [1, 1, 1], [5, 1, 900])]
    pool = max(len(c["kv_cache"]) for c in cases)
    pps = max(len(c["page_indices"]) // 3 for c in cases)
    for c in cases:
        cache = np.zeros((pool, *c["kv_cache"].shape[1:]), BF16)
        cache[: len(c["kv_cache"])] = c["kv_cache"]
        table = np.zeros((3, pps), np.int32)
        old = c["page_indices"].reshape(3, -1)
        table[:, : old.shape[1]] = old
        c["kv_cache"], c["page_indices"] = cache, table.reshape(-1)
    dev = {k: to_device(v) for k, v in cases[0].items()}
    ops.rpa_tree_attention(**dev, sm_scale=0.1)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.rpa_tree_attention(**dev, sm_scale=0.1)
    for c in (*cases, cases[0]):
        for k, v in c.items():
            dev[k].copy_(to_device(v))
        graph.replay()
        eager = ops.rpa_tree_attention(**dev, sm_scale=0.1)
        assert torch.equal(out.view(torch.int16), eager.view(torch.int16))
        want, size = oracle.tree_attention_f64(*c.values(), 0.1)
        close(to_host(out), want, size, 2.0**-8 + 2.0**-11)
    assert ops.device_status() == 0


def test_calls_on_two_streams_at_once():
    cases = [{k: to_device(v) for k, v in tree_case([12, 30, 5], [3000, 900, 2000], 8, 2, 16, seed=s).items()} for s in (1, 2)]
    alone = [ops.rpa_tree_attention(**c, sm_scale=0.1) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[], []]
    for _ in range(20):
        for i, (c, s) in enumerate(zip(cases, streams)):
            with torch.cuda.stream(s):
                got[i].append(ops.rpa_tree_attention(**c, sm_scale=0.1))
    torch.cuda.synchronize()
    assert all(torch.equal(g.view(torch.int16), a.view(torch.int16)) for gs, a in zip(got, alone) for g in gs)


def test_rows_behind_two_to_the_32_bytes():
    # A cache of more than 2^31 elements, the sequences' pages at its end: write, attention and commit reach them.
    page, kv_heads = 16, 8
    pages = (1 << 31) // (page * kv_heads * 2 * 128) + 64
    cache = torch.empty((pages, page, kv_heads, 2, 128), dtype=torch.bfloat16, device="cuda")
    small = tree_case([9, 4], [150, 40], 16, kv_heads, page, seed=3, poison=False)
    shift = pages - len(small["kv_cache"])
    cache[shift:].copy_(to_device(small["kv_cache"]))
    dev = {k: to_device(v) for k, v in small.items() if k != "kv_cache"}
    low = {**dev, "kv_cache": to_device(small["kv_cache"])}
    want = ops.rpa_tree_attention(**low, sm_scale=0.1)
    dev["page_indices"] = dev["page_indices"] + shift
    assert torch.equal(ops.rpa_tree_attention(**dev, kv_cache=cache, sm_scale=0.1).view(torch.int16), want.view(torch.int16))
    paths, accepted = dev32([[0, 3, 5], [1, 2, 0]]), dev32([3, 2])
    names = ("kv_lens", "page_indices", "cu_q_lens")
    for c, d in ((cache, dev), (low["kv_cache"], low)):
        ops.rpa_commit(c, *(d[n] for n in names), paths, accepted)
    assert torch.equal(cache[shift:].view(torch.int16), low["kv_cache"].view(torch.int16))
    k = to_device(rand_bf16((2, kv_heads, 128), 1))
    slots = dev32([pages * page - 1, pages * page - 40])
    ops.rpa_norm_rope_write(to_device(rand_bf16((2, 16, 128), 2)), k, k, None, None, dev32([0, 0]),
                            torch.cat([torch.ones(1, 4), torch.zeros(1, 4)], 1).cuda(), cache, slots)
    rows = cache.view(-1, kv_heads, 2, 128)
    assert all(torch.equal(rows[int(s), :, i], k[t]) for t, s in enumerate(slots) for i in (0, 1))


# ------------------------------------------------------------------------------------------ commit


@pytest.mark.parametrize(("kv_heads", "page"), [(3, 16), (1, 48), (12, 32)])
def test_commit_is_exact(kv_heads, page):
    rng = np.random.default_rng(4)
    for seed, (q_lens, kv_lens) in enumerate([([5], [5]), ([1, 16, 64, 9, 4, 40, 70], [30, 100, 64, 10, 4, 300, 200])]):
        inp = tree_case(q_lens, kv_lens, kv_heads, kv_heads, page, seed=seed, poison=False)
        P = 40
        paths = np.stack([np.sort(rng.permutation(80)[:P]) for _ in q_lens]).astype(np.int32)
        for s, n in enumerate(q_lens):
            take = min(n, P)
            paths[s, :take] = np.sort(rng.permutation(n)[:take])
        accepted = np.array([min(n, P) for n in q_lens], np.int32)
        if len(q_lens) > 1:
            accepted[3], accepted[4] = -1, 0
            accepted[5] = 99            # more than the path holds
            paths[1, 4] = paths[1, 3]   # does not ascend: the path ends there
        names = ("kv_cache", "kv_lens", "page_indices", "cu_q_lens")
        want_lens, want = oracle.rpa_commit_ref(*(inp[n] for n in names), paths, accepted)
        dev = [to_device(inp[n]) for n in names]
        out = torch.empty(len(q_lens), dtype=torch.int32, device="cuda")
        lens = ops.rpa_commit(*dev, to_device(paths), to_device(accepted), out=out)
        assert lens is out
        np.testing.assert_array_equal(to_host(lens), want_lens)
        np.testing.assert_array_equal(to_host(dev[0]).view(np.uint16), want.view(np.uint16))
        with pytest.raises(ValueError, match="overlaps an input"):
            ops.rpa_commit(*dev, to_device(paths), to_device(accepted), out=dev[1])


# ------------------------------------------------------------------------------------------ together


def test_two_steps_of_drafted_tokens_with_a_prompt_beside_them():
    # Plan, norm + rotation + write, tree attention, prefill of the one prompt, commit; then a step on what was kept. The
    # cache the second step sees is checked against the tokens that were kept, its attention against float64.
    rng = np.random.default_rng(11)
    H, Hkv, page, pps, scale = 8, 2, 128, 4, 128**-0.5
    table = angles(600, 128)
    ctx, nodes, prompt = [100, 250], [7, 12], 60
    total = 16
    pages = dev32(np.full(3 * pps, -1))
    cache = torch.zeros(total, page, Hkv, 2, 128, dtype=torch.bfloat16, device="cuda")
    free, n_free = dev32(rng.permutation(total)), dev32([total])
    gq, gk = (to_device(rand_bf16((128,), i)) for i in (1, 2))
    cos_sin = to_device(table)

    def step(ctx_lens, new, depths, n_free, held, seed):
        T = sum(new)
        qkv = to_device(rand_bf16((T, H + 2 * Hkv, 128), seed))
        plan = ops.rpa_plan(ctx_lens, dev32(new), pages, free, n_free, page, T, pages_held=held,
                            depths=None if depths is None else dev32(depths))
        q, _ = ops.rpa_norm_rope_write(qkv[:, :H], qkv[:, H : H + Hkv], qkv[:, H + Hkv :], gq, gk, plan.positions,
                                       cos_sin, cache, plan.slots)
        return plan, q

    # The prefixes themselves, by the same operators: chunks of a prompt are paths.
    plan, _ = step(dev32([0, 0, 0]), [*ctx, 0], None, n_free, dev32([0, 0, 0]), 1)
    sees = [tree(n, rng) for n in nodes]
    depths = np.concatenate([s.sum(1) - 1 for s in sees] + [np.arange(prompt)])
    first, q = step(plan.kv_lens, [*nodes, prompt], depths, plan.n_free, plan.pages_held, 2)
    np.testing.assert_array_equal(to_host(first.positions)[: nodes[0]], ctx[0] + sees[0].sum(1) - 1)
    mask = to_device(np.concatenate([oracle.pack_tree_mask(s) for s in sees] + [np.zeros((prompt, 1), np.int32)]))
    dist = dev32([2, 2, 3])
    out = ops.rpa_tree_attention(q, cache, first.kv_lens, pages, first.cu_q_lens, mask, dist, scale)
    out = ops.rpa_prefill(out, cache, first.kv_lens, pages, first.cu_q_lens, dist, scale, out=out)
    assert ops.device_status() == 0
    host = [to_host(x) for x in (q, cache, first.kv_lens, pages, first.cu_q_lens)]
    want, size = oracle.tree_attention_f64(*host, to_host(mask), [2, 2, 3], scale)
    trees = sum(nodes)
    close(to_host(out)[:trees], want[:trees], size[:trees], 2.0**-8 + 2.0**-11)
    want = oracle.rpa_prefill_f64(*host, np.array([2, 2, 3]), scale)
    assert np.abs(f64(to_host(out))[trees:] - want[trees:]).max() <= 2e-2

    # Keep the longest path of each tree; the prompt keeps all its tokens.
    paths, accepted = np.zeros((3, 12), np.int32), np.array([0, 0, -1], np.int32)
    for s in range(2):
        deepest = np.flatnonzero(sees[s][int(sees[s].sum(1).argmax())])
        paths[s, : len(deepest)], accepted[s] = deepest, len(deepest)
    before = to_host(cache)
    lens = ops.rpa_commit(cache, first.kv_lens, pages, first.cu_q_lens, to_device(paths), to_device(accepted))
    want_lens, want_cache = oracle.rpa_commit_ref(before, *host[2:], paths, accepted)
    np.testing.assert_array_equal(to_host(lens), want_lens)
    np.testing.assert_array_equal(to_host(cache).view(np.uint16), want_cache.view(np.uint16))
    second, q = step(lens, [3, 3, 1], [0, 1, 1, 0, 1, 2, 0], first.n_free, first.pages_held, 3)
    mask = to_device(np.concatenate([oracle.pack_tree_mask(tree(n, rng)) for n in (3, 3, 1)]))
    out = ops.rpa_tree_attention(q, cache, second.kv_lens, pages, second.cu_q_lens, mask, dev32([3, 3, 3]), scale)
    host = [to_host(x) for x in (q, cache, second.kv_lens, pages, second.cu_q_lens, mask)]
    want, size = oracle.tree_attention_f64(*host, [3, 3, 3], scale)
    close(to_host(out), want, size, 2.0**-8 + 2.0**-11)
    assert to_host(second.n_free)[1] == 0


def test_a_captured_step_of_all_four_follows_its_inputs():
    # Plan, norm and write, attention and commit in one graph, replayed with other lengths, stacks, tables, masks, paths and data
    # copied into the same tensors. In the last one the stack runs out: the sequence that lacks pages sees what it has. Each
    # replay is checked against the oracles, from the cache as it was.
    S, H, Hkv, page, pps, T, P, scale = 3, 8, 2, 16, 12, 40, 6, 128**-0.5
    pool = 30
    table = angles(300, 128)
    gammas = [rand_bf16((128,), i) for i in (1, 2)]

    def case(seed, ctx, new, n_free):
        rng = np.random.default_rng(seed)
        held = [-(-c // page) for c in ctx]
        order = rng.permutation(pool)
        pages = np.full((S, pps), -1, np.int32)
        at = 0
        for s, n in enumerate(held):
            pages[s, :n] = order[at : at + n]
            at += n
        sees = [tree(n, rng) for n in new]
        mask, depths = np.zeros((T, 1), np.int32), np.zeros(T, np.int32)
        mask[: sum(new)] = np.concatenate([oracle.pack_tree_mask(s) for s in sees])
        depths[: sum(new)] = np.concatenate([s.sum(1) - 1 for s in sees])
        paths, accepted = np.zeros((S, P), np.int32), np.zeros(S, np.int32)
        for s, x in enumerate(sees):
            deepest = np.flatnonzero(x[int(x.sum(1).argmax())])[:P]
            paths[s, : len(deepest)], accepted[s] = deepest, len(deepest)
        free = np.zeros(pool, np.int32)
        free[: pool - at] = order[at:]
        return dict(ctx=np.array(ctx, np.int32), new=np.array(new, np.int32), pages=pages.reshape(-1), free=free,
                    n_free=np.array([pool - at if n_free is None else n_free], np.int32), held=np.array(held, np.int32), depths=depths,
                    mask=mask, paths=paths, accepted=accepted, qkv=rand_bf16((T, H + 2 * Hkv, 128), seed),
                    cache=rand_bf16((pool, page, Hkv, 2, 128), seed + 50))

    cases = [case(1, [100, 31, 0], [12, 9, 17], None), case(2, [1, 150, 16], [1, 30, 4], None), case(3, [40, 90, 70], [8, 20, 12], 1)]
    dev = {k: to_device(v) for k, v in cases[0].items()}
    dist, cos_sin = dev32([S, S, S]), to_device(table)
    dgammas = [to_device(g) for g in gammas]

    def step():
        d = dev
        plan = ops.rpa_plan(d["ctx"], d["new"], d["pages"], d["free"], d["n_free"], page, T, pages_held=d["held"], depths=d["depths"])
        q, k, v = d["qkv"][:, :H], d["qkv"][:, H : H + Hkv], d["qkv"][:, H + Hkv :]
        turned, _ = ops.rpa_norm_rope_write(q, k, v, *dgammas, plan.positions, cos_sin, d["cache"], plan.slots)
        apart = ops.qk_norm_rope(q, k, *dgammas, plan.positions, cos_sin)
        out = ops.rpa_tree_attention(turned, d["cache"], plan.kv_lens, d["pages"], plan.cu_q_lens, d["mask"], dist, scale)
        lens = ops.rpa_commit(d["cache"], plan.kv_lens, d["pages"], plan.cu_q_lens, d["paths"], d["accepted"])
        return plan, turned, apart, out, lens

    def load(c):
        for k, v in c.items():
            dev[k].copy_(to_device(v))

    step()
    load(cases[0])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan, turned, apart, out, lens = step()
    for c in (*cases, cases[1]):
        load(c)
        graph.replay()
        want = oracle.rpa_plan_ref(c["ctx"], c["new"], c["pages"], c["free"], c["n_free"], page, T, c["held"], c["depths"])
        for g, w in zip((*plan, dev["pages"]), want):
            np.testing.assert_array_equal(to_host(g), w)
        kv_lens, cu, positions, slots, _, left, pages = want
        assert (left[1] > 0) == (c is cases[2])
        q, size = oracle.norm_rope_f64(c["qkv"][:, :H], gammas[0], positions, table, 1e-6, False)
        close(to_host(turned), q, size)
        assert torch.equal(apart[0], turned)
        k, size = oracle.norm_rope_f64(c["qkv"][:, H : H + Hkv], gammas[1], positions, table, 1e-6, False)
        close(to_host(apart[1]), k, size)
        cache = c["cache"].copy()
        rows = cache.reshape(-1, Hkv, 2, 128)
        for t in np.flatnonzero(slots >= 0):
            rows[slots[t], :, 0], rows[slots[t], :, 1] = to_host(apart[1])[t], c["qkv"][t, H + Hkv :]
        want_out, size = oracle.tree_attention_f64(to_host(turned), cache, kv_lens, pages, cu, c["mask"], [S] * 3, scale)
        close(to_host(out), want_out, size, 2.0**-8 + 2.0**-11)
        want_lens, cache = oracle.rpa_commit_ref(cache, kv_lens, pages, cu, c["paths"], c["accepted"])
        np.testing.assert_array_equal(to_host(lens), want_lens)
        np.testing.assert_array_equal(to_host(dev["cache"]).view(np.uint16), cache.view(np.uint16))
    assert ops.device_status() == 0
