"""A step over drafted tokens, on the CPU: the oracle on cases small enough to write down, and what the operators refuse
before anything is launched."""

import numpy as np
import pytest
import torch

import oracle
from tilejax_b200 import ops


@pytest.fixture(scope="module", autouse=True)
def host_side(native):
    """The operators' compiled host side (built on demand, as the library is)."""
    from tilejax_b200.csrc.build import BINDING, build_binding

    if not BINDING.exists():
        build_binding()


def test_the_host_side_names_itself_when_it_is_missing(monkeypatch):
    import sys

    import tilejax_b200

    monkeypatch.setattr(ops, "_binding", None)
    monkeypatch.setitem(sys.modules, "tilejax_b200._binding", None)
    monkeypatch.delattr(tilejax_b200, "_binding", raising=False)
    with pytest.raises(RuntimeError, match="csrc.build"):
        ops.rpa_commit(None, None, None, None, None, None)


def test_what_is_no_tensor_is_a_type_error():
    with pytest.raises(TypeError, match="kv_lens must be a tensor"):
        ops.rpa_commit(heads(4, 16, 2, 2, 128), [9, 4], i32(0, 1), i32(0, 1), i32(0)[None], i32(1))
    with pytest.raises(TypeError):
        ops.rpa_plan(i32(1), i32(1), i32(0), i32(0), i32(1), "4", 1)


def i32(*values):
    return torch.tensor(values, dtype=torch.int32)


def test_the_plan_oracle_on_a_step_by_hand():
    # Pages of 4. Sequence 0: 3 cached positions, 2 new ones: one more page. Sequence 1: new, 5 tokens: two pages, of
    # which the stack holds none but one. Sequence 2: nothing new.
    table = [7, -1, -1, -1, -1, -1, 2, -1, -1]
    got = oracle.rpa_plan_ref([3, 0, 4], [2, 5, 0], table, [9, 5], [2], 4, 8)
    assert [g.tolist() for g in got] == [[5, 5, 4], [0, 2, 7, 7], [3, 4, 0, 1, 2, 3, 4, 0],
                                         [31, 20, 36, 37, 38, 39, -1, -1], [2, 1, 1], [0, 1],
                                         [7, 5, -1, 9, -1, -1, 2, -1, -1]]


def test_the_tree_oracle_is_causal_attention_on_a_path():
    rng = np.random.default_rng(0)
    q_lens, kv_lens = [5, 3], [12, 3]
    inp = oracle.rpa_inputs(q_lens, kv_lens, heads=4, kv_heads=2, page_size=16, max_len=32, dtype=np.float64)
    inp["distribution"][:] = [2, 2, 2]
    mask = np.concatenate([oracle.pack_tree_mask(np.tril(np.ones((n, n), bool))) for n in q_lens])
    names = ("kv_lens", "page_indices", "cu_q_lens")
    got, size = oracle.tree_attention_f64(inp["q"], inp["kv_cache"], *(inp[n] for n in names), mask, [2, 2, 2], 0.1)
    want = oracle.rpa_prefill_f64(inp["q"], inp["kv_cache"], *(inp[n] for n in names), np.array([0, 0, 2]), 0.1)
    np.testing.assert_allclose(got, want, rtol=0, atol=1e-12)
    assert (size >= np.abs(got) - 1e-12).all() and rng is not None


def test_the_commit_oracle_moves_rows_along_the_path():
    cache = np.arange(8, dtype=np.float64).reshape(2, 4, 1, 1, 1) * np.ones((1, 1, 1, 2, 1))
    lens, after = oracle.rpa_commit_ref(cache, [7], [1, 0], [0, 5], np.array([[0, 2, 4, 3]]), [4])
    # Positions 2.. of pages (1, 0): nodes are rows 6, 7, 0, 1, 2; kept are nodes 0, 2, 4 (3 does not ascend).
    assert lens.tolist() == [5]
    assert after[..., 0, 0, 0].reshape(-1).tolist() == [2, 1, 2, 3, 4, 5, 6, 0]


def heads(*shape):
    return torch.zeros(shape, dtype=torch.bfloat16)


def refused(fn, good, bad):
    with pytest.raises(ValueError, match="CUDA tensors"):  # everything else is in order
        fn(**good())
    for message, name, change in bad:
        args = good()
        args[name] = change(args[name])
        with pytest.raises(ValueError, match=message):
            fn(**args)


def test_plan_refusals():
    def good():
        return dict(ctx_lens=i32(3, 0), q_lens=i32(2, 5), page_indices=i32(0, -1, -1, -1), free_pages=i32(1, 2, 3),
                    n_free=i32(3), page_size=4, tokens=7, pages_held=i32(1, 0), depths=i32(*range(7)))

    refused(ops.rpa_plan, good, [
        ("ctx_lens must be an int32 vector", "ctx_lens", lambda t: t.long()),
        ("q_lens must be an int32 vector", "q_lens", lambda t: t[None]),
        (r"\(S,\)", "q_lens", lambda t: t[:1]),
        ("pages_per_seq", "page_indices", lambda t: t[:3]),
        ("number of free pages", "n_free", lambda t: t[:0]),
        ("pages_held is", "pages_held", lambda t: t[:1]),
        ("depths is", "depths", lambda t: t[:6]),
        ("page_size must be positive", "page_size", lambda t: 0),
        ("tokens not negative|depths is", "tokens", lambda t: -1),
    ])


def test_norm_rope_refusals():
    def good():
        return dict(q=heads(3, 4, 128), k=heads(3, 2, 128), q_gamma=heads(128), k_gamma=heads(128), positions=i32(0, 1, 2),
                    cos_sin=torch.zeros(8, 128))

    bad = [
        (r"q is \(T, H, D\)", "q", lambda t: t[0]),
        ("q must be bfloat16", "q", lambda t: t.float()),
        ("k must be bfloat16", "k", lambda t: t[:2]),
        ("strides multiples of 4", "q", lambda t: heads(3, 4, 130)[:, :, :128]),
        ("last dimension must be dense", "q", lambda t: heads(3, 128, 4).transpose(1, 2)),
        ("given together", "k_gamma", lambda t: None),
        ("gammas are", "q_gamma", lambda t: t[:64]),
        ("positions is", "positions", lambda t: t.long()),
        ("cos_sin is", "cos_sin", lambda t: t.double()),
        ("cos_sin is", "cos_sin", lambda t: t[:, :12]),
        ("cos_sin is", "cos_sin", lambda t: torch.zeros(8, 136)),
    ]
    refused(ops.qk_norm_rope, good, bad)

    def good_write():
        return dict(**good(), v=heads(3, 2, 128), kv_cache=heads(4, 16, 2, 2, 128), slots=i32(3, 4, 5))

    refused(ops.rpa_norm_rope_write, good_write, [b for b in bad if b[1] not in ("q", "k") or "strides" in b[0]] + [
        ("k and v", "v", lambda t: t[:, :1]),
        ("side by side", "kv_cache", lambda t: t.float()),
        ("the cache's Hkv and D", "kv_cache", lambda t: heads(4, 16, 4, 2, 128)),
        ("slots is", "slots", lambda t: t[:2]),
    ])


def test_norm_rope_refuses_outputs_among_what_it_looks_up():
    # Other warps may still read the gammas, positions, angles and slots while one writes.
    memory = torch.zeros(1 << 14, dtype=torch.bfloat16)
    ints, floats = memory.view(torch.int32), memory.view(torch.float32)

    def good():
        return dict(q=heads(3, 4, 128), k=heads(3, 2, 128), q_gamma=heads(128), k_gamma=heads(128), positions=i32(0, 1, 2),
                    cos_sin=torch.zeros(8, 128))

    def good_write():
        return dict(**good(), v=heads(3, 2, 128), kv_cache=heads(4, 16, 2, 2, 128), slots=i32(3, 4, 5))

    looked_up = dict(q_gamma=memory[:128], k_gamma=memory[128:256], positions=ints[100:103], cos_sin=floats[4:1028].view(8, 128),
                     slots=ints[200:203])
    q_out, k_out = memory[: 3 * 4 * 128].view(3, 4, 128), memory[: 3 * 2 * 128].view(3, 2, 128)
    for name, tensor in looked_up.items():
        if name != "slots":
            for out in ((q_out, heads(3, 2, 128)), (heads(3, 4, 128), k_out)):
                with pytest.raises(ValueError, match="overlaps"):
                    ops.qk_norm_rope(**{**good(), name: tensor}, out=out)
        with pytest.raises(ValueError, match="overlaps"):
            ops.rpa_norm_rope_write(**{**good_write(), name: tensor}, out=q_out)
        with pytest.raises(ValueError, match="overlaps"):
            ops.rpa_norm_rope_write(**{**good_write(), name: tensor, "kv_cache": memory[: 2 * 16 * 2 * 2 * 128].view(2, 16, 2, 2, 128)})
    # Side by side is fine: what is left to refuse is the CPU.
    with pytest.raises(ValueError, match="CUDA tensors"):
        ops.qk_norm_rope(**{**good(), "q_gamma": memory[3 * 4 * 128 : 3 * 4 * 128 + 128]}, out=(q_out, heads(3, 2, 128)))


def test_tree_attention_refusals():
    def good():
        return dict(q=heads(3, 4, 128), kv_cache=heads(4, 16, 2, 2, 128), kv_lens=i32(9, 4), page_indices=i32(0, 1, 2, 3),
                    cu_q_lens=i32(0, 2, 3), tree_mask=torch.zeros(3, 1, dtype=torch.int32), distribution=i32(2, 2, 2))

    refused(ops.rpa_tree_attention, good, [
        ("side by side", "kv_cache", lambda t: t[:, :, :, 0]),
        ("page_indices is", "page_indices", lambda t: t[:3]),
        ("must be int32", "kv_lens", lambda t: t.long()),
        (r"q is \(T, H, D\)", "q", lambda t: t.float()),
        (r"q is \(T, H, D\)", "q", lambda t: t[:, :, :64]),
        ("cu_q_lens is", "cu_q_lens", lambda t: t[:2]),
        ("cu_q_lens is", "distribution", lambda t: t.long()),
        ("tree_mask is", "tree_mask", lambda t: t[:2]),
        ("tree_mask is", "tree_mask", lambda t: t.bool()),
    ])


def test_commit_refusals():
    def good():
        return dict(kv_cache=heads(4, 16, 2, 2, 128), kv_lens=i32(9, 4), page_indices=i32(0, 1, 2, 3), cu_q_lens=i32(0, 2, 3),
                    paths=torch.zeros(2, 2, dtype=torch.int32), n_accepted=i32(1, 1))

    refused(ops.rpa_commit, good, [
        ("side by side", "kv_cache", lambda t: t[:, :, :, 0]),
        ("page_indices is", "page_indices", lambda t: t[:3]),
        ("cu_q_lens is", "cu_q_lens", lambda t: t[:2]),
        ("paths is", "paths", lambda t: t[:1]),
        ("paths is", "paths", lambda t: t.long()),
        ("n_accepted", "n_accepted", lambda t: t[:1]),
    ])


def test_commit_refuses_a_cache_among_its_tables():
    # Each sequence's block reads its own lengths, path and entries while others move rows.
    memory = torch.zeros(1 << 15, dtype=torch.bfloat16)
    ints = memory.view(torch.int32)
    good = dict(kv_cache=memory[: 2 * 16 * 2 * 2 * 128].view(2, 16, 2, 2, 128), kv_lens=i32(9, 4), page_indices=i32(0, 1, 2, 3),
                cu_q_lens=i32(0, 2, 3), paths=torch.zeros(2, 2, dtype=torch.int32), n_accepted=i32(1, 1))
    inside = dict(kv_lens=ints[:2], page_indices=ints[40:44], cu_q_lens=ints[8189:8192], paths=ints[10:14].view(2, 2),
                  n_accepted=ints[100:102])
    for name, tensor in inside.items():
        with pytest.raises(ValueError, match="the cache overlaps"):
            ops.rpa_commit(**{**good, name: tensor})
    with pytest.raises(ValueError, match="CUDA tensors"):  # behind it is fine
        ops.rpa_commit(**{**good, "paths": ints[8192:8196].view(2, 2)})
