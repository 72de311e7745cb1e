"""What the speculative serving operators refuse, and their C ABI's checks (CPU)."""

from __future__ import annotations

import ctypes
import threading
import types

import pytest
import torch

from local_kimi_b200 import _lib, kernels, ops, registry
from local_kimi_b200 import build as build_mod
from oracle import speculative as ref


@pytest.fixture(scope="module")
def library() -> ctypes.CDLL:
    build_mod.build()
    return _lib.lib()


@pytest.fixture()
def any_device(monkeypatch):
    # The checks behind the device check, on CPU tensors.
    monkeypatch.setattr(ops, "_require_cuda", lambda tensor, what: None)


def heads(tokens=4, h=2, d=64, dtype=torch.bfloat16):
    return torch.zeros((tokens, h, d), dtype=dtype)


def i32(*values):
    return torch.tensor(values, dtype=torch.int32)


def test_operators_are_registered():
    for op in ("paged_plan", "paged_append", "prompt_attention", "tree_attention",
               "verify_drafts"):
        assert registry.default_of(op) == kernels.VARIANT


def test_cpu_tensors_are_refused():
    x, cache = heads(), torch.zeros((2, 8, 2, 64), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="requires CUDA"):
        ops.prompt_attention(x, x, x, i32(0, 4), 4)
    with pytest.raises(ValueError, match="requires CUDA"):
        ops.tree_attention(x, cache, cache, i32(0, 1)[None], i32(3), i32(0, 4), 4)
    with pytest.raises(ValueError, match="requires CUDA"):
        ops.paged_append(x, x, cache, cache, torch.arange(4))
    with pytest.raises(ValueError, match="requires CUDA"):
        ops.paged_plan(i32(1), i32(1), i32(0, 1)[None], i32(0), i32(0), 8, 1)
    with pytest.raises(ValueError, match="requires CUDA"):
        ops.verify_drafts(torch.zeros(1, 4), torch.zeros(1, dtype=torch.long), i32(0, 1), 1,
                          torch.zeros(1), torch.ones(1, 4), torch.ones(1))


def test_prompt_attention_refusals(any_device):
    x = heads()
    with pytest.raises(TypeError, match="BF16 or FP16"):
        ops.prompt_attention(x.float(), x, x, i32(0, 4), 4)
    with pytest.raises(TypeError, match="one type"):
        ops.prompt_attention(x, x.half(), x, i32(0, 4), 4)
    with pytest.raises(ValueError, match="shape"):
        ops.prompt_attention(x[0], x, x, i32(0, 4), 4)
    with pytest.raises(ValueError, match="multiple of key/value heads"):
        ops.prompt_attention(heads(h=3), x, x, i32(0, 4), 4)
    with pytest.raises(ValueError, match="width of q"):
        ops.prompt_attention(x, heads(d=128), x, i32(0, 4), 4)
    with pytest.raises(ValueError, match="multiples of 8"):
        ops.prompt_attention(heads(d=60), heads(d=60), x, i32(0, 4), 4)
    with pytest.raises(ValueError, match="multiples of 8"):
        ops.prompt_attention(heads(d=256), heads(d=256), x, i32(0, 4), 4)
    with pytest.raises(ValueError, match="multiples of 8"):
        ops.prompt_attention(x, x, heads(d=136), i32(0, 4), 4)
    with pytest.raises(TypeError, match="cu_seqlens"):
        ops.prompt_attention(x, x, x, i32(0, 4).long(), 4)
    with pytest.raises(ValueError, match="cu_seqlens_k is needed"):
        ops.prompt_attention(x, heads(5), heads(5), i32(0, 4), 4)
    with pytest.raises(ValueError, match="2 entries"):
        ops.prompt_attention(x, x, x, i32(0, 4), 4, cu_seqlens_k=i32(0, 1, 4))
    with pytest.raises(ValueError, match="max_seqlen"):
        ops.prompt_attention(x, x, x, i32(0, 4), -1)


def test_tree_attention_refusals(any_device):
    x, cache = heads(), torch.zeros((2, 8, 2, 64), dtype=torch.bfloat16)
    table = i32(0, 1)[None]
    call = lambda **kw: ops.tree_attention(**{**dict(  # noqa: E731
        q=x, k_cache=cache, v_cache=cache, block_table=table, context_lens=i32(3),
        cu_tokens=i32(0, 4), max_tokens=4), **kw})
    with pytest.raises(TypeError, match="one type"):
        call(k_cache=cache.half())
    with pytest.raises(TypeError, match="block_table"):
        call(block_table=table.long())
    with pytest.raises(ValueError, match="width of q"):
        call(k_cache=torch.zeros((2, 8, 2, 128), dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="power of two"):
        odd = torch.zeros((2, 12, 2, 64), dtype=torch.bfloat16)
        call(k_cache=odd, v_cache=odd)
    with pytest.raises(ValueError, match="unit stride"):
        wide = torch.zeros((2, 8, 2, 128), dtype=torch.bfloat16)[..., ::2]
        call(k_cache=wide)
    with pytest.raises(ValueError, match="1 entries"):
        call(context_lens=i32(3, 4))
    with pytest.raises(ValueError, match="at most 64"):
        call(max_tokens=65, tree_mask=torch.zeros(4, dtype=torch.long))
    with pytest.raises(TypeError, match="tree_mask"):
        call(tree_mask=i32(0, 0, 0, 0))
    with pytest.raises(ValueError, match="4 entries"):
        call(tree_mask=torch.zeros(5, dtype=torch.long))


def test_append_and_plan_refusals(any_device):
    x, cache = heads(), torch.zeros((2, 8, 2, 64), dtype=torch.bfloat16)
    with pytest.raises(TypeError, match="one type"):
        ops.paged_append(x, x.half(), cache, cache, torch.arange(4))
    with pytest.raises(TypeError, match="slots"):
        ops.paged_append(x, x, cache, cache, i32(0, 1, 2, 3))
    with pytest.raises(ValueError, match="4 entries"):
        ops.paged_append(x, x, cache, cache, torch.arange(3))
    with pytest.raises(ValueError, match="heads and widths"):
        ops.paged_append(heads(h=1), heads(h=1), cache, cache, torch.arange(4))
    with pytest.raises(ValueError, match="same pages"):
        ops.paged_append(x, x, cache, cache[:1], torch.arange(4))
    args = dict(context_lens=i32(1), new_lens=i32(1), block_table=i32(0, 1)[None],
                free_pages=i32(0), free_head=i32(0), page_size=8, num_tokens=1)
    call = lambda **kw: ops.paged_plan(**{**args, **kw})  # noqa: E731
    with pytest.raises(TypeError, match="new_lens"):
        call(new_lens=torch.tensor([1]))
    with pytest.raises(ValueError, match="1 entries"):
        call(new_lens=i32(1, 2))
    with pytest.raises(ValueError, match="page_size"):
        call(page_size=0)
    with pytest.raises(ValueError, match="1 entries"):
        call(parents=i32(0, 1))
    with pytest.raises(ValueError, match="unit stride"):
        call(block_table=i32(0, 1, 2, 3).view(2, 2).t()[:1])
    with pytest.raises(ValueError, match="at least one request"):
        call(context_lens=i32(), new_lens=i32(), block_table=i32().view(0, 2))


def test_verify_refusals(any_device):
    args = dict(logits=torch.zeros(3, 10), tokens=torch.zeros(3, dtype=torch.long),
                cu_tokens=i32(0, 3), max_tokens=3, accept_u=torch.zeros(3),
                noise=torch.ones(1, 10), temperature=torch.ones(1))
    call = lambda **kw: ops.verify_drafts(**{**args, **kw})  # noqa: E731
    with pytest.raises(TypeError, match="logits"):
        call(logits=torch.zeros(3, 10, dtype=torch.double))
    with pytest.raises(TypeError, match="tokens"):
        call(tokens=i32(0, 0, 0))
    with pytest.raises(ValueError, match="from 1 to 64"):
        call(max_tokens=65)
    with pytest.raises(ValueError, match="from 1 to 64"):
        call(max_tokens=0)
    with pytest.raises(ValueError, match="noise"):
        call(noise=torch.ones(2, 10))
    with pytest.raises(ValueError, match="chains"):
        call(parents=i32(-1, 0, 0), draft_probs=torch.zeros(3, 10))
    with pytest.raises(ValueError, match="draft_probs"):
        call(draft_probs=torch.zeros(2, 10))
    with pytest.raises(ValueError, match="2 entries"):
        call(cu_tokens=i32(0, 1, 3))


def test_c_abi_checks_arguments_before_any_launch(library):
    s3 = (ctypes.c_int64 * 3)(512, 64, 64)
    # Widths, pages, alignment, limits and workspaces, in that order.
    assert library.kb_prompt_attention(None, 0, 0, None, 0, 0, None, 0, 0, 0, None, None, 1, 1, 1,
                                       1, 2, 2, 60, 64, 1.0, None, None, None) == 6
    assert library.kb_prompt_attention(None, 0, 0, None, 0, 0, None, 0, 0, 0, None, None, 1, 1, 1,
                                       1, 3, 2, 64, 64, 1.0, None, None, None) == 2
    assert library.kb_prompt_attention(None, 0, 0, None, 0, 0, None, 0, 0, 0, None, None, 1, 1, 1,
                                       1, 2, 2, 64, 64, 1.0, None, None, None) == 1
    assert library.kb_prompt_attention(None, 0, 0, None, 0, 0, None, 0, 0, 0, None, None, 0, 0, 0,
                                       0, 2, 2, 64, 64, 1.0, None, None, None) == 0
    assert library.kb_tree_attention(None, 0, 0, None, s3, None, s3, 0, 1, 12, None, 1, 1, None,
                                     None, None, 1, 1, 1, 2, 2, 64, 64, 1.0, None, None, None, 0,
                                     None) == 6
    assert library.kb_tree_attention(None, 0, 0, None, s3, None, s3, 0, 1, 16, None, 1, 1, None,
                                     None, None, 1, 1, 1, 2, 2, 64, 64, 1.0, None, None, None, 0,
                                     None) == 1
    assert library.kb_paged_append(16, 64, 64, 16, 64, 64, 1, 1, 64, 64, 24, s3, 16, s3, 1, 8,
                                   16, None) == 4
    assert library.kb_paged_plan(None, None, None, 20000, None, 1, 1, None, 0, None, 8, 1, None, None,
                                 None, None, None, None, None, None) == 6
    assert library.kb_verify_drafts(None, 10, 1, 10, 0, None, None, None, 1, 65, None, None, 10,
                                    None, None, 10, None, None, None, None, 0, None) == 6
    assert library.kb_verify_drafts(16, 10, 1, 10, 0, 16, None, 16, 1, 3, 16, 16, 10, 16, None,
                                    10, 16, 16, 16, 256, 8, None) == 5
    assert "workspace" in _lib.last_error()
    assert library.kb_verify_drafts_workspace_size(0, 0) == 0
    assert library.kb_verify_drafts_workspace_size(17, 100) == \
        library.kb_verify_drafts_workspace_size(32, 128)
    # A call that succeeds clears the message.
    assert library.kb_paged_append(None, 0, 0, None, 0, 0, 0, 1, 64, 64, None, None, None, None,
                                   0, 8, None, None) == 0
    assert _lib.last_error() == ""


def test_oracle_attention_agrees_with_a_dense_softmax():
    gen = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(9, 2, 16, generator=gen) for _ in range(3))
    out, lse, _ = ref.prompt_attention(q, k, v, [0, 9], [0, 9], 0.25)
    s = torch.einsum("thd,shd->hts", q.double(), k.double()) * 0.25
    s = s.masked_fill(torch.ones(9, 9, dtype=torch.bool).triu(1), float("-inf"))
    torch.testing.assert_close(out, torch.einsum("hts,shd->thd", s.softmax(-1), v.double()))
    torch.testing.assert_close(lse, s.logsumexp(-1).T)


def test_oracle_verification_known_answers():
    # Greedy: the argmax chain 1, 2 is accepted, then 3 follows.
    logits = torch.full((4, 5), -9.0)
    logits[0, 1] = logits[1, 2] = logits[2, 3] = logits[3, 4] = 9.0
    tokens = torch.tensor([0, 1, 2, 0])
    got = ref.verify(logits, tokens, [-1, 0, 1, 2], [0, 4], 4, torch.zeros(4), torch.ones(1, 5),
                     torch.zeros(1))
    assert got == ([[1, 2, 3, -1]], [[0, 1, 2, -1]], [2])
    # A refused child's mass leaves: with p = (1/2, 1/2) and child 0 refused,
    # child 1 has all of the rest.
    logits = torch.zeros(3, 2)
    got = ref.verify(logits, torch.tensor([0, 0, 1]), [-1, 0, 0], [0, 3], 3,
                     torch.tensor([0.0, 0.9, 0.99]), torch.ones(1, 2), torch.ones(1))
    assert got == ([[1, 0, -1]], [[0, 2, -1]], [1])


def test_scales_must_be_positive(any_device):
    x, cache = heads(), torch.zeros((2, 8, 2, 64), dtype=torch.bfloat16)
    for scale in (0.0, -1.0, float("nan")):
        with pytest.raises(ValueError, match="scale must be positive"):
            ops.prompt_attention(x, x, x, i32(0, 4), 4, scale=scale)
        with pytest.raises(ValueError, match="scale must be positive"):
            ops.tree_attention(x, cache, cache, i32(0, 1)[None], i32(3), i32(0, 4), 4,
                               scale=scale)


def test_prompts_with_tokens_need_a_longest_length(any_device):
    x = heads()
    with pytest.raises(ValueError, match="max_seqlen"):
        ops.prompt_attention(x, x, x, i32(0, 4), 0)


def test_rows_without_a_request_are_zero(any_device):
    x, cache = heads(), torch.zeros((2, 8, 2, 64), dtype=torch.bfloat16)
    none = torch.zeros(0, dtype=torch.int32)
    for out, lse in (
            ops.prompt_attention(x, x, x, i32(0), 4, return_lse=True),
            ops.tree_attention(x, cache, cache, torch.zeros((0, 2), dtype=torch.int32), none,
                               i32(0), 4, return_lse=True)):
        assert out.shape == (4, 2, 64) and not out.any()
        assert lse.shape == (4, 2) and (lse == -float("inf")).all()


@pytest.mark.parametrize("capturing", [False, True])
def test_verification_calls_in_flight_share_no_scratch(library, any_device, monkeypatch, capturing):
    # Another thread's call on the same stream may come before the first one is done, and
    # a graph may be replayed while another runs.
    seen = []

    def call(name, *args):
        seen.append((args[-3], args[-2]))
        if len(seen) == 1:
            other = threading.Thread(target=again)
            other.start()
            other.join()

    def again():
        return ops.verify_drafts(torch.zeros(3, 10), torch.zeros(3, dtype=torch.long), i32(0, 3),
                                 3, torch.zeros(3), torch.ones(1, 10), torch.ones(1))

    monkeypatch.setattr(ops, "_raw_stream", lambda device: 0)
    monkeypatch.setattr(ops, "_capturing", lambda: capturing, raising=False)
    monkeypatch.setattr(_lib, "call", call)
    again()
    (a, n), (b, m) = seen
    assert min(n, m) >= library.kb_verify_drafts_workspace_size(1, 3) > 0
    assert a + n <= b or b + m <= a


def test_graphs_have_scratch_of_their_own(monkeypatch):
    # Scratch made while a graph is captured is zeroed by that graph alone: no other graph
    # and no call outside may find it, nor a graph the scratch of calls outside.
    state = {"capture": 0}
    monkeypatch.setattr(ops, "_capturing", lambda: state["capture"] > 0, raising=False)
    monkeypatch.setattr(ops, "_capture_id", lambda stream: state["capture"], raising=False)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: state["capture"] > 0)
    monkeypatch.setattr(torch.cuda, "current_stream",
                        lambda device: types.SimpleNamespace(cuda_stream=7))
    cpu = torch.device("cpu", 0)
    for scratch in (lambda: ops._kept_scratch(("tree", 0, 7, 512), cpu, 7, 512, 64),
                    lambda: ops._workspace("router", cpu, 512, (3, 4))):
        found = {}
        for capture in (0, 1, 2, 0, 3):
            state["capture"] = capture
            ws = scratch()
            assert ws.numel() == 512 and not ws[:64].any()
            assert scratch() is ws                    # calls of one capture share it
            assert found.setdefault(capture, ws) is ws
            assert all(ws is not other for c, other in found.items() if c != capture)


def test_paged_reserve_refusals(any_device, library):
    args = dict(context_lens=i32(1), new_lens=i32(1), block_table=i32(0, 1)[None],
                reserved_lens=i32(1), page_size=8)
    call = lambda **kw: ops.paged_reserve(**{**args, **kw})  # noqa: E731
    with pytest.raises(TypeError, match="reserved_lens"):
        call(reserved_lens=torch.tensor([1]))
    with pytest.raises(ValueError, match="1 entries"):
        call(reserved_lens=i32(1, 2))
    with pytest.raises(ValueError, match="in place"):
        call(context_lens=i32(1, 2), new_lens=i32(1, 2), block_table=i32(0, 1, 2, 3).view(2, 2),
             reserved_lens=i32(1, 2, 3, 4)[::2])
    with pytest.raises(ValueError, match="page size"):
        call(page_size=0)
    assert library.kb_paged_reserve(None, None, 1, None, 1, 1, 8, None, None) == 1
    assert library.kb_paged_reserve(16, 16, 1, 16, 1, 2, 8, 16, None) == 2
    assert library.kb_paged_reserve(16, 16, 20000, 16, 1, 1, 8, 16, None) == 6
    # A call that succeeds clears the message.
    assert library.kb_paged_append(None, 0, 0, None, 0, 0, 0, 1, 64, 64, None, None, None, None,
                                   0, 8, None, None) == 0


def test_expanded_caches_are_refused(any_device, library):
    # Heads, places or pages that share memory: a token would write over another's rows.
    x, cache = heads(), torch.zeros((2, 8, 2, 64), dtype=torch.bfloat16)
    for wide in (cache[:, :, :1].expand(2, 8, 2, 64), cache[:, :1].expand(2, 8, 2, 64),
                 cache[:1].expand(2, 8, 2, 64)):
        for caches in ((wide, cache), (cache, wide)):
            with pytest.raises(ValueError, match="positive strides"):
                ops.paged_append(x, x, *caches, torch.arange(4))
            with pytest.raises(ValueError, match="positive strides"):
                ops.tree_attention(x, *caches, i32(0, 1)[None], i32(3), i32(0, 4), 4)
    # An extent of one has no use for its stride.
    one = torch.zeros((1, 8, 1, 64), dtype=torch.bfloat16).as_strided((1, 8, 1, 64), (0, 64, 0, 1))
    ops.paged_append(heads(0, 1), heads(0, 1), one, one, torch.arange(0))
    s3, bad = (ctypes.c_int64 * 3)(1024, 128, 64), (ctypes.c_int64 * 3)(1024, 64, 0)
    assert library.kb_paged_append(16, 128, 64, 16, 128, 64, 4, 2, 64, 64, 16, bad, 16, s3, 2, 8,
                                   16, None) == 2
    assert library.kb_paged_append(None, 0, 0, None, 0, 0, 0, 1, 64, 64, None, None, None, None,
                                   0, 8, None, None) == 0


def test_expanded_rows_are_copied():
    x = heads(4, 1).expand(4, 2, 64)
    assert ops._rows_of_heads(x, "k").stride() == (128, 64, 1)
    x = heads(1, 2).expand(4, 2, 64)
    assert ops._rows_of_heads(x, "q").stride() == (128, 64, 1)
    assert ops._rows_of_heads(x, "k", expanded=True) is x
    x = heads(4, 2)
    assert ops._rows_of_heads(x, "v") is x


def test_calls_go_to_the_tensors_device(library, any_device, monkeypatch):
    # A kernel is launched on the current device, so the call makes the tensors' current.
    state, seen = {"device": 0}, []

    class device:
        def __init__(self, to):
            self.to = to

        def __enter__(self):
            self.back, state["device"] = state["device"], self.to.index

        def __exit__(self, *_):
            state["device"] = self.back

    monkeypatch.setattr(ops, "_current_device", lambda: state["device"], raising=False)
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(_lib, "call", lambda name, *args: seen.append((name, state["device"])))
    ops._on(torch.device("cuda", 1))("kb_x", 1, 2)
    ops._on(torch.device("cuda", 0))("kb_y")
    assert seen == [("kb_x", 1), ("kb_y", 0)] and state["device"] == 0

    # Every operator says which device its tensors are on.
    monkeypatch.setattr(ops, "_on",
                        lambda device: lambda name, *args: seen.append((name, device)))
    monkeypatch.setattr(ops, "_raw_stream", lambda device: 0)
    monkeypatch.setattr(ops, "_capturing", lambda: False)
    seen.clear()
    x, cache = heads(), torch.zeros((2, 8, 2, 64), dtype=torch.bfloat16)
    table = i32(0, 1)[None]
    ops.paged_plan(i32(1), i32(1), table, i32(0), i32(0), 8, 1)
    ops.paged_reserve(i32(1), i32(1), table, i32(1), 8)
    ops.paged_append(x, x, cache, cache, torch.arange(4))
    ops.prompt_attention(x, x, x, i32(0, 4), 4)
    ops.tree_attention(x, cache, cache, table, i32(3), i32(0, 4), 4)
    ops.verify_drafts(torch.zeros(3, 10), torch.zeros(3, dtype=torch.long), i32(0, 3), 3,
                      torch.zeros(3), torch.ones(1, 10), torch.ones(1))
    assert seen == [(f"kb_{name}", torch.device("cpu")) for name in (
        "paged_plan", "paged_reserve", "paged_append", "prompt_attention", "tree_attention",
        "verify_drafts")]


def test_scratch_is_given_up_after_a_wait_ran_out(monkeypatch):
    # A call that ended early may leave counters that the next call would go on from.
    bits = {"now": 0}

    class fake:
        @staticmethod
        def kb_device_errors(stream, out):
            out._obj.value = bits["now"]
            return 0

    monkeypatch.setattr(_lib, "lib", lambda: fake)
    monkeypatch.setattr(ops, "_capturing", lambda: False)
    cpu = torch.device("cpu", 0)
    held = lambda: ops._kept_scratch(("wait", 0, 7, 256), cpu, 7, 256, 64)  # noqa: E731
    first = held()
    first.fill_(1)
    for word, kept in ((0, True), (4, True), (2, False)):
        bits["now"] = word
        assert _lib.device_errors() == word
        assert (held() is first) == kept
    assert not held().any()
