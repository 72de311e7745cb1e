"""What the operators of requests that share a prompt refuse, and their C ABI's checks (CPU)."""

from __future__ import annotations

import contextlib
import ctypes

import pytest
import torch

from local_kimi_b200 import _lib, kernels, ops, registry
from local_kimi_b200 import build as build_mod
from oracle import sharing as ref


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


def i64(*values):
    return torch.tensor(values, dtype=torch.long)


def test_operators_are_registered():
    for op in ("linear_attention", "linear_attention_step", "paged_fork", "paged_free",
               "paged_compact", "paged_copy", "adjust_logits"):
        assert registry.default_of(op) == kernels.VARIANT


def test_cpu_tensors_are_refused():
    x, g, s = heads(), torch.zeros(2), torch.zeros(4, 2, 64, 64)
    table, cache = i32(0, 1)[None], torch.zeros((2, 8, 2, 64), dtype=torch.bfloat16)
    calls = [
        lambda: ops.linear_attention(x, x, x, g, i32(0, 4), 4),
        lambda: ops.linear_attention_step(s, x, x, x, g),
        lambda: ops.paged_fork(i32(1), table, i32(0), i32(0), i32(1), i32(0), 8),
        lambda: ops.paged_free(table, i32(1), i32(0), i32(1), i32(0), 8, 2),
        lambda: ops.paged_compact(table, i32(1), i32(1), i32(0), 8, 2),
        lambda: ops.paged_copy(cache, cache, i32(0), i32(1)),
        lambda: ops.adjust_logits(torch.zeros(1, 4)),
    ]
    for call in calls:
        with pytest.raises(ValueError, match="requires CUDA"):
            call()


def test_linear_attention_refusals(any_device):
    x, g, s = heads(), torch.zeros(2), torch.zeros(1, 2, 64, 64)
    cu = i32(0, 4)
    run = lambda q=x, k=x, v=x, d=g, c=cu, n=4, **kw: ops.linear_attention(  # noqa: E731
        q, k, v, d, c, n, **kw)
    with pytest.raises(TypeError, match="BF16, FP16 or FP32"):
        run(q=x.double(), k=x.double(), v=x.double())
    with pytest.raises(TypeError, match="one type"):
        run(k=x.half())
    with pytest.raises(TypeError, match="log_decay"):
        run(d=g.bfloat16())
    with pytest.raises(TypeError, match="log_decay"):
        run(d=torch.zeros(1, 4, 2))
    with pytest.raises(ValueError, match="log_decay"):
        run(d=torch.zeros(3, 2))
    with pytest.raises(ValueError, match="log_decay"):
        run(d=torch.zeros(4))
    with pytest.raises(ValueError, match="shape"):
        run(q=x[0])
    with pytest.raises(ValueError, match="same tokens"):
        run(k=heads(5))
    with pytest.raises(ValueError, match="same tokens"):
        run(k=heads(d=128))
    with pytest.raises(ValueError, match="multiple of the query heads"):
        run(q=heads(h=3))
    with pytest.raises(ValueError, match="multiple of the query heads"):
        run(k=heads(h=4))
    with pytest.raises(ValueError, match="multiples of 8"):
        run(q=heads(d=136), k=heads(d=136))
    with pytest.raises(ValueError, match="multiples of 8"):
        run(v=heads(d=12))
    with pytest.raises(TypeError, match="cu_seqlens"):
        run(c=i64(0, 4))
    with pytest.raises(ValueError, match="one entry more"):
        run(c=i32())
    with pytest.raises(ValueError, match="max_seqlen"):
        run(n=0)
    with pytest.raises(ValueError, match="scale"):
        run(scale=0.0)
    with pytest.raises(ValueError, match="scale"):
        run(scale=float("nan"))
    with pytest.raises(TypeError, match="state must be"):
        run(state=s.bfloat16())
    with pytest.raises(ValueError, match="heads and widths"):
        run(state=torch.zeros(1, 2, 64, 32))
    with pytest.raises(ValueError, match="dense"):
        run(state=s.transpose(2, 3))
    with pytest.raises(ValueError, match="dense"):
        run(state=s[:, :1].expand(1, 2, 64, 64))
    with pytest.raises(ValueError, match="dense"):
        run(state=s.expand(3, 2, 64, 64))
    with pytest.raises(ValueError, match="slot for every request"):
        run(c=i32(0, 2, 4), state=s)
    with pytest.raises(ValueError, match="goes with state"):
        run(state_index=i32(0))
    with pytest.raises(TypeError, match="state_index"):
        run(state=s, state_index=i64(0))
    with pytest.raises(ValueError, match="1 entries"):
        run(state=s, state_index=i32(0, 0))
    with pytest.raises(ValueError, match="slot for every request"):
        ops.linear_attention_step(s, x, x, x, g)
    with pytest.raises(ValueError, match="scale"):
        ops.linear_attention_step(torch.zeros(4, 2, 64, 64), x, x, x, g, scale=-1.0)


def test_ranks_of_a_step(any_device):
    x, g, s = heads(), torch.zeros(2), torch.zeros(4, 2, 64, 64)
    for q in (x[0, 0, 0], x[0, 0], x[0], x[None]):
        with pytest.raises(ValueError, match="q must have shape"):
            ops.linear_attention_step(s, q, x, x, g)


def test_states_that_overlap_are_refused(c_calls, library):
    x, g, size = heads(), torch.zeros(2), 64 * 64
    memory = torch.zeros(16 * size)
    step = lambda slot, head: ops.linear_attention_step(  # noqa: E731
        memory.as_strided((4, 2, 64, 64), (slot, head, 64, 1)), x, x, x, g)
    for slot, head in ((size, size), (2 * size, 2 * size), (size, 3 * size), (size + 4, size),
                       (2 * size, size + 4), (size, 4 * size - 4)):
        with pytest.raises(ValueError, match="of its own"):
            step(slot, head)
    # Slots outside, heads outside, slots apart.
    for slot, head in ((2 * size, size), (size, 4 * size), (4 * size, size), (2 * size + 4, size + 4)):
        step(slot, head)
    assert len(c_calls) == 4
    some = ctypes.c_void_p(1 << 20)       # never read: without tokens a call only checks
    call = lambda slot, head, slots=4, h=2: library.kb_linear_attention_step(  # noqa: E731
        some, 128, 64, 2, some, 128, 64, 2, some, 128, 64, h, 64, 64, 0, some, 1, some, slot, head,
        slots, None, 0, 1.0, some, None)
    assert call(size, size) == call(size - 4, 4 * size) == call(2 * size, size - 4) == 2
    assert call(size, 3 * size) == call(1 << 61, 1 << 61, slots=1 << 29) == 2
    assert call(2 * size, size) == call(size, 4 * size) == call(1 << 61, size, slots=1 << 62) == 0
    assert call(0, size, slots=1) == call(0, 0, slots=0) == 0


def test_workspace_size_is_asked_for_on_the_tensors_device(monkeypatch, c_calls):
    # It depends on the SMs of the device that the call runs on, which need not be current.
    current, asked = [0], []

    class Library:
        @staticmethod
        def kb_linear_attention_workspace_size(*args):
            asked.append((current[0], args))
            return 640 + current[0]

    @contextlib.contextmanager
    def on(device):
        before, current[0] = current[0], device.index
        yield
        current[0] = before

    monkeypatch.setattr(ops, "_current_device", lambda: current[0])
    monkeypatch.setattr(ops._lib, "lib", lambda: Library)
    monkeypatch.setattr(torch.cuda, "device", on)
    size = "kb_linear_attention_workspace_size"
    assert ops._size_on(torch.device("cuda", 1), size, 1, 2) == 641 and current == [0]
    assert ops._size_on(torch.device("cuda", 0), size, 3) == 640
    assert asked == [(1, (1, 2)), (0, (3,))]
    ask = lambda device, *args: (asked.append(device), 4096)[1]  # noqa: E731
    monkeypatch.setattr(ops, "_size_on", ask)
    x = heads()
    ops.linear_attention(x, x, x, torch.zeros(2), i32(0, 4), 4)
    assert asked[-1] == x.device and c_calls[0][-2] == 4096


def test_page_refusals(any_device):
    table, one = i32(0, 1, 2, 3).view(2, 2), i32(1, 1)
    fork = lambda c=one, t=table, s=i32(0), d=i32(1), f=i32(4), h=i32(0), n=8, **kw: (  # noqa: E731
        ops.paged_fork(c, t, s, d, f, h, n, **kw))
    with pytest.raises(TypeError, match="block_table"):
        fork(t=table.long())
    with pytest.raises(ValueError, match="unit stride"):
        fork(t=table.T)
    with pytest.raises(ValueError, match="unit stride"):
        fork(t=table[:1].expand(2, 2))
    with pytest.raises(ValueError, match="requires a request"):
        fork(t=table[:, :0])
    with pytest.raises(ValueError, match="requires a request"):
        fork(n=0)
    with pytest.raises(ValueError, match="2 entries"):
        fork(c=i32(1))
    with pytest.raises(ValueError, match="in place"):
        fork(c=i32(1, 1, 1, 1)[::2])
    with pytest.raises(ValueError, match="in place"):
        fork(reserved_lens=i32(1, 1, 1, 1)[::2])
    with pytest.raises(ValueError, match="1 entries"):
        fork(d=i32(1, 0))
    with pytest.raises(TypeError, match="sources"):
        fork(s=i64(0))
    none = fork(s=i32(), d=i32())
    assert none.free_head.tolist() == [0] and none.missing.tolist() == [0]
    free = lambda t=table, r=one, k=one, f=i32(4, 5), h=i32(1), n=8, p=6: (  # noqa: E731
        ops.paged_free(t, r, k, f, h, n, p))
    with pytest.raises(ValueError, match="num_pages"):
        free(p=0)
    with pytest.raises(ValueError, match="in place"):
        free(f=i32(1, 2, 3, 4)[::2])
    with pytest.raises(ValueError, match="2 entries"):
        free(k=i32(1))
    with pytest.raises(TypeError, match="free_head"):
        free(h=i64(0))
    with pytest.raises(ValueError, match="num_pages"):
        ops.paged_compact(table, one, i32(4), i32(0), 8, -1)
    with pytest.raises(ValueError, match="2 entries"):
        ops.paged_compact(table, i32(1), i32(4), i32(0), 8, 6)
    cache = torch.zeros((4, 8, 2, 64), dtype=torch.bfloat16)
    with pytest.raises(TypeError, match="BF16 or FP16"):
        ops.paged_copy(cache, cache.half(), i32(0), i32(1))
    with pytest.raises(TypeError, match="BF16 or FP16"):
        ops.paged_copy(cache.float(), cache.float(), i32(0), i32(1))
    with pytest.raises(ValueError, match="same pages"):
        ops.paged_copy(cache, cache[:3], i32(0), i32(1))
    with pytest.raises(ValueError, match="multiples of 8"):
        ops.paged_copy(cache[..., :20], cache, i32(0), i32(1))
    with pytest.raises(ValueError, match="positive strides"):
        ops.paged_copy(cache[:1].expand(4, 8, 2, 64), cache, i32(0), i32(1))
    with pytest.raises(ValueError, match="1 entries"):
        ops.paged_copy(cache, cache, i32(0), i32(1), i32(1, 2))
    ops.paged_copy(cache, cache, i32(), i32())


def test_adjust_logits_refusals(any_device):
    x, lens, one = torch.zeros(2, 40), i32(3, 3), torch.ones(2)
    history = torch.zeros(2, 5, dtype=torch.long)
    words = torch.zeros(2, 2, dtype=torch.int32)
    run = ops.adjust_logits
    with pytest.raises(TypeError, match="logits"):
        run(x.double())
    with pytest.raises(TypeError, match="logits"):
        run(x[0])
    with pytest.raises(ValueError, match="vocabulary"):
        run(x[:, :0])
    with pytest.raises(ValueError, match="go with cu_tokens"):
        run(x, tokens=i64(0, 0))
    with pytest.raises(ValueError, match="goes with tokens"):
        run(x, cu_tokens=i32(0, 2), tree_mask=i64(1, 1))
    with pytest.raises(ValueError, match="one entry more"):
        run(x, cu_tokens=i32())
    with pytest.raises(ValueError, match="2 entries"):
        run(x, cu_tokens=i32(0, 2), tokens=i64(0))
    with pytest.raises(ValueError, match="go with history"):
        run(x, history_lens=lens)
    with pytest.raises(ValueError, match="needs history_lens"):
        run(x, history=history)
    with pytest.raises(TypeError, match="history"):
        run(x, history=history.int(), history_lens=lens)
    with pytest.raises(ValueError, match="2 rows"):
        run(x, history=history[:1], history_lens=lens)
    with pytest.raises(TypeError, match="repetition"):
        run(x, repetition=one.bfloat16())
    with pytest.raises(ValueError, match="2 entries"):
        run(x, presence=one[:1])
    with pytest.raises(ValueError, match="go together"):
        run(x, bias_ids=history)
    with pytest.raises(ValueError, match="shape of bias_ids"):
        run(x, bias_ids=history, bias_values=torch.zeros(2, 4))
    with pytest.raises(ValueError, match="at most 4096"):
        run(x, bias_ids=torch.zeros(2, 4097, dtype=torch.long), bias_values=torch.zeros(2, 4097))
    with pytest.raises(TypeError, match="allowed"):
        run(x, allowed=words.long())
    with pytest.raises(ValueError, match="bit for every token"):
        run(x, allowed=words[:, :1])
    with pytest.raises(ValueError, match="2 rows"):
        run(x, allowed=words[:1])
    with pytest.raises(ValueError, match="type, shape and device"):
        run(x, out=torch.zeros(2, 41))
    with pytest.raises(ValueError, match="unit stride"):
        run(x, out=torch.zeros(40, 2).T)
    with pytest.raises(ValueError, match="unit stride"):
        run(x, out=torch.zeros(1, 40).expand(2, 40))
    both = torch.zeros(100)
    with pytest.raises(ValueError, match="lie apart"):
        run(both[:80].view(2, 40), out=both[10:90].view(2, 40))


@pytest.fixture()
def c_calls(monkeypatch, any_device):
    # The arguments that reach the C entries, of CPU tensors.
    calls: list = []
    monkeypatch.setattr(ops, "_on", lambda device: lambda *args: calls.append(args))
    monkeypatch.setattr(ops, "_raw_stream", lambda device: 0)
    return calls


def test_rows_that_share_memory_keep_their_stride(c_calls):
    # One grammar, one history, one list of biases for all rows: their rows stay where they are.
    x, lens = torch.zeros(8, 100), i32(*[3] * 8)
    one = lambda width, dtype: torch.zeros(1, width, dtype=dtype)  # noqa: E731
    history, ids, values = one(5, torch.long), one(7, torch.long), one(7, torch.float32)
    words = one(4, torch.int32)
    spread = lambda t: t.expand(8, t.shape[1])  # noqa: E731
    ops.adjust_logits(x, history=spread(history), history_lens=lens, bias_ids=spread(ids),
                      bias_values=spread(values), allowed=spread(words))
    # Rows that overlap (one word further each), and rows of a wider matrix.
    sliding = torch.zeros(11, dtype=torch.int32).as_strided((8, 4), (1, 1))
    ops.adjust_logits(x, allowed=sliding)
    wide = torch.zeros(8, 9, dtype=torch.int32)[:, 2:6]
    ops.adjust_logits(x, allowed=wide)
    for args, held, stride in ((c_calls[0], words, 0), (c_calls[1], sliding, 1),
                               (c_calls[2], wide, 9)):
        assert args[0] == "kb_adjust_logits"
        at = args.index(held.data_ptr())
        assert args[at + 1] == stride
    for t, stride_at in ((history, 1), (ids, 1), (values, 1)):
        assert c_calls[0][c_calls[0].index(t.data_ptr()) + stride_at] == 0


def test_adjust_logits_in_place_by_any_view(c_calls, library):
    # The logits themselves are one row of a wider matrix here, of other strides there.
    wide = torch.zeros(3, 100)
    row, same = wide[:1, :40], wide[0, :40].view(1, 40)
    assert row.stride() != same.stride()
    assert ops.adjust_logits(row, out=same) is same
    assert c_calls[0][1] == c_calls[0][6] == wide.data_ptr()
    with pytest.raises(ValueError, match="lie apart"):
        ops.adjust_logits(wide[:2, :40], out=wide.view(-1)[:80].view(2, 40))
    some = ctypes.c_void_p(1 << 20)       # never read
    call = lambda stride, n=2: library.kb_adjust_logits(  # noqa: E731
        some, 50, n, 40, 2, some, stride, 0, None, 0, 0, *[None] * 6, 0, None, 0, 0, None, 0, some,
        None, None, None)
    assert call(60) == 2


def test_c_checks(library):
    some = ctypes.c_void_p(1 << 20)       # never read: the checks come first
    step = lambda **kw: library.kb_linear_attention_step(  # noqa: E731
        some, 128, 64, kw.get("hq", 2), some, 128, 64, 2, kw.get("v", some), kw.get("vs", 128), 64,
        2, kw.get("dk", 64), 64, kw.get("dtype", 0), some, 1, some, 8192, 4096, 4, None,
        kw.get("b", 1), kw.get("scale", 1.0), some, None)
    assert step(hq=3) == 2 and step(scale=0.0) == 2 and step(b=-1) == 2
    assert step(dk=136) == 6 and step(dk=60) == 6 and step(dtype=3) == 6 and step(b=1 << 40) == 6
    assert step(v=None) == 1 and step(vs=4) == 4 and step(b=0) == 0
    lin = lambda total=100, longest=100, cu=some, ws=0: library.kb_linear_attention(  # noqa: E731
        some, 128, 64, 2, some, 128, 64, 2, some, 128, 64, 2, 64, 64, 0, some, 1, None, 0, 0, 0,
        None, cu, 1, total, longest, 1.0, some, None, ws, None)
    assert lin(total=0) == 0 and lin(cu=None) == 1 and lin(longest=0) == 2
    assert library.kb_linear_attention_workspace_size(1, 2, 64, 64, 0, 5000, 5000) > 0
    assert library.kb_linear_attention_workspace_size(1, 400, 64, 64, 0, 5, 5) == 0
    assert library.kb_linear_attention_workspace_size(1, 2, 64, 64, 2, 5000, 5000) == 0
    assert library.kb_linear_attention_workspace_size(0, 2, 64, 64, 0, 0, 0) == 0
    fork = lambda b=2, n=1, free=some, w=4: library.kb_paged_fork(  # noqa: E731
        some, None, b, some, w, 4, some, some, n, free, 5, some, 8, some, some, some, some, some,
        None)
    assert fork(b=0) == 2 and fork(n=0) == 2 and fork(w=3) == 2
    assert fork(b=20_000) == 6 and fork(n=20_000) == 6 and fork(free=None) == 1
    free = lambda p=100, keep=some: library.kb_paged_free(  # noqa: E731
        some, keep, 2, some, 4, 4, some, 5, some, 8, p, some, None)
    assert free(p=0) == 2 and free(p=(1 << 19) + 1) == 6 and free(keep=None) == 1
    compact = lambda p=100, out=some: library.kb_paged_compact(  # noqa: E731
        some, 2, some, 4, 4, some, 5, some, 8, p, out, some, some, some, some, some, None)
    assert compact(p=0) == 2 and compact(out=None) == 1
    strides = (ctypes.c_int64 * 3)(1024, 128, 64)
    odd, none = (ctypes.c_int64 * 3)(1024, 128, 4), (ctypes.c_int64 * 3)(0, 128, 64)
    copy = lambda s=strides, n=3, d=64, a=some: library.kb_paged_copy(  # noqa: E731
        some, s, some, strides, 4, 8, 2, d, 64, a, some, None, n, None)
    assert copy(n=0) == 0 and copy(n=-1) == 2 and copy(d=60) == 6 and copy(s=odd) == 4
    assert copy(s=none) == 2 and copy(a=None) == 1
    adjust = lambda rows=2, b=2, stride=40, x=some, n=0, dtype=2, mask=None: (  # noqa: E731
        library.kb_adjust_logits(x, stride, rows, 40, dtype, some, 40, b, None, 0, 0, None, None,
                                 None, None, None, some, 0, some, 0, n, None, 0, None, None, mask,
                                 None))
    assert adjust(rows=0) == 0 and adjust(stride=39) == 2 and adjust(n=5000) == 6
    assert adjust(dtype=3) == 6 and adjust(x=None) == 1 and adjust(b=3) == 1
    assert adjust(mask=some) == 1 and adjust(b=70_000, rows=70_000) == 6
    assert adjust(x=ctypes.c_void_p((1 << 20) + 2)) == 4


def test_c_checks_of_alignment(library):
    at = lambda n: ctypes.c_void_p((1 << 20) + n)  # noqa: E731
    adjust = lambda history=at(0), lens=at(0), ids=at(0), allowed=at(0): (  # noqa: E731
        library.kb_adjust_logits(at(0), 40, 2, 40, 2, at(0), 40, 3, history, 9, 9, lens, None, None,
                                 None, None, ids, 4, at(0), 4, 4, allowed, 2, at(0), None, None,
                                 None))
    assert adjust(history=at(4)) == 4 and adjust(ids=at(4)) == 4
    assert adjust(lens=at(2)) == 4 and adjust(allowed=at(1)) == 4


def test_the_definitions_themselves():
    # The oracle against closed forms.
    q = torch.ones(3, 1, 8)
    out, size, end, _ = ref.linear_attention(q, q, q, torch.zeros(1), [0, 3], 0.5)
    assert out[:, 0, 0].tolist() == [4.0, 8.0, 12.0] and torch.equal(out, size)
    assert float(end[0, 0, 0, 0]) == 3.0
    g = torch.tensor([0.0, float("-inf"), 0.0])[:, None]
    assert ref.linear_attention(q, q, q, g, [0, 3], 0.5)[0][:, 0, 0].tolist() == [4.0, 4.0, 8.0]
    got = ref.fork([5, 0, 0], [[7, 8], [-1, -1], [-1, -1]], [0, 0], [1, 2], [3], 0, 4)
    assert got[0] == [5, 5, 0] and got[1][1] == [7, 3] and got[2:5] == ([8, -1], [3, -1], [1, 0])
    assert got[5:] == (1, 1)
    assert ref.free([[7, 8], [7, 2]], [8, 8], [0, 5], [0, 0, 5], 2, 4) == ([0, 8, 5], 1)
    rows, listed, head, moves = ref.compact([[9, 4]], [8], [1, 2, 3], 0, 4)
    assert rows == [[2, 1]] and moves == [(4, 1), (9, 2)] and (listed, head) == ([3, 4, 9], 0)
    x, _ = ref.adjust(torch.tensor([2.0, -2.0, 1.0]), [0], [1, 1], 2.0, 0.5, 0.25, [(2, 1.0)], {0, 1})
    assert x.tolist() == [1.0, -5.0, float("-inf")]
