"""What the operators of drafted trees refuse, how their launches are cut, on a machine without a GPU."""
import re
from types import SimpleNamespace

import pytest
import torch

from einf_b200 import ops
from einf_b200.engine import ModelRunner, StepError
from einf_b200.ops import build


@pytest.fixture
def on_this_machine(monkeypatch):
    """Tensors of the CPU pass for tensors of the current device, and a launch is recorded instead of made."""
    calls = []

    def fn(symbol, argtypes, variant=""):
        def launch(*args):
            assert len(args) == len(argtypes)
            calls.append(symbol)
            return 0
        return launch

    def pointer(t, name):
        if not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous")
        return t.data_ptr()

    monkeypatch.setattr(ops, "_fn", fn)
    monkeypatch.setattr(ops, "_dev", pointer)
    monkeypatch.setattr(ops, "_current", lambda: (-1, 0))
    monkeypatch.setattr(ops, "_sm_count", lambda: 148)
    return calls


def ints(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def attention_arguments(**change):
    given = dict(
        q=torch.zeros(5, 4, 48), k_cache=torch.zeros(6, 2, 4, 48), v_cache=torch.zeros(6, 2, 4, 48), block_table=ints(2, 3),
        q_start=ints(3), cached_lens=ints(2), tree_mask=torch.zeros(5, 1, dtype=torch.int64), out=torch.zeros(5, 4, 48), scale=0.1,
        status=ints(1))
    given.update(change)
    return given


@pytest.mark.parametrize("change, error", [
    (dict(out=torch.zeros(5, 4, 32)), ValueError),
    (dict(v_cache=torch.zeros(6, 2, 8, 48)), ValueError),
    (dict(out=torch.zeros(5, 4, 48, dtype=torch.bfloat16)), TypeError),
    (dict(q=torch.zeros(5, 4, 48).half(), k_cache=torch.zeros(6, 2, 4, 48).half(), v_cache=torch.zeros(6, 2, 4, 48).half(),
          out=torch.zeros(5, 4, 48).half()), TypeError),
    (dict(q=torch.zeros(5, 3, 48), out=torch.zeros(5, 3, 48)), ops.UnsupportedSize),
    (dict(q=torch.zeros(5, 4, 260), out=torch.zeros(5, 4, 260), k_cache=torch.zeros(6, 2, 4, 260), v_cache=torch.zeros(6, 2, 4, 260)),
     ops.UnsupportedSize),
    (dict(q_start=ints(2)), ValueError),
    (dict(block_table=ints(1, 3)), ValueError),
    (dict(tree_mask=ints(5, 1)), TypeError),
    (dict(tree_mask=torch.zeros(4, 1, dtype=torch.int64)), ValueError),
    (dict(tree_mask=torch.zeros(5, 0, dtype=torch.int64)), ValueError),
    (dict(window=0), ValueError),
    (dict(window=7), ValueError),
    (dict(window=7, positions=ints(4)), ValueError),
    (dict(softcap=0.0), ValueError),
    (dict(softcap=float("nan")), ValueError),
    (dict(scale=0.0), ValueError),
    (dict(cached_lens=torch.zeros(2, dtype=torch.int64)), TypeError),
    (dict(status=torch.zeros(1)), TypeError),
    (dict(q=torch.zeros(4, 5, 48).transpose(0, 1)), ValueError),
])
def test_tree_attention_refuses(on_this_machine, change, error):
    with pytest.raises(error):
        ops.tree_attention(**attention_arguments(**change))
    assert on_this_machine == []


def test_tree_attention_launches(on_this_machine):
    ops.tree_attention(**attention_arguments())
    assert on_this_machine == ["einf_tree_attention"]
    ops.tree_attention(**attention_arguments(window=3, positions=ints(5), softcap=5.0, max_nodes=3, max_cached=0))
    none = dict(q=torch.zeros(0, 4, 48), out=torch.zeros(0, 4, 48), tree_mask=torch.zeros(0, 1, dtype=torch.int64))
    ops.tree_attention(**attention_arguments(**none))
    assert len(on_this_machine) == 2


def logits_arguments(**change):
    given = dict(logits=torch.zeros(6, 50), out=torch.zeros(6, 50), row_start=ints(3), status=ints(1), history=ints(2, 9),
                 history_lens=ints(2), prompt_lens=ints(2), repetition=torch.ones(2), presence=torch.ones(2), frequency=torch.ones(2),
                 node_tokens=ints(6), tree_mask=torch.zeros(6, 1, dtype=torch.int64), bias_ids=ints(2, 3), bias=torch.zeros(2, 3),
                 allowed=ints(6, 2))
    given.update(change)
    return given


@pytest.mark.parametrize("change, error", [
    (dict(logits=torch.zeros(6, 50, dtype=torch.bfloat16)), TypeError),
    (dict(out=torch.zeros(6, 51)), ValueError),
    (dict(row_start=ints(0)), ValueError),
    (dict(history=None), ValueError),
    (dict(history=None, history_lens=None), ValueError),
    (dict(history=ints(3, 9)), ValueError),
    (dict(history_lens=ints(3)), ValueError),
    (dict(prompt_lens=ints(1)), ValueError),
    (dict(repetition=torch.ones(6)), ValueError),
    (dict(repetition=torch.ones(2, dtype=torch.float64)), TypeError),
    (dict(node_tokens=None), ValueError),
    (dict(tree_mask=None), ValueError),
    (dict(node_tokens=ints(5)), ValueError),
    (dict(bias=None), ValueError),
    (dict(bias=torch.zeros(2, 4)), ValueError),
    (dict(allowed=ints(6, 1)), ValueError),
    (dict(allowed=ints(5, 2)), ValueError),
    (dict(allowed_rows=ints(5)), ValueError),
    (dict(allowed=None, allowed_rows=ints(6)), ValueError),
    (dict(allowed=torch.zeros(6, 2, dtype=torch.int64)), TypeError),
])
def test_shape_logits_refuses(on_this_machine, change, error):
    with pytest.raises(error):
        ops.shape_logits(**logits_arguments(**change))
    assert on_this_machine == []


def test_shape_logits_launches(on_this_machine):
    ops.shape_logits(**logits_arguments())
    ops.shape_logits(torch.zeros(4, 7), torch.zeros(4, 7), None, ints(1))
    ops.shape_logits(**logits_arguments(allowed=ints(1, 2), allowed_rows=ints(6)))
    assert on_this_machine == ["einf_shape_logits"] * 3
    ops.shape_logits(torch.zeros(0, 7), torch.zeros(0, 7), None, ints(1))
    assert len(on_this_machine) == 3


@pytest.mark.parametrize("change, error", [
    (dict(targets=ints(5)), ValueError),
    (dict(parents=ints(7)), ValueError),
    (dict(q_start=ints(2)), ValueError),
    (dict(path=ints(2, 0), answer=ints(2, 0)), ValueError),
    (dict(answer=ints(2, 5)), ValueError),
    (dict(path=ints(3, 4), answer=ints(3, 4)), ValueError),
    (dict(targets=torch.zeros(6, dtype=torch.int64)), TypeError),
])
def test_accept_drafts_refuses(on_this_machine, change, error):
    given = dict(node_tokens=ints(6), targets=ints(6), parents=ints(6), q_start=ints(3), path=ints(2, 4), answer=ints(2, 4), counts=ints(2))
    ops.accept_drafts(**given)
    with pytest.raises(error):
        ops.accept_drafts(**dict(given, **change))
    assert on_this_machine == ["einf_accept_drafts"]


def test_cache_rows_refuses_what_two_of_them_share(on_this_machine):
    both = torch.zeros(2, 6, 2, 4, 8)
    ops.CacheRows([both[1], both[0]])
    for caches in ([both[0], both[0]], [both[0], both.view(-1)[8:8 + 6 * 2 * 4 * 8].view(6, 2, 4, 8)], [both[1], both[0], both.view(12, 2, 4, 8)[3:9]]):
        with pytest.raises(ValueError, match="share memory"):
            ops.CacheRows(caches)


def test_tree_attention_of_the_widest_window_and_the_most_nodes(on_this_machine):
    ops.tree_attention(**attention_arguments(window=1 << 40, positions=ints(5)))
    assert on_this_machine == ["einf_tree_attention"]
    many = (1 << 19) + 1
    with pytest.raises(ops.UnsupportedSize):
        ops.tree_attention(**attention_arguments(
            q=torch.zeros(many, 2, 1), out=torch.zeros(many, 2, 1), k_cache=torch.zeros(6, 2, 4, 1), v_cache=torch.zeros(6, 2, 4, 1),
            tree_mask=torch.zeros(many, 1, dtype=torch.int64)))


def test_cache_rows_refuses(on_this_machine):
    good = [torch.zeros(6, 2, 4, 8), torch.zeros(6, 1, 4, 3, dtype=torch.bfloat16)]
    assert ops.CacheRows(good[:1]).unit == 16 and ops.CacheRows(good).unit == 2
    for caches, error in (([], ValueError), ([torch.zeros(6, 2, 4)], ValueError), ([good[0], torch.zeros(5, 2, 4, 8)], ValueError),
                          ([good[0], torch.zeros(6, 2, 8, 8)], ValueError), ([torch.zeros(6, 2, 4, 8, dtype=torch.int32)], TypeError),
                          ([torch.zeros(2, 6, 4, 8).transpose(0, 1)], ValueError), ([torch.zeros(0, 2, 4, 8)], ValueError)):
        with pytest.raises(error):
            ops.CacheRows(caches)


@pytest.mark.parametrize("change, error", [
    (dict(path=ints(3, 4)), ValueError),
    (dict(counts=ints(3)), ValueError),
    (dict(block_table=ints(1, 2)), ValueError),
    (dict(path=torch.zeros(2, 4, dtype=torch.int64)), TypeError),
])
def test_move_accepted_refuses(on_this_machine, change, error):
    caches = ops.CacheRows([torch.zeros(6, 2, 4, 8) for _ in range(200)])
    given = dict(caches=caches, block_table=ints(2, 2), cached_lens=ints(2), path=ints(2, 4), counts=ints(2), status=ints(1))
    ops.move_accepted(**given)
    assert on_this_machine == ["einf_move_accepted"] * 2      # 200 tensors: two launches
    ops.move_accepted(**dict(given, path=ints(2, 1)))         # a path of roots alone moves nothing
    with pytest.raises(error):
        ops.move_accepted(**dict(given, **change))
    assert len(on_this_machine) == 2


def test_tensors_of_the_cpu_are_refused():
    with pytest.raises(ops.KernelError):
        ops.tree_attention(**attention_arguments())
    with pytest.raises(ops.KernelError):
        ops.shape_logits(**logits_arguments())
    with pytest.raises(ops.KernelError):
        ops.accept_drafts(ints(6), ints(6), ints(6), ints(3), ints(2, 4), ints(2, 4), ints(2))
    with pytest.raises(ops.KernelError):
        ops.CacheRows([torch.zeros(6, 2, 4, 8)])


@pytest.mark.parametrize("source, kernel", [("drafts", "move_accepted_kernel"), ("drafts", "accept_drafts_kernel"), ("pointwise", "advance_decode_kernel")])
def test_kernels_that_change_what_a_later_step_reads_early_are_waited_for(source, kernel):
    """Decode kernels read positions, slots and the keys of earlier steps before they wait for the kernel before them: none may
    start before a kernel has ended that writes these."""
    text = (build.KERNEL_DIR / f"{source}.cu").read_text()
    body = re.search(rf"__global__ void[^;{{]*\b{kernel}\(.*?\n}}\n", text, re.S).group(0)
    assert "pdl_wait();" in body and "pdl_launch_dependents();" not in body


@pytest.mark.parametrize("source", ["logits.cu", "attention_tree_tcgen05.cu"])
def test_every_bounded_wait_is_asked_whether_it_ran_out(source):
    """A kernel goes on from a wait on a barrier only if what it waited for is there."""
    lines = (build.KERNEL_DIR / source).read_text().splitlines()
    assert any("bar_wait" in line for line in lines)
    assert [line for line in lines if re.match(r"\s*bar_wait\w*\(", line)] == []


@pytest.mark.parametrize("source", ["logits.cu", "attention_tree_tcgen05.cu"])
def test_no_kernel_leaves_copies_behind(source):
    """Where a wait has run out, the copies that were asked for are waited for, with a limit, before the CTA ends."""
    text = (build.KERNEL_DIR / source).read_text()
    assert re.search(r"// [^\n]*no (?:CTA|copy)\b[^\n]*under way.{0,300}bar_poll\(", text, re.S)


def test_a_device_that_does_not_say_what_it_holds_is_asked_again(monkeypatch):
    answers = {1: [0, 148], 4: [0, 36]}
    monkeypatch.setattr(ops, "_fn", lambda symbol, argtypes, variant="": lambda cluster: answers[cluster].pop(0))
    monkeypatch.setattr(ops, "_tree_room", {})
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    with pytest.raises(ops.KernelError):
        ops.tree_cluster_room(1)
    assert [ops.tree_cluster_room(1) for _ in range(2)] == [148, 148]
    assert [ops.tree_cluster_room(4) for _ in range(3)] == [0, 36, 36]
    # larger clusters that it does not hold are not chosen
    workers, cluster, whole = ops._tree_workers(2, 9, False, 148, lambda c: 148 if c == 1 else 0)
    assert cluster == 1 and workers >= 1


def test_a_launch_is_cut_for_the_device_that_it_is_on(on_this_machine, monkeypatch):
    """What is remembered of one device's launches is not taken for another's."""
    cuts = []
    monkeypatch.setattr(ops, "_SHAPE_CALL", SimpleNamespace(pack=lambda *values: cuts.append(values[-2:]) or b""))
    ops._shape_pieces.cache_clear()
    for device, sms in ((-1, 148), (-2, 1), (-1, 148)):
        monkeypatch.setattr(ops, "_current", lambda: (device, 0))
        monkeypatch.setattr(ops, "_sm_count", lambda: sms)
        monkeypatch.setattr(ops, "_at", lambda t, name, dtype, device: t.data_ptr())
        ops.shape_logits(torch.zeros(8, 5000), torch.zeros(8, 5000), ints(2), ints(1))
    ops._shape_pieces.cache_clear()
    assert cuts[0] == cuts[2] != cuts[1]


@pytest.mark.parametrize("change", [dict(q_start=ints(3, 1)), dict(q_start=ints(3, 2)), dict(cached_lens=ints(2, 1)), dict(cached_lens=ints(2, 2)),
                                    dict(window=3, positions=ints(5, 1))])
def test_tree_attention_looks_at_whole_shapes(on_this_machine, change):
    with pytest.raises(ValueError):
        ops.tree_attention(**attention_arguments(**change))
    assert on_this_machine == []


@pytest.mark.parametrize("name", ["history_lens", "prompt_lens", "repetition", "presence", "frequency"])
@pytest.mark.parametrize("shape", [(2, 1), (2, 2)])
def test_shape_logits_looks_at_whole_shapes(on_this_machine, name, shape):
    with pytest.raises(ValueError):
        ops.shape_logits(**logits_arguments(**{name: (ints if name.endswith("lens") else torch.ones)(*shape)}))
    with pytest.raises(ValueError):
        ops.shape_logits(**logits_arguments(row_start=ints(3, 2)))
    assert on_this_machine == []


def test_accept_drafts_looks_at_whole_shapes(on_this_machine):
    with pytest.raises(ValueError):
        ops.accept_drafts(ints(6), ints(6), ints(6), ints(3, 2), ints(2, 4), ints(2, 4), ints(2))
    assert on_this_machine == []


@pytest.mark.parametrize("rows, words", [((1 << 19), 64), ((1 << 25), 1)])
def test_shape_logits_refuses_more_rows_and_nodes_than_it_counts(on_this_machine, rows, words):
    def given(rows):
        return dict(logits=torch.zeros(1, 2).expand(rows, 2), out=torch.zeros(1, 2).expand(rows, 2), row_start=ints(2), status=ints(1),
                    node_tokens=ints(1).expand(rows), tree_mask=torch.zeros(1, words, dtype=torch.int64).expand(rows, words))

    with pytest.raises(ops.UnsupportedSize):
        ops.shape_logits(**given(rows))
    with pytest.raises(ValueError, match="contiguous"):      # a row less is not too many
        ops.shape_logits(**given(rows - 1))
    assert on_this_machine == []


def test_a_bad_index_fails_the_step():
    ModelRunner.check_status(0)
    with pytest.raises(StepError, match="an index outside what it points into") as caught:
        ModelRunner.check_status(ops.STATUS_BAD_INDEX)
    assert "page" not in str(caught.value)


@pytest.mark.parametrize("change", [dict(softcap=float("inf")), dict(scale=float("inf")), dict(scale=float("nan"))])
def test_tree_attention_refuses_scales_and_caps_that_are_not_finite(on_this_machine, change):
    """The kernels differ in what becomes of them: uncapped scores in one, no numbers in the other."""
    with pytest.raises(ValueError, match="finite"):
        ops.tree_attention(**attention_arguments(**change))
    assert on_this_machine == []


def test_tree_attention_without_heads_has_nothing_to_do(on_this_machine):
    ops.tree_attention(**attention_arguments(q=torch.zeros(5, 0, 48), out=torch.zeros(5, 0, 48)))
    assert on_this_machine == []


def test_a_status_without_a_word_is_refused(on_this_machine):
    caches = ops.CacheRows([torch.zeros(6, 2, 4, 8)])
    for call in (lambda: ops.tree_attention(**attention_arguments(status=ints(0))), lambda: ops.shape_logits(**logits_arguments(status=ints(0))),
                 lambda: ops.move_accepted(caches, ints(2, 2), ints(2), ints(2, 4), ints(2), ints(0))):
        with pytest.raises(ValueError, match="status"):
            call()
    assert on_this_machine == []
