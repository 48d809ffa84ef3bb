"""CPU tests of the logit rules' launcher: what it refuses, before anything is launched."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest


def _call(gx, rules, **change):
    """The launcher with good host memory everywhere, one thing changed."""
    a = dict(logits=np.zeros(256, np.float32), row_stride=100, vocabulary=70, batch=2, output=np.zeros(256, np.float32),
             output_stride=100, tokens=np.zeros(2, np.uint32), workspace=np.zeros(64, np.uint64), bytes=512)
    a.update(change)
    at = lambda x: None if x is None else x if isinstance(x, int) else x.ctypes.data  # noqa: E731
    return gx.lib().gfxinfer_launch_logit_rules(at(a["logits"]), a["row_stride"], a["vocabulary"], a["batch"],
                                                None if rules is None else ctypes.byref(rules), at(a["output"]),
                                                a["output_stride"], at(a["tokens"]), at(a["workspace"]), a["bytes"], None)


@pytest.mark.parametrize("change,word", [
    (dict(logits=None), "arguments"), (dict(output=None, tokens=None), "arguments"), (dict(vocabulary=0), "arguments"),
    (dict(vocabulary=(1 << 24) + 1, row_stride=1 << 25, output_stride=1 << 25), "arguments"), (dict(batch=0), "arguments"),
    (dict(batch=65536), "arguments"), (dict(row_stride=69), "arguments"), (dict(output_stride=69), "arguments"),
    (dict(workspace=None), "workspace"), (dict(bytes=15), "workspace"),
    (dict(vocabulary=1 << 24, row_stride=1 << 24, output_stride=1 << 24, batch=2048, bytes=1 << 40), "too many rows")])
def test_bad_arguments_are_refused(gx, change, word):
    assert _call(gx, gx.LogitRules(), **change) == gx.INVALID_ARGUMENT
    assert word in gx.last_error()


def test_null_rules_misaligned_workspace_and_shifted_rows_are_refused(gx):
    assert _call(gx, None) == gx.INVALID_ARGUMENT
    work = np.zeros(64, np.uint64)
    assert _call(gx, gx.LogitRules(), workspace=work.ctypes.data + 4) == gx.INVALID_ARGUMENT
    same = np.zeros(512, np.float32)
    assert _call(gx, gx.LogitRules(), logits=same, output=same, output_stride=101) == gx.INVALID_ARGUMENT
    assert "in place" in gx.last_error()


@pytest.mark.parametrize("fields", [
    dict(history=8, history_stride=4, history_row_count=2),                                # no lengths
    dict(history=8, history_lengths=8, history_stride=0, history_row_count=2),
    dict(history=8, history_lengths=8, history_stride=1 << 19, history_row_count=2),
    dict(history=8, history_lengths=8, history_stride=4, history_row_count=1),             # a row each without history_rows
    dict(bias_tokens=8, bias_stride=4), dict(bias_values=8, bias_stride=4),
    dict(bias_tokens=8, bias_values=8, bias_stride=0), dict(bias_tokens=8, bias_values=8, bias_stride=4096),
    dict(allowed=8, allowed_stride=2, allowed_row_count=2),                                # 70 tokens need 3 words
    dict(allowed=8, allowed_stride=3, allowed_row_count=1)])
def test_bad_rules_are_refused(gx, fields):
    """The addresses are never followed: a refused call launches nothing."""
    rules = gx.LogitRules()
    for k, v in fields.items():
        setattr(rules, k, v)
    assert _call(gx, rules) == gx.INVALID_ARGUMENT


def test_workspace_bytes_of_bad_sizes(gx):
    for vocabulary, batch in ((0, 1), ((1 << 24) + 1, 1), (10, 0), (10, 65536)):
        assert gx.logit_rules_workspace_bytes(vocabulary, batch) == 0
    assert gx.logit_rules_workspace_bytes(10, 3) >= 24


def test_rules_from_tensors_check_shapes(gx):
    import torch
    i = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    f = lambda *s: torch.zeros(s)  # noqa: E731
    rules = gx.LogitRules.of(history=i(3, 9), history_rows=i(4), history_lengths=i(4), bias_tokens=i(4, 5), bias_values=f(4, 5),
                             allowed=i(2, 7), allowed_rows=i(4), presence=None)
    assert (rules.history_row_count, rules.history_stride, rules.bias_stride, rules.allowed_row_count, rules.allowed_stride,
            rules.batch) == (3, 9, 5, 2, 7, 4)
    for bad in (dict(history=i(9)), dict(presence=f(2, 2)), dict(presence=f(2).double()), dict(history=i(3, 9)[:, ::2]),
                dict(bias_tokens=i(4, 5)), dict(bias_tokens=i(4, 5), bias_values=f(4, 6)), dict(presence=f(2), frequency=f(3))):
        with pytest.raises(ValueError):
            gx.LogitRules.of(**bad)
    with pytest.raises(TypeError):
        gx.LogitRules.of(temperature=f(2))
    for logits, output in ((f(3, 70), f(3, 70)), (f(4, 70).t().contiguous().t(), None), (f(4, 70).double(), None),
                           (f(4, 70), f(3, 70))):
        with pytest.raises(ValueError):
            gx.launch_logit_rules(logits, rules, output, i(4), i(100), stream=0)


def test_rules_from_tensors_check_types_and_room(gx):
    import torch
    i = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    f = lambda *s: torch.zeros(s)  # noqa: E731
    for bad in (dict(presence=i(2)), dict(repetition=i(2)), dict(history=f(2, 9)), dict(bias_counts=f(2)), dict(allowed=f(2, 3)),
                dict(bias_tokens=i(2, 3), bias_values=i(2, 3))):
        with pytest.raises(ValueError):
            gx.LogitRules.of(**bad)
    rules = gx.LogitRules.of(presence=f(4))
    for output, tokens, vocabulary in ((None, i(3), 70), (None, i(8)[::2], 70), (None, i(4).long(), 70), (None, i(4), 71),
                                       (f(4, 60), i(4), 70)):
        with pytest.raises(ValueError):
            gx.launch_logit_rules(f(4, 70), rules, output, tokens, i(100), vocabulary, stream=0)


def test_integer_logits_and_host_memory_are_refused(gx):
    import torch
    i = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    f = lambda *s: torch.zeros(s)  # noqa: E731
    rules = gx.LogitRules.of(presence=f(4))
    assert rules.device == -1
    for logits, output in ((i(4, 70), None), (f(4, 70), i(4, 70))):
        with pytest.raises(ValueError):
            gx.launch_logit_rules(logits, rules, output, i(4), i(100), stream=0)
    with pytest.raises(gx.GfxinferError, match="memory"):
        gx.launch_logit_rules(f(4, 70), rules, f(4, 70), i(4), i(100), stream=0)
