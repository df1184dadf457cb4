"""The whole-model example's handling of its options and steps, as far as no GPU is needed."""

import sys

import pytest


def test_a_step_that_comes_by_twice_is_counted_once():
    """(a step whose capture failed is made eagerly)"""
    from examples.llama_step import step_counter

    class Optimizer:
        reads_device_hyper, counted = True, 0

        def pre_step(self):
            self.counted += 1

    opt = Optimizer()
    count = step_counter(opt)
    for step in (0, 1, 2, 2, 3):
        count(step)
    assert opt.counted == 4
    opt = Optimizer()
    opt.reads_device_hyper = False
    step_counter(opt)(0)
    step_counter(object())(0)
    assert opt.counted == 0


@pytest.mark.parametrize("options,named", [(("--tp", "2", "--fp8-products"), "--fp8-products"), (("--baseline", "--fp8-products"), "--fp8-products"),
                                           (("--baseline", "--rest-state", "int8"), "--rest-state")])
def test_options_that_would_be_ignored_are_refused(options, named, capsys, monkeypatch):
    from examples import llama_step
    monkeypatch.setattr(sys, "argv", ["llama_step.py", *options])
    with pytest.raises(SystemExit) as e:
        llama_step.main()
    assert e.value.code == 2 and named in capsys.readouterr().err
