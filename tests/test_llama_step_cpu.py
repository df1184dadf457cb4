"""The whole-model example's handling of its options and steps, as far as no GPU is needed."""


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
