"""The generation loop with prompts run once for several requests (no GPU)."""
import pytest

from pytorch_transformers_b200.config import GenerationConfig
from pytorch_transformers_b200.engine import run_generation
from test_generation_loop import ArgmaxSelector, FakeStepper


class ForkingStepper(FakeStepper):
    def fork(self, slot):
        new = self.open()
        self.length[new] = self.length[slot]
        return new


@pytest.mark.parametrize("max_batch", [1, 2, 3, 4, 6])
def test_one_prompt_step_for_equal_requests(max_batch):
    prompts = [[3, 4]] * 3 + [[9]] * 3
    kw = dict(budget=3, max_batch=max_batch)
    apart = run_generation(FakeStepper(6), ArgmaxSelector(), prompts, GenerationConfig(), **kw)
    stepper, selector = ForkingStepper(6), ArgmaxSelector()
    shared = run_generation(stepper, selector, prompts, GenerationConfig(), same_as=[0, 0, 0, 3, 3, 3], **kw)
    assert [r.tokens for r in shared] == [r.tokens for r in apart]
    assert [ids for ids, _, _ in selector.seen] == [ids for ids, _, _ in _seen(prompts, kw)]
    assert len(stepper.free) == 6                                 # every slot came back
    for slots, tokens in stepper.calls:
        if len(tokens[0]) == 2:
            assert sum(t == [3, 4] for t in tokens) == 1          # a batch runs the prompt once


def _seen(prompts, kw):
    selector = ArgmaxSelector()
    run_generation(FakeStepper(6), selector, prompts, GenerationConfig(), **kw)
    return selector.seen


def test_requests_that_are_alone_are_not_forked():
    stepper = FakeStepper(4)                                      # has no fork
    out = run_generation(stepper, ArgmaxSelector(), [[1], [2]], GenerationConfig(), 2, 2, same_as=[0, 1])
    assert [r.tokens for r in out] == [[2, 3], [3, 4]]


def test_a_fork_that_fails_gives_everything_back():
    class Full(ForkingStepper):
        def fork(self, slot):
            raise RuntimeError("no page")
    stepper = Full(4)
    with pytest.raises(RuntimeError):
        run_generation(stepper, ArgmaxSelector(), [[1], [1]], GenerationConfig(), 2, 2, same_as=[0, 0])
    assert len(stepper.free) == 4
