"""DensityState.count is the device's step count, whatever was skipped or refused."""
import pytest

from tests.test_gpu_adamw_skip import _bad
from tests.test_gpu_adamw_train import _state

pytestmark = pytest.mark.gpu


def test_the_count_is_the_devices_after_a_skip():
    from gs_b200.training.trainer import CapturedStep, train_step
    st, opt, cam, views = _state(max_grad_norm=1.0)
    train_step(st, *views[0], cam, opt, sh_degree=3)
    train_step(st, *_bad(views[1]), cam, opt, sh_degree=3)
    assert int(st.skipped) == 1 and st.count == int(st.adam_state[0]) == 1
    step = CapturedStep(st, *_bad(views[1]), cam, opt, sh_degree=3)
    assert int(st.skipped) == 2 and st.count == int(st.adam_state[0]) == 1
    step(*views[2])
    assert st.count == int(st.adam_state[0]) == 2
    step(*_bad(views[1]))
    step(*views[3])
    assert int(st.skipped) == 3 and st.count == int(st.adam_state[0]) == 3


def test_a_refused_step_is_not_counted():
    from gs_b200 import _lib
    from gs_b200.training.trainer import train_step
    for kw in (dict(b1=1.0, max_grad_norm=1.0), dict(transition_steps=-1)):
        st, opt, cam, views = _state(max_grad_norm=kw.pop("max_grad_norm", None))
        for k, v in kw.items():
            setattr(opt, k, v)
        with pytest.raises(_lib.GsError):
            train_step(st, *views[0], cam, opt, sh_degree=3)
        assert st.count == int(st.adam_state[0]) == 0
