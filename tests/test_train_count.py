"""The trainer's step count without a GPU."""
import pytest
import torch

from gs_b200 import _lib


def _raise(*a, **k):
    raise _lib.GsError("gs_adamw_step", _lib.GS_ERR_INVALID_ARGUMENT, "refused")


def test_a_refused_update_is_not_counted(monkeypatch):
    from gs_b200.training import trainer
    st = trainer.DensityState(4, 1, "cpu")
    mask = st.active_mask.view(torch.uint8)

    class Plan:
        def update(self):
            _raise()
        step = update
    monkeypatch.setattr(_lib, "call", _raise)
    monkeypatch.setattr(_lib, "ptr", lambda t: None)
    with pytest.raises(_lib.GsError):
        trainer._update(st, trainer.AdamConfig(), mask, 0)
    monkeypatch.setattr(trainer.DensityState, "adamw", lambda self, opt: Plan())
    with pytest.raises(_lib.GsError):
        trainer._update(st, trainer.AdamConfig(max_grad_norm=1.0), mask, 0)
    assert st.count == 0


def test_the_count_is_the_devices_once_steps_may_be_skipped(monkeypatch):
    from gs_b200.training import trainer
    st = trainer.DensityState(4, 1, "cpu")
    mask = st.active_mask.view(torch.uint8)

    class Plan:
        def update(self):
            pass  # skipped: the device does not advance adam_state[0]
    monkeypatch.setattr(_lib, "call", lambda *a: None)
    monkeypatch.setattr(_lib, "ptr", lambda t: None)
    monkeypatch.setattr(trainer.DensityState, "adamw", lambda self, opt: Plan())
    trainer._update(st, trainer.AdamConfig(), mask, 0)
    assert st.count == 1  # plain Adam never skips: the host's own count
    st.adam_state[0] = 1
    trainer._update(st, trainer.AdamConfig(max_grad_norm=1.0), mask, 0)
    assert st.count == 1
    st.adam_state[0] = 2
    assert st.count == 2
