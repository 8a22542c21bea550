"""The hooks that torch lets a user register around an optimizer's dictionaries."""
import pytest

from bit_reproducible_training_b200 import repro_optim
from test_gpu_optim import HYPER, make
from test_gpu_optim_groups import fill

pytestmark = pytest.mark.gpu


def test_state_dict_hooks_run():
    ps, gs = make([40], 37)
    fill(ps, gs)
    opt = repro_optim.AdamW(ps, **HYPER)
    opt.step()
    seen = []
    opt.register_state_dict_pre_hook(lambda o: seen.append("save"))
    opt.register_state_dict_post_hook(lambda o, d: {**d, "note": 5})
    opt.register_load_state_dict_pre_hook(lambda o, d: (seen.append(d.pop("note")), d)[1])
    opt.register_load_state_dict_post_hook(lambda o: seen.append("loaded"))
    saved = opt.state_dict()
    assert saved["note"] == 5
    opt.load_state_dict(saved)
    assert seen == ["save", 5, "loaded"] and saved["note"] == 5
