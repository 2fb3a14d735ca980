"""AdamW's attributes, its flat ranges and what its 8-bit state's rounding adds up to."""
import pytest
import torch

from tests.test_optim_gpu import HYPER, _check_step, _views

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [32, 8])
def test_attributes_take_effect_at_the_next_step(bits):
    """each hyper-parameter that can be assigned is what the following steps use; a bad value is refused and changes nothing"""
    from cfd_amd import trainer
    sizes, wd = [300, 5], [0.02, 0.0]
    opt = trainer.AdamW(_views(sizes, torch.float32, 1, 0.05), weight_decay=wd, state_bits=bits, **HYPER)
    lr = HYPER["lr"]
    _check_step(opt, _views(sizes, torch.float32, 10), None, lr, wd)
    opt.b1, opt.b2 = 0.5, 0.9
    _check_step(opt, _views(sizes, torch.float32, 11), 0.5, lr, wd)
    opt.eps = 0.25
    _check_step(opt, _views(sizes, torch.float32, 12), None, lr, wd)
    opt.weight_decay = 0.3
    _check_step(opt, _views(sizes, torch.float32, 13), None, lr, [0.3, 0.3])
    opt.weight_decay = wd = [0.0, 0.9]
    _check_step(opt, _views(sizes, torch.float32, 14), None, lr, wd)
    opt.seed = 123456789
    _check_step(opt, _views(sizes, torch.float32, 15), None, lr, wd)
    opt.lr = lr = 0.01
    _check_step(opt, _views(sizes, torch.float32, 16), None, lr, wd)
    for name, bad in (("b1", 1.0), ("b2", -0.1), ("b2", float("nan")), ("eps", 0.0), ("weight_decay", [0.1])):
        kept = getattr(opt, name)
        with pytest.raises(ValueError):
            setattr(opt, name, bad)
        assert getattr(opt, name) == kept
    with pytest.raises(TypeError):
        opt.weight_decay[0] = 0.5
    _check_step(opt, _views(sizes, torch.float32, 17), None, lr, wd)
