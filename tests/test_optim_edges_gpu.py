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


@pytest.mark.parametrize("beta_2", [0.999, 0.9999])
def test_what_the_8_bit_state_settles_at(beta_2):
    """v of a constant gradient after four times 1 / (1 - beta_2) steps.  Each step stores it low by 0 to 2^-16 spacings of a quarter at
    most, 2^-18 of the value: 2^-18 / (1 - beta_2) in all.  The recursion's four fp32 roundings a step, 2^-24 each, add
    2^-22 / (1 - beta_2) either way; the mean of n elements has a standard error."""
    from cfd_amd import trainer
    n, steps = 1 << 18, int(4 / (1 - beta_2))
    g = torch.full((n,), 1.3, device="cuda").sqrt()
    opt = trainer.AdamW([torch.zeros(n, device="cuda")], lr=0.0, beta_2=beta_2, weight_decay=0.0, state_bits=8, seed=11)
    for _ in range(steps):
        opt.step([g])
    v = (opt.v.float() * opt.v_scale.repeat_interleave(256)).double()
    want = 1.3 * (1 - beta_2 ** steps)
    off, noise = (float(v.mean()) - want) / want, 5 * float(v.std()) / n ** 0.5 / want + 2.0 ** -22 / (1 - beta_2)
    print(f"beta_2 {beta_2}: v {100 * off:.3f} %, 5 standard errors and fp32 {100 * noise:.3f} %")
    assert -(2.0 ** -18 / (1 - beta_2)) - noise <= off <= noise


def test_slow_betas_need_a_32_bit_state():
    from cfd_amd import trainer
    p = torch.zeros(8, device="cuda")
    opt = trainer.AdamW([p], beta_1=0.9999, beta_2=0.9999, state_bits=8)
    for kw in (dict(beta_1=0.99991), dict(beta_2=0.99999)):
        with pytest.raises(ValueError):
            trainer.AdamW([p], state_bits=8, **kw)
        trainer.AdamW([p], **kw).step([torch.ones_like(p)])
    with pytest.raises(ValueError):
        opt.b2 = 0.99999
    opt.step([torch.ones_like(p)])


def test_a_norm_past_fp32_reads_as_infinity_and_still_clips():
    """the factor is the fp64 quotient rounded once: half of fp32's smallest subnormal"""
    from cfd_amd import ops
    n = ops.grad_norm([torch.full((100,), 3e38, device="cuda")], 1.0)
    assert float(n[0]) == float("inf") and abs(float(n[1]) - 1 / (10 * float(torch.tensor(3e38)))) <= 2.0 ** -150
