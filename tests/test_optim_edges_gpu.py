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


def test_flat_ranges_of_a_parameter_store_step_like_its_tensors():
    """neighbours of one decay as one tensor, their zero padding between them: parameters, copies and norm are those of the list of views"""
    from cfd_amd import nets, ops, trainer
    got = []
    for flat in (False, True):
        net = nets.CnnRegressor((16, 64, 1), dtype=torch.bfloat16, seed=5)
        P = net.params
        P.enable_training()
        P.grad.copy_(torch.randn(P.n_trainable, generator=torch.Generator().manual_seed(3)))
        names, spans = [], []
        for name, s in sorted(P.specs.items(), key=lambda kv: kv[1].offset):
            if s.kind != "stat":
                decay = 0.004 if name.endswith("kernel") else 0.0
                spans = spans if spans and spans[-1][1] == decay else spans + [(s.offset, decay)]
                names.append((name, decay))
        cuts = [a for a, _ in spans] + [P.n_trainable]
        ranges = [slice(a, b) for a, b in zip(cuts, cuts[1:])]
        live = torch.zeros_like(P.grad)
        for name, _ in names:
            o, n = P.specs[name].offset, P.specs[name].numel
            live[o:o + n] = 1
        P.grad.mul_(live)
        assert not (P.master[:P.n_trainable] * (1 - live)).any() and len(ranges) < len(names)
        if flat:
            opt = trainer.AdamW([P.master[r] for r in ranges], copies=[P.compute[r] for r in ranges], weight_decay=[d for _, d in spans], **HYPER)
            grads = [P.grad[r] for r in ranges]
        else:
            opt = trainer.AdamW([P.m(n) for n, _ in names], copies=[P.c(n) for n, _ in names], weight_decay=[d for _, d in names], **HYPER)
            grads = [P.g(n) for n, _ in names]
        norms = [ops.grad_norm(P.grad if flat else grads, 0.1) for _ in range(3)]
        for n in norms:
            opt.step(grads, torch.full((1,), 0.01, device="cuda"))
        got.append((P.master.clone(), P.compute.clone(), norms[0]))
    (a, ca, na), (b, cb, nb) = got
    assert torch.equal(a, b) and torch.equal(ca, cb)
    assert (na - nb).abs().max() <= 2.0 ** -23 * na.abs().max()     # (fp64 sums in another order, rounded once)
