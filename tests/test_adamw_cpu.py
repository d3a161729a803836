"""The 8-bit moments' format, from its definition: scales, dither, rounding (the oracle of test_gpu_adamw.py), and what it promises."""
import pytest
import torch

BLOCK = 256
M32 = 0xFFFFFFFF


def mix(x):
    """the dither's mixing of 32-bit numbers (int64 tensors)"""
    for shift, mul in ((16, 0x85A308D3), (15, 0x13198A2F)):
        x = x ^ (x >> shift)
        x = ((x & 0xFFFF) * mul + ((((x >> 16) * mul) & 0xFFFF) << 16)) & M32
    return x ^ (x >> 16)


def mix_dither(sizes, seed, step):
    key = mix(torch.tensor(seed & M32) ^ mix(torch.tensor(step)))
    out = [mix(torch.arange(-(-n // BLOCK) * BLOCK) ^ mix(key ^ mix(torch.tensor(i)))) for i, n in enumerate(sizes)]
    x = torch.cat(out)
    return (x & 0xFFFF).float() / 65536, (x >> 16).float() / 65536


def moments(m, v, g, b1, b2):
    """fp32, one rounding per operation"""
    f = lambda s: torch.tensor(s, dtype=torch.float64).float()  # noqa: E731
    return f(b1) * m + f(1 - b1) * g, f(b2) * v + f(1 - b2) * (g * g)


def hold(x, u, top, least, digits, floor):
    """(values in steps of the block's scale, scales)"""
    x = x.view(-1, BLOCK)
    most = torch.where(x.isfinite(), x.abs(), torch.zeros_like(x)).amax(1)
    s = torch.ldexp(torch.ones_like(most), (torch.frexp(most).exponent - 1 - top).clamp(min=-126))
    s = torch.where(most > 0, s, torch.ones_like(s))
    y = x / s[:, None]
    q = torch.ldexp(torch.ones_like(y), (torch.frexp(y).exponent - 1).clamp(min=least) - digits)
    k = torch.floor(y.abs() / q + u.view(-1, BLOCK))
    if floor:
        k = torch.where(y != 0, k.clamp(min=1), k)
    return torch.copysign(k * q, y).view(-1), s


def test_values_fit_the_8_bit_types():
    x = torch.randn(64 * BLOCK, generator=torch.Generator().manual_seed(1)) * 3
    x = x * (torch.arange(64 * BLOCK) % 7 * -3.0).exp()
    for u in (0.0, 0.5, 1 - 2.0 ** -16):
        m, s = hold(x, torch.full_like(x, u), 7, -6, 3, False)
        assert torch.equal(m.to(torch.float8_e4m3fn).float(), m) and m.abs().max() <= 256
        v, s = hold(x.abs(), torch.full_like(x, u), 14, -14, 2, True)
        assert torch.equal(v.to(torch.float8_e5m2).float(), v) and v.min() > 0 and v.max() <= 2 ** 15


def test_rounding_is_right_on_average_and_keeps_what_is_on_the_grid():
    x = torch.linspace(0.3, 1.7, BLOCK)
    draws = []
    for step in range(1, 4001):
        draws.append(hold(x, mix_dither([BLOCK], 9, step)[0], 7, -6, 3, False)[0] * hold(x, torch.zeros(BLOCK), 7, -6, 3, False)[1])
    mean = torch.stack(draws).double().mean(0)
    # a draw is off by up to a step of 2^-3 of the value: standard deviation of 4,000 draws' mean below 2^-3 / 2 / sqrt(4000); six of them
    assert ((mean - x.double()).abs() <= 6 * 2.0 ** -4 / 4000 ** 0.5 * x.double() + 2.0 ** -17 * x).all()
    m, s = hold(x, torch.full((BLOCK,), 0.5), 7, -6, 3, False)
    on = m * s
    for u in (0.0, 0.999):
        again, s2 = hold(on, torch.full((BLOCK,), u), 7, -6, 3, False)
        assert torch.equal(again * s2, on)


def test_dither_is_even_and_differs_by_step_and_tensor():
    a, b = mix_dither([4096, 4096], 1, 1), mix_dither([4096, 4096], 1, 2)
    for u in a + b:
        # the mean of 8,192 numbers even in [0, 1): standard deviation 0.2887 / sqrt(8192) = 0.0032; six of them
        assert abs(u.mean().item() - 0.5) < 0.0192 and u.min() >= 0 and u.max() < 1
    assert (a[0] == b[0]).float().mean() < 0.01 and (a[0][:4096] == a[0][4096:]).float().mean() < 0.01


def test_second_moment_follows_its_average():
    """4,000 steps at b2 = 0.999 on gradients of constant size 1 from v = 4: rounding to nearest never leaves 4; the dither does."""
    v, s = hold(torch.full((BLOCK,), 4.0), torch.zeros(BLOCK), 14, -14, 2, True)
    stuck = v * s
    v = v * s
    for step in range(1, 4001):
        x = 0.999 * v + 0.001
        q, sc = hold(x, mix_dither([BLOCK], 3, step)[1], 14, -14, 2, True)
        v = q * sc
        q, sc = hold(0.999 * stuck + 0.001, torch.full((BLOCK,), 0.5), 14, -14, 2, True)
        stuck = q * sc
    assert (stuck == 4.0).all()
    want = 1 + 3 * 0.999 ** 4000
    # the values' spread is about 30 %; the mean of 256 of them within 0.3 / 16 = 0.019: six of them
    assert abs(v.mean().item() - want) < 0.12 and v.min() >= 0.25 and v.max() <= 4


def moved_state(p, bits):
    """An optimizer over p whose moments are not zeros, and what they stand for, in p's shape."""
    from selfc_amd import optim
    opt = optim.AdamW([p], state_bits=bits)
    opt.ensure_state()
    b, = opt._buckets[0]
    x = torch.randn(b.m.numel(), generator=torch.Generator().manual_seed(2)) * (torch.arange(b.m.numel()) // BLOCK % 5 * -3.0).exp()
    if bits == 8:
        codes, s = hold(x, torch.full_like(x, 0.5), 7, -6, 3, False)
        b.m.copy_(codes.to(torch.float8_e4m3fn))
        b.scales[0].copy_(s)
    else:
        b.m.copy_(x)
    return opt, held(opt, p)


def held(opt, p):
    """exp_avg as numbers, from the buffers in p's memory order"""
    b, = opt._buckets[0]
    m = b.m.float() if b.scales[0] is None else b.m.float() * b.scales[0].repeat_interleave(BLOCK)
    return m[:p.numel()].as_strided(p.shape, p.stride())


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("shape", [(32, 16, 3, 3), (24, 40, 1, 1), (7, 3, 5, 5)])
def test_state_of_another_memory_format(bits, shape):
    """The blocks of 8-bit moments follow memory: a state either means what it meant where it was saved, or is refused."""
    kinds = (torch.contiguous_format, torch.channels_last)
    for a in kinds:
        for b in kinds:
            p, q = (torch.nn.Parameter(torch.zeros(shape).to(memory_format=k)) for k in (a, b))
            opt, want = moved_state(p, bits)
            again, before = moved_state(q, bits)
            again._buckets[0][0].m.view(torch.uint8).zero_()
            saved = opt.state_dict()
            same = p.stride() == q.stride() or shape[2:] == (1, 1)
            if bits == 8 and not same:
                with pytest.raises(ValueError, match="memory format"):
                    again.load_state_dict(saved)
                assert not held(again, q).any()                # refused before anything was changed
            else:
                again.load_state_dict(saved)
                assert torch.equal(held(again, q), want)


def test_a_loaded_rate_is_a_copy():
    """A rate that is a tensor of the saving optimizer's: its later changes stay there."""
    from selfc_amd import optim
    p, q, r = (torch.nn.Parameter(torch.zeros(3)) for _ in range(3))
    a, b, c = optim.AdamW([p], lr=torch.tensor(0.5)), optim.AdamW([q], lr=0.25), optim.AdamW([r], lr=torch.tensor(0.125))
    a.param_groups[0]["initial_lr"] = torch.tensor(0.75)
    own = c.param_groups[0]["lr"]
    for other in (b, c):
        other.load_state_dict(a.state_dict())
    a.param_groups[0]["lr"].fill_(9.0)
    a.param_groups[0]["initial_lr"].fill_(9.0)
    for other in (b, c):
        assert float(other.param_groups[0]["lr"]) == 0.5 and float(other.param_groups[0]["initial_lr"]) == 0.75
    assert c.param_groups[0]["lr"] is own


@pytest.mark.parametrize("bits", [32, 8])
def test_a_restart_clears_the_moments_where_they_are(bits):
    """MultiStepLR_Restart(clear_state): the buffers that a captured step holds are cleared, and stay the optimizer's."""
    from selfc_amd.train import MultiStepLR_Restart
    p = torch.nn.Parameter(torch.zeros(300, 5))
    opt, before = moved_state(p, bits)
    b, = opt._buckets[0]
    b.steps.fill_(7)
    assert before.any()
    sch = MultiStepLR_Restart(opt, [100], restarts=[3], weights=[0.5], clear_state=True)
    opt._opt_called = True                                   # (what a step leaves for the scheduler's check of their order)
    at = [t.data_ptr() for t in (b.m, b.v, b.steps)]
    for k in range(3):
        assert torch.equal(held(opt, p), before) and opt.state[p]["step"].item() == 7
        sch.step()
    assert opt.param_groups[0]["lr"] == 0.5e-3
    again, = opt._group_buckets(0)
    assert again is b and at == [t.data_ptr() for t in (b.m, b.v, b.steps)]
    assert not held(opt, p).any() and opt.state[p]["step"].item() == 0 and set(opt.state_dict()["state"]) == {0}
    if bits == 8:
        assert (b.scales[0] == 1).all() and (b.scales[1] == 1).all()
