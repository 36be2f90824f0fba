"""AdamW on the GPU against its definition (oracle/lowbit_oracle.py).

Tolerances.  The new moments are compared to the bit with float32 arithmetic that rounds every operation, and with them the
8-bit codes.  A parameter: three roundings of 2^-24 on p (decay factor, product, difference; doubled for the sum of both terms),
and on the update term ten operations of at most 2^-23 each (square root and reciprocal to one unit in the last place):
4 * 2^-24 |p| + 10 * 2^-23 |update|, and half a step of bf16 (2^-8 |p'|) where the parameter is kept in it.  Among the denormal
numbers the product lr / (1 - b1^t) * m' is rounded to a multiple of 2^-149, off by 2^-150, and then divided by eps or more:
2^-150 / eps (1e-37 at eps = 1e-8)."""
import numpy as np
import pytest
import torch

from conv1d_text_vae_amd import _lib as L
from oracle import lowbit_oracle as O

pytestmark = pytest.mark.gpu
KIND = {'f32': torch.float32, 'bf16': torch.bfloat16}


@pytest.fixture(scope='module')
def optim():
    from conv1d_text_vae_amd import optim as m
    return m


def f64(t):
    return t.detach().float().cpu().numpy().astype(np.float64)


def f32(t):
    return t.detach().float().cpu().numpy()


def tensors(sizes, kind, seed, scale=1.0):
    rng = np.random.RandomState(seed)
    out = []
    for s in sizes:
        x = rng.standard_normal(s) * scale * np.exp(rng.standard_normal())
        if x.size > 4:
            x.reshape(-1)[::5] *= 1e-5                     # small values beside large ones
            x.reshape(-1)[2] = 0.0
        out.append(torch.from_numpy(x.astype(np.float32)).to(KIND[kind]).cuda())
    return out


def held(opt):
    """(m, v) per tensor, float32, padded to whole blocks"""
    out = []
    m, v = opt.m.view(torch.uint8).cpu().numpy() if opt.states == '8bit' else opt.m.cpu().numpy(), opt.v.cpu().numpy()
    for d in opt._host:
        a, b = d.offset, d.offset + -(-d.n // 128) * 128
        if opt.states == '8bit':
            sm, sv = opt.m_scale.cpu().numpy()[a // 128:b // 128], opt.v_scale.cpu().numpy()[a // 128:b // 128]
            out.append((O.unpack_m(m[a:b], sm), O.unpack_v(v[a:b], sv)))
        else:
            out.append((m[a:b], v[a:b]))
    return out


def check_step(opt, grads, lr, wd, clip=0.0, grad_scale=1.0):
    """One step of the optimizer against the oracle; the states before it are taken as they are held."""
    before = held(opt)
    p0 = [f64(p) for p in opt.params]
    t = int(opt.t.item()) + 1
    opt.step(grads, grad_scale)
    torch.cuda.synchronize()
    b1, b2 = opt.betas
    live = [g for g in grads if g is not None]
    factor, norm = O.clip_factor([f64(g) for g in live], clip, grad_scale)
    if clip > 0:
        n32 = np.float32(np.sqrt(sum(np.square(f64(g)).sum() for g in live))) * np.float32(abs(grad_scale))
        assert float(opt.norm.item()) == float(n32)
        f = (np.float32(1.0) / n32 * np.float32(clip) if n32 >= np.float32(clip) else np.float32(1.0)) * np.float32(grad_scale)
    else:
        f = np.float32(grad_scale)
    assert int(opt.t.item()) == t
    total = opt.m.numel()
    r = O.halves(total, opt.seed, t) if opt.states == '8bit' else None
    after_m = opt.m.view(torch.uint8).cpu().numpy() if opt.states == '8bit' else opt.m.cpu().numpy()
    after_v = opt.v.cpu().numpy()
    for i, (p, g, d) in enumerate(zip(opt.params, grads, opt._host)):
        a, b = d.offset, d.offset + -(-d.n // 128) * 128
        if g is None:
            np.testing.assert_array_equal(f64(p), p0[i])
            continue
        gp = np.zeros(b - a, dtype=np.float32)
        gp[:d.n] = f32(g).reshape(-1)
        m, v = O.moments(before[i][0], before[i][1], gp, f, b1, b2)
        if opt.states == '8bit':
            cm, sm = O.pack_m(m, r[a:b])
            cv, sv = O.pack_v(v, r[a:b])
            np.testing.assert_array_equal(opt.m_scale.cpu().numpy()[a // 128:b // 128], sm)
            np.testing.assert_array_equal(opt.v_scale.cpu().numpy()[a // 128:b // 128], sv)
            np.testing.assert_array_equal(after_m[a:b], cm)
            np.testing.assert_array_equal(after_v[a:b], cv)
        else:
            np.testing.assert_array_equal(after_m[a:b], m)
            np.testing.assert_array_equal(after_v[a:b], v)
        m, v = m[:d.n].astype(np.float64), v[:d.n].astype(np.float64)
        with np.errstate(all='ignore'):
            u = lr * (m / (1 - b1 ** t)) / (np.sqrt(v / (1 - b2 ** t)) + opt.eps)
            want = p0[i].reshape(-1) * (1 - lr * wd[i]) - u
        got = f64(p).reshape(-1)
        tol = 4 * 2.0 ** -24 * np.abs(p0[i].reshape(-1)) + 10 * 2.0 ** -23 * np.abs(u) + 2.0 ** -150 / opt.eps
        if p.dtype == torch.bfloat16:
            tol = tol + 2.0 ** -8 * np.abs(want)
        bad = ~np.isfinite(want)
        assert np.array_equal(np.isnan(got), np.isnan(want))
        assert (np.abs(got - want)[~bad] <= tol[~bad]).all(), np.nanmax(np.abs(got - want) / tol)


SIZES = [[(1,)], [(128,), (127,), (129,)], [(3, 5), (2048,), (1,), (2049,), (40, 60), (0,), (7,)], [(300, 257), (5000,), (64, 1000)]]


@pytest.mark.parametrize('states', ['f32', '8bit'])
@pytest.mark.parametrize('pk,gk', [('f32', 'f32'), ('f32', 'bf16'), ('bf16', 'bf16')])
@pytest.mark.parametrize('which', range(len(SIZES)))
def test_steps_follow_the_definition(optim, states, pk, gk, which):
    sizes = SIZES[which]
    params = tensors(sizes, pk, 1, 0.05)
    wd = [0.01 * (i % 3) for i in range(len(sizes))]
    clip = (0.0, 1.0, 1e6)[which % 3]
    opt = optim.AdamW(params, lr=3e-3, weight_decay=wd, clipnorm=clip, states=states, seed=77 + which)
    for t in range(4):
        check_step(opt, tensors(sizes, gk, 10 + t, 10.0 ** (t - 2)), 3e-3, wd, clip)


@pytest.mark.parametrize('states', ['f32', '8bit'])
def test_more_tensors_than_one_launch_takes(optim, states):
    sizes = [(i % 37 + 1, i % 5 + 1) for i in range(2 * L.ADAMW_GROUP + 9)]
    params = tensors(sizes, 'f32', 3)
    opt = optim.AdamW(params, lr=1e-2, weight_decay=0.1, clipnorm=0.5, states=states)
    for t in range(2):
        check_step(opt, tensors(sizes, 'f32', 20 + t), 1e-2, [0.1] * len(sizes), 0.5)


@pytest.mark.parametrize('states', ['f32', '8bit'])
def test_more_chunks_than_workgroups(optim, states):
    sizes = [(2050, 2048 + 13), (70000,)]
    params = tensors(sizes, 'f32', 4)
    opt = optim.AdamW(params, lr=1e-2, weight_decay=0.0, clipnorm=1.0, states=states, seed=1 << 40)
    check_step(opt, tensors(sizes, 'bf16', 5), 1e-2, [0.0, 0.0], 1.0)


@pytest.mark.parametrize('kind', ['f32', 'bf16'])
def test_norm_and_step_where_workgroups_take_several_turns(optim, kind):
    """18 M weights: the norm to the bit (its squares are exact in 64 bits and summed in them: the order of 2^24 additions of 2^-53
    shows in the 24 bits of the result only for a sum that lies on a border), the first step against its formula, and a step left
    out for one bad value in the last turn."""
    rng = torch.Generator('cuda').manual_seed(11)
    sizes = [2048 * 4100 + 77, 3, 2048 * 4600 + 1001]
    params = [torch.randn(n, generator=rng, device='cuda') for n in sizes]
    grads = [torch.randn(n, generator=rng, device='cuda').to(KIND[kind]) for n in sizes]
    before = [p.double() for p in params]
    opt = optim.AdamW(params, lr=0.01, weight_decay=0.1, clipnorm=5.0)
    opt.step(grads)
    norm = torch.cat([g.double().square() for g in grads]).sum().sqrt().item()
    assert opt.norm.item() == np.float32(norm)
    f = 5.0 / norm
    for p, p0, g in zip(params, before, grads):
        x = g.double() * f
        u = 0.01 * x / (x.abs() + opt.eps)                      # first step: m / (1 - b1) = g, v / (1 - b2) = g^2
        # the tolerance of this file, and the factor's own three roundings of 2^-24, which |x| / (|x| + eps) passes on at most whole
        tol = 4 * 2.0 ** -24 * p0.abs() + 13 * 2.0 ** -23 * u.abs() + 2.0 ** -150 / opt.eps
        assert ((p.double() - (p0 * (1 - 0.01 * 0.1) - u)).abs() <= tol).all()
    held = [p.clone() for p in params]
    grads[2][-1] = float('nan')
    opt.step(grads)
    assert np.isnan(opt.norm.item()) and int(opt.t.item()) == 1 and all(torch.equal(p, h) for p, h in zip(params, held))


@pytest.mark.parametrize('states', ['f32', '8bit'])
def test_offsets_beyond_32_bits(optim, states):
    """4.4 G weights in one tensor and a small one behind it: both ends move as the formula's first step says."""
    n = 2 ** 32 + 2 ** 27 + 5
    p, q = torch.zeros(n, dtype=torch.bfloat16, device='cuda'), torch.zeros(300, device='cuda')
    g = torch.ones(n, dtype=torch.bfloat16, device='cuda')
    g[n // 2:] = -1.0
    opt = optim.AdamW([p, q], lr=0.5, weight_decay=0.0, states=states)
    opt.step([g, torch.full((300,), 2.0, device='cuda')])
    # first step: -lr sign(g) (1 - 1e-8), half a step of bf16 and twelve of fp32 roundings near 0.5
    assert float((p[:n // 2].float() + 0.5).abs().max()) <= 0.5 * 2.0 ** -8 and float((p[n // 2:].float() - 0.5).abs().max()) <= 0.5 * 2.0 ** -8
    assert float((q + 0.5).abs().max()) <= 1e-5


@pytest.mark.parametrize('states', ['f32', '8bit'])
def test_views_at_odd_places_and_grad_scale(optim, states):
    flat = torch.zeros(4000, device='cuda')
    flat[:] = torch.linspace(-1, 1, 4000)
    params = [flat[3:1003], flat[1003:1004], flat[1005:3334].view(17, 137)]
    gflat = torch.randn(4001, generator=torch.Generator('cuda').manual_seed(1), device='cuda')
    grads = [gflat[1:1001], gflat[1001:1002], gflat[1002:3331].view(17, 137)]
    rest = flat[[0, 1, 2, 1004]].clone(), flat[3334:].clone()
    opt = optim.AdamW(params, lr=0.1, weight_decay=0.1, clipnorm=2.0, states=states)
    for _ in range(2):
        check_step(opt, grads, 0.1, [0.1] * 3, 2.0, 0.125)
    check_step(opt, grads, 0.1, [0.1] * 3, 2.0, -1.0)                        # an ascent is clipped as well
    assert torch.equal(flat[[0, 1, 2, 1004]], rest[0]) and torch.equal(flat[3334:], rest[1])


@pytest.mark.parametrize('states', ['f32', '8bit'])
def test_missing_and_strided_gradients(optim, states):
    sizes = [(10, 13), (200,), (9, 9)]
    opt = optim.AdamW(tensors(sizes, 'f32', 6), lr=0.1, weight_decay=0.1, states=states)
    g = tensors(sizes, 'f32', 7)
    check_step(opt, g, 0.1, [0.1] * 3)
    check_step(opt, [g[0], None, g[2].t()], 0.1, [0.1] * 3)
    for p, x in zip(opt.params, g):
        p.grad = x
    opt.params[1].grad = None
    q = opt.params[1].clone()
    opt.step()
    assert torch.equal(opt.params[1], q) and int(opt.t.item()) == 3


@pytest.mark.parametrize('states', ['f32', '8bit'])
@pytest.mark.parametrize('bad', [float('nan'), float('inf')])
def test_gradients_that_are_no_numbers(optim, states, bad):
    sizes = [(300,), (20, 10)]
    grads = tensors(sizes, 'f32', 8)
    # with the clip: the step is left out
    opt = optim.AdamW(tensors(sizes, 'f32', 9), lr=0.1, clipnorm=1.0, states=states)
    opt.step(grads)
    kept = [x.clone() for x in opt.params + opt.state_tensors()]
    grads[0][17] = bad
    opt.step(grads)
    assert not np.isfinite(opt.norm.item())
    for a, b in zip(kept, opt.params + opt.state_tensors()):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    # without: what depends on that value is NaN (or, in 8 bits, held as NaN), the rest of its block is not
    opt = optim.AdamW(tensors(sizes, 'f32', 9), lr=0.1, weight_decay=0.0, states=states)
    opt.step(grads)
    opt.step(tensors(sizes, 'f32', 10))
    p = opt.params[0]
    assert torch.isnan(p[17]) and torch.isfinite(p[torch.arange(300, device='cuda') != 17]).all()
    assert torch.isfinite(opt.params[1]).all()


def test_extreme_second_moments_in_8_bits(optim):
    """Gradients over 30 binades in one block: codes as defined, and no update explodes, for nothing is held as zero that is not."""
    g = torch.from_numpy((2.0 ** np.linspace(-40, 8, 256)).astype(np.float32)).cuda()
    opt = optim.AdamW([torch.zeros(256, device='cuda')], lr=1.0, weight_decay=0.0, states='8bit', eps=1e-20)
    for t in range(6):
        before = opt.params[0].clone()
        check_step(opt, [g * (1.0 if t % 2 else -1.0)], 1.0, [0.0])
        assert float((opt.params[0] - before).abs().max()) < 20.0
    check_step(opt, [torch.zeros(256, device='cuda')], 1.0, [0.0])
    tiny = torch.full((256,), 1e-30, device='cuda')
    opt = optim.AdamW([torch.zeros(256, device='cuda')], lr=1.0, weight_decay=0.0, states='8bit')
    check_step(opt, [tiny], 1.0, [0.0])
    check_step(opt, [tiny * 1e25], 1.0, [0.0])
    opt = optim.AdamW([torch.zeros(300, device='cuda')], lr=1.0, weight_decay=0.0, states='8bit')
    for t in range(3):                                       # moments among the denormal numbers
        check_step(opt, [torch.linspace(-1, 1, 300, device='cuda') * 10.0 ** (-37 - t)], 1.0, [0.0])


def test_8bit_moments_follow_the_32bit_ones_in_the_mean(optim):
    """600 steps of random gradients of known spread in 4096 weights.  The held v starts on its grid, so one step's rounding has
    the variance |change| x step <= 0.001 E|g^2/v - 1| (about 1) x v x v/8, remembered for 1 / (1 - 0.999^2) = 500 steps:
    0.063 v^2 at most, 0.25 v each; the mean over 4096 weights is off by 0.25 / 64 = 0.004 of it (one standard deviation), and
    2 % is five of them.  Rounding to nearest would leave it tens of percent off."""
    n = 4096
    gen = torch.Generator('cuda').manual_seed(5)
    a, b = torch.zeros(n, device='cuda'), torch.zeros(n, device='cuda')
    o8 = optim.AdamW([a], lr=0.0, states='8bit', weight_decay=0.0, seed=3)
    o32 = optim.AdamW([b], lr=0.0, states='f32', weight_decay=0.0)
    spread = torch.exp(0.5 * torch.randn(n, generator=gen, device='cuda'))
    for _ in range(600):
        g = spread * torch.randn(n, generator=gen, device='cuda')
        o8.step([g])
        o32.step([g])
    v8, v32 = o8.moments(0)[1], o32.moments(0)[1]
    assert abs(float((v8 / v32).mean()) - 1.0) < 0.02
    assert float((v8 / v32 - 1.0).std()) < 0.35


@pytest.mark.parametrize('states', ['f32', '8bit'])
def test_captured_step_replays(optim, states):
    sizes = [(300, 7), (129,)]
    grads = tensors(sizes, 'f32', 30)
    start = tensors(sizes, 'f32', 31)
    eager = optim.AdamW([p.clone() for p in start], lr=0.01, clipnorm=1.0, states=states, seed=9)
    opt = optim.AdamW([p.clone() for p in start], lr=0.01, clipnorm=1.0, states=states, seed=9)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        opt.step(grads)
    for k in range(4):
        with torch.no_grad():
            for x in grads:
                x.mul_(1.5)
        if k == 2:
            opt.set_lr(0.3)
            eager.set_lr(0.3)
        g.replay()
        eager.step(grads)
        torch.cuda.synchronize()
        for a, b in zip(opt.params + opt.state_tensors(), eager.params + eager.state_tensors()):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    assert int(opt.t.item()) == 4


def test_state_dict_continues_a_run(optim):
    sizes = [(300, 7), (129,)]
    grads = [tensors(sizes, 'f32', 40 + t) for t in range(4)]
    for states in ('f32', '8bit'):
        a = optim.AdamW(tensors(sizes, 'f32', 31), states=states)
        for t in range(2):
            a.step(grads[t])
        b = optim.AdamW([p.clone() for p in a.params], states=states)
        b.load_state_dict(a.state_dict())
        for t in (2, 3):
            a.step(grads[t])
            b.step(grads[t])
        for x, y in zip(a.params + a.state_tensors(), b.params + b.state_tensors()):
            assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))
        a.reset()
        assert int(a.t.item()) == 0 and not a.moments(0)[0].any() and not a.moments(0)[1].any()
    with pytest.raises(ValueError):
        a.load_state_dict(optim.AdamW([torch.zeros(5, device='cuda')]).state_dict())


def test_parameters_may_move_between_steps(optim):
    p = torch.nn.Parameter(torch.ones(200, device='cuda'))
    opt = optim.AdamW([p], lr=0.1, weight_decay=0.0)
    g = torch.ones(200, device='cuda')
    opt.step([g])
    p.data = torch.full((200,), 5.0, device='cuda')
    opt.step([g])
    assert torch.allclose(p.data, torch.full((200,), 4.9, device='cuda'), atol=1e-5)
    for other in (torch.ones(200, device='cuda').half(), torch.ones(200, device='cuda').bfloat16(), torch.ones(201, device='cuda'),
                  torch.ones(400, device='cuda')[::2], torch.ones(200)):
        q = torch.nn.Parameter(torch.ones(200, device='cuda'))
        opt = optim.AdamW([q], lr=0.1)
        q.data = other
        with pytest.raises(ValueError):
            opt.step([g])


def test_gradients_of_mixed_types(optim):
    sizes = [(10, 13), (200,), (9, 9), (5,)]
    opt = optim.AdamW(tensors(sizes, 'f32', 6), lr=0.1, weight_decay=0.1, clipnorm=1.0)
    a, b = tensors(sizes, 'f32', 7), tensors(sizes, 'bf16', 8)
    check_step(opt, [a[0], b[1], b[2].t(), None], 0.1, [0.1] * 4, 1.0)
    opt.params.pop()
    with pytest.raises(ValueError):
        opt.step(a)
    with pytest.raises(ValueError):
        opt.step(a[:3])


def test_refusals(optim):
    p = torch.zeros(10, 10, device='cuda')
    for bad in (lambda: optim.AdamW([]), lambda: optim.AdamW([p, p]), lambda: optim.AdamW([p, p[3:]]), lambda: optim.AdamW([p.t()[1:]]),
                lambda: optim.AdamW([p.double()]), lambda: optim.AdamW([p], weight_decay=[0.1, 0.2]), lambda: optim.AdamW([p], states='f16'),
                lambda: optim.AdamW([p], lr=-1.0), lambda: optim.AdamW([p], eps=0.0), lambda: optim.AdamW([p], betas=(1.0, 0.9)),
                lambda: optim.AdamW([p, torch.zeros(3)]), lambda: optim.AdamW([p]).step([]), lambda: optim.AdamW([p]).step([p[0]]),
                lambda: optim.AdamW([p]).step([p.double()]), lambda: optim.AdamW([p]).step([p], grad_scale=float('nan'))):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(L.C1VError):
        optim.AdamW([torch.zeros(4)])


@pytest.mark.parametrize('states', ['f32', '8bit'])
def test_states_beside_moments_that_are_no_numbers(optim, states):
    """Without the clip: NaN, infinities and a square that overflows at every place of a group of four bytes and before the padding;
    every other state of their blocks to the bit, then a step from what is held.  (The sign of a NaN is nobody's business.)"""
    n = 300
    bad = {4: float('nan'), 9: float('inf'), 14: float('-inf'), 19: 3e19, 130: 3e19, 133: float('nan'), 160: float('nan'), 163: -3e19, 299: float('inf')}
    g = torch.linspace(-1, 1, n).double() ** 3
    g[5], g[10], g[131] = 0.0, 1e-12, 0.0
    for i, x in bad.items():
        g[i] = x
    first, second = g.float().cuda(), torch.linspace(1, -1, n, device='cuda')
    opt = optim.AdamW([torch.ones(n, device='cuda')], lr=0.1, weight_decay=0.1, states=states, seed=5)
    for t, grad in ((1, first), (2, second), (3, second)):
        before, p0 = held(opt)[0], f64(opt.params[0])
        opt.step([grad])
        gp = np.zeros(384, dtype=np.float32)
        gp[:n] = f32(grad)
        m, v = O.moments(before[0], before[1], gp, np.float32(1.0), *opt.betas)
        if states == '8bit':
            r = O.halves(384, opt.seed, t)
            cm, sm = O.pack_m(m, r)
            cv, sv = O.pack_v(v, r)
            got = opt.m.view(torch.uint8).cpu().numpy()
            np.testing.assert_array_equal(opt.m_scale.cpu().numpy(), sm)
            np.testing.assert_array_equal(opt.v_scale.cpu().numpy(), sv)
            np.testing.assert_array_equal(np.where(np.isnan(m), got & 0x7F, got), np.where(np.isnan(m), cm & 0x7F, cm))
            np.testing.assert_array_equal(opt.v.cpu().numpy(), cv)
        else:
            np.testing.assert_array_equal(opt.m.cpu().numpy(), m)
            np.testing.assert_array_equal(opt.v.cpu().numpy(), v)
        m, v = m[:n].astype(np.float64), v[:n].astype(np.float64)
        with np.errstate(all='ignore'):
            u = 0.1 * (m / (1 - 0.9 ** t)) / (np.sqrt(v / (1 - 0.999 ** t)) + opt.eps)
            want = p0 * (1 - 0.1 * 0.1) - u
            tol = 4 * 2.0 ** -24 * np.abs(p0) + 10 * 2.0 ** -23 * np.abs(u) + 2.0 ** -150 / opt.eps
        got = f64(opt.params[0])
        assert np.array_equal(np.isnan(got), np.isnan(want))
        fine = np.isfinite(want)
        assert fine.sum() >= n - len(bad) and (np.abs(got - want)[fine] <= tol[fine]).all()


@pytest.mark.parametrize('states', ['f32', '8bit'])
def test_second_moments_among_the_denormal_numbers_and_a_tiny_eps(optim, states):
    """eps at its lower limit, gradients whose squares are denormal or vanish: the update divides by the root of the held v, not by
    eps alone.  v / (1 - b2^t) is rounded to a multiple of 2^-149 there, off by 2^-150, which the root passes on by half."""
    g = torch.from_numpy((10.0 ** np.linspace(-24, -16, 256)).astype(np.float32)).cuda()
    opt = optim.AdamW([torch.zeros(256, device='cuda')], lr=1.0, weight_decay=0.0, states=states, eps=1e-30)
    for t in range(1, 4):
        before, p0 = held(opt)[0], f64(opt.params[0])
        opt.step([g])
        m, v = O.moments(before[0], before[1], f32(g), np.float32(1.0), *opt.betas)
        m, v = m.astype(np.float64), v.astype(np.float64)
        x = v / (1 - 0.999 ** t)
        u = (m / (1 - 0.9 ** t)) / (np.sqrt(x) + opt.eps)
        want = p0 - u
        tol = 4 * 2.0 ** -24 * np.abs(p0) + (10 * 2.0 ** -23 + 2.0 ** -150 / np.maximum(x, 2.0 ** -149)) * np.abs(u) + 2.0 ** -150 / opt.eps
        assert (np.abs(f64(opt.params[0]) - want) <= tol).all(), np.abs(f64(opt.params[0]) - want).max()
