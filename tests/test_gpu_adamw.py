"""The AdamW step on the GPU against its formula in float64.

Tolerances, e = 2^-24. 32-bit states: m = fma(b1, m, c1 g) with rounded b1, c1 and (clipped) g: 4 e of the sum of the
terms' sizes covers it; v has g twice more: 6 e. q = m / bc1 / (sqrt(v / bc2) + eps): its numerator carries m's error and
2 e, its denominator half of v's error and 3 e, the division e: |dq| <= dm / (bc1 den) + 10 e |q|. p -= lr (q + wd p):
lr (dq + 3 e (|q| + |wd p|)) and the last rounding, e |p|. 8-bit states: scales and codes are formed in 64 bits and have
to be equal; m and v enter q rounded to f32 (2 e)."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
E = 2.0 ** -24
LR, WD, B1, B2, EPS = 1e-2, 0.1, 0.9, 0.999, 1e-7
SIZES = [[1], [127], [128], [129], [4096], [4097, 3, 1, 640], [5, 12289, 2, 2, 255, 33]]


@pytest.fixture(autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.fail("needs a GPU")


def _adamw(**kw):
    from realtime_style_transfer_amd.optimizers import AdamW
    return AdamW(**{**dict(learning_rate=LR, weight_decay=WD, beta_1=B1, beta_2=B2, epsilon=EPS), **kw})


def _make(sizes, seed=0, gap=0):
    """Variables with odd starts inside one buffer, their gradients' bucket, which of them decay."""
    rng = np.random.default_rng(seed)
    n = sum(sizes)
    flat = torch.from_numpy(rng.standard_normal(n + 1).astype(np.float32)).cuda()[1:]
    grad = torch.from_numpy((rng.standard_normal(n) * np.exp(rng.standard_normal(n))).astype(np.float32)).cuda()
    return list(flat.split(sizes)), grad, [k % 2 == 0 for k in range(len(sizes))]


def _mix(x):
    x = x.astype(np.uint32)
    with np.errstate(over='ignore'):
        x = (x ^ (x >> np.uint32(16))) * np.uint32(0x7FEB352D)
        x = (x ^ (x >> np.uint32(15))) * np.uint32(0x846CA68B)
    return x ^ (x >> np.uint32(16))


def _spacing(y):
    return np.ldexp(1.0, np.maximum(np.frexp(np.maximum(np.abs(y), 1e-300))[1] - 1, -6) - 3)


class Reference:
    """The documented step in float64 on the host, states as the optimizer holds them."""

    def __init__(self, opt, variables, decay):
        self.sizes = [v.numel() for v in variables]
        self.bits, self.seed, self.clip = opt.state_bits, opt.seed, opt.global_clipnorm
        self.decay = np.concatenate([np.full(n, float(d)) for n, d in zip(self.sizes, decay)])
        at = np.cumsum([0] + [-(-n // 128) * 128 for n in self.sizes])
        self.place = np.concatenate([a + np.arange(n) for a, n in zip(at, self.sizes)])
        self.padded = int(at[-1])

    def read(self, opt, variables):
        f = lambda t: t.detach().float().cpu().numpy().astype(np.float64)  # noqa: E731
        s = {"p": np.concatenate([f(v).reshape(-1) for v in variables]), "m": f(opt.m), "v": f(opt.v),
             "t": opt.iterations}
        if self.bits == 8:
            s["ms"], s["vs"] = f(opt.m_scale), f(opt.v_scale)
        return s

    def step(self, s, g):
        g = g.astype(np.float64)
        norm = np.sqrt((g * g).sum())
        c = min(1.0, self.clip / norm) if self.clip else 1.0
        t = s["t"] + 1
        if self.bits == 32:
            m0, v0 = s["m"], s["v"]
        else:
            m0, v0 = ((s[k] * s[k + "s"][:, None]).reshape(-1)[self.place] for k in "mv")
        g = c * g
        m, v = B1 * m0 + (1 - B1) * g, B2 * v0 + (1 - B2) * g * g
        den = np.sqrt(v / (1 - B2 ** t)) + EPS
        q = m / (1 - B1 ** t) / den
        p = s["p"] - LR * (q + WD * self.decay * s["p"])
        size_m = B1 * np.abs(m0) + (1 - B1) * np.abs(g)
        dm = 4 * E * size_m if self.bits == 32 else 2 * E * np.abs(m)
        dq = dm / (1 - B1 ** t) / den + 10 * E * np.abs(q)
        out = {"p": p, "m": m, "v": v, "t": t, "norm": norm, "dm": dm, "dv": 6 * E * v,
               "dp": LR * (dq + 3 * E * (np.abs(q) + np.abs(WD * s["p"]))) + E * np.abs(p) + 1e-38}
        if self.bits == 8:
            full = np.zeros((2, self.padded))
            full[0, self.place], full[1, self.place] = m, v
            for k, x in zip("mv", full.reshape(2, -1, 128)):
                scale = (np.abs(x).max(1) / 448).astype(np.float32).astype(np.float64)
                y = np.divide(x, scale[:, None], where=scale[:, None] > 0, out=np.zeros_like(x))
                y = y.astype(np.float32).astype(np.float64)
                step = _spacing(y)
                if k == "m":
                    code = np.round(y / step) * step
                else:
                    with np.errstate(over='ignore'):
                        key = _mix(np.array([self.seed + t * 0x9E3779B9 & 0xFFFFFFFF]))
                        h = _mix(np.arange(self.padded // 2).astype(np.uint32) ^ key)
                    u = np.stack([h & np.uint32(0xFFFF), h >> np.uint32(16)], 1).reshape(y.shape)
                    code = np.floor(y / step + u / 65536.0) * step
                    code = np.where((x > 0) & (scale[:, None] > 0), np.maximum(code, 2.0 ** -9), code)
                out[k], out[k + "s"] = np.clip(code, -448, 448), scale
        return out


def _compare(want, got, bits):
    def near(k, tol):
        off = np.abs(got[k] - want[k]) - tol
        assert (off <= 0).all(), (k, float(off.max()), int(off.argmax()))
    near("p", want["dp"])
    assert got["t"] == want["t"]
    if bits == 32:
        near("m", want["dm"])
        near("v", want["dv"])
    else:
        for k in ("m", "v", "ms", "vs"):
            assert np.array_equal(got[k], want[k]), (k, int((got[k] != want[k]).sum()))


@pytest.mark.parametrize("clip", [None, 0.7])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("sizes", SIZES)
def test_steps(sizes, bits, dtype, clip):
    variables, _, decay = _make(sizes)
    opt = _adamw(state_bits=bits, global_clipnorm=clip, seed=3)
    opt.build(variables, decay=decay)
    ref = Reference(opt, variables, decay)
    for k in range(4):                                  # from zero states on, each step from the device's own state
        grad = (_make(sizes, seed=20 + k)[1] * (0.1 if k == 2 else 1.0)).to(dtype)
        want = ref.step(ref.read(opt, variables), grad.float().cpu().numpy())
        opt.apply_gradients(grad)
        _compare(want, ref.read(opt, variables), bits)
        if clip:
            assert abs(float(opt.global_norm) - want["norm"]) <= 2 * E * want["norm"]


@pytest.mark.parametrize("bits", [32, 8])
def test_a_large_step(bits):
    """17 M elements: past the caches, the other sizes of a workgroup's share."""
    sizes = [9, 17000003, 4097]
    variables, grad, decay = _make(sizes)
    opt = _adamw(state_bits=bits, global_clipnorm=100.0)
    opt.build(variables, decay=decay)
    ref = Reference(opt, variables, decay)
    for _ in range(2):
        want = ref.step(ref.read(opt, variables), grad.cpu().numpy())
        opt.apply_gradients(grad)
        _compare(want, ref.read(opt, variables), bits)


@pytest.mark.parametrize("bits", [32, 8])
def test_offsets_past_32_bits(bits):
    """One variable of 2^31 + 4099 elements (8.6 GB). The first step from zero states: m / bc1 = g, sqrt(v / bc2) = |g|."""
    n = 2 ** 31 + 4099
    p, step = torch.ones(n, device='cuda'), 2 ** 27
    g = torch.empty(n, dtype=torch.bfloat16, device='cuda')
    value = lambda lo, hi: ((torch.arange(lo, hi, device='cuda') % 997 - 498).float() * 1e-3).bfloat16()  # noqa: E731
    for lo in range(0, n, step):
        g[lo:lo + step] = value(lo, min(lo + step, n))
    opt = _adamw(state_bits=bits)
    opt.build([p])
    opt.apply_gradients(g)
    for lo in range(0, n, step):
        gd = value(lo, min(lo + step, n)).double()
        want = 1.0 - LR * (gd / (gd.abs() + EPS))
        assert float((p[lo:lo + step].double() - want).abs().max()) <= E + LR * 16 * E
    assert opt.iterations == 1
    if bits == 32:
        assert float((opt.m[-4099:].double() - 0.1 * g[-4099:].double()).abs().max()) <= 0.05 * 4 * E
    else:
        last = g[-3:].double()                       # the last block: three elements and zeros
        got = opt.m[-1].double() * opt.m_scale[-1].double()
        assert float((got[:3] - 0.1 * last).abs().max()) <= 2.0 ** -4 * 0.1 * float(last.abs().max())
        assert not got[3:].any() and opt.m.shape[0] == (n + 127) // 128


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("t", [10 ** 3, 10 ** 6, 2 ** 33])
def test_late_steps(bits, t):
    """Step counts far on: 1 - beta^t from expm1 in 64 bits, the count in 64."""
    variables, grad, decay = _make([700, 9])
    opt = _adamw(state_bits=bits)
    opt.build(variables, decay=decay)
    rng = np.random.default_rng(4)
    opt.set_slots([torch.from_numpy(rng.standard_normal(n)) for n in (700, 9)],
                  [torch.from_numpy(rng.random(n)) for n in (700, 9)])
    opt.iterations = t
    ref = Reference(opt, variables, decay)
    want = ref.step(ref.read(opt, variables), grad.cpu().numpy())
    opt.apply_gradients(grad)
    _compare(want, ref.read(opt, variables), bits)


@pytest.mark.parametrize("bits", [32, 8])
def test_many_variables_as_a_bucket_and_as_a_list(bits):
    """600 variables (more pointers than one launch carries): the same bits either way, and from separate tensors."""
    rng = np.random.default_rng(5)
    sizes = [int(n) for n in rng.integers(1, 300, 600)]
    variables, grad, decay = _make(sizes)
    copies = [v.clone() for v in variables]
    a, b = _adamw(state_bits=bits, global_clipnorm=1.0), _adamw(state_bits=bits, global_clipnorm=1.0)
    a.build(variables, decay=decay)
    b.build(copies, decay=decay)
    ref = Reference(a, variables, decay)
    for k in range(3):
        want = ref.step(ref.read(a, variables), grad.cpu().numpy())
        a.apply_gradients(grad)
        b.apply_gradients([g.clone() for g in grad.split(sizes)])
        _compare(want, ref.read(a, variables), bits)
        assert all(torch.equal(p, q) for p, q in zip(variables, copies))
    assert torch.equal(a.m.view(torch.uint8), b.m.view(torch.uint8))
    assert torch.equal(a.v.view(torch.uint8), b.v.view(torch.uint8))


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("bad", [float('nan'), float('inf')])
def test_a_clipped_step_with_a_bad_gradient_changes_nothing(bits, bad):
    variables, grad, decay = _make([300, 5000])
    opt = _adamw(state_bits=bits, global_clipnorm=1.0)
    opt.build(variables, decay=decay)
    opt.apply_gradients(grad)
    before = [t.clone() for t in (*variables, opt.m.view(torch.uint8), opt.v.view(torch.uint8))]
    worse = grad.clone()
    worse[4321] = bad
    opt.apply_gradients(worse)
    assert not torch.isfinite(opt.global_norm)
    assert all(torch.equal(p, q) for p, q in zip(before, (*variables, opt.m.view(torch.uint8), opt.v.view(torch.uint8))))
    assert opt.iterations == 1
    opt.apply_gradients(grad)                            # and the next one goes on
    assert opt.iterations == 2 and torch.isfinite(opt.global_norm)


@pytest.mark.parametrize("bits", [32, 8])
def test_zero_gradients_and_decay_alone(bits):
    variables, grad, decay = _make([640, 130])
    opt = _adamw(state_bits=bits, global_clipnorm=1.0)
    opt.build(variables, decay=decay)
    before = [v.clone() for v in variables]
    opt.apply_gradients(torch.zeros_like(grad))
    assert torch.equal(variables[1], before[1])          # no decay: untouched, no 0 / 0
    off = (variables[0].double() - before[0].double() * (1 - LR * WD)).abs()
    assert bool((off <= 3 * E * before[0].abs()).all())
    assert not opt.m.float().any() and not opt.v.float().any() and float(opt.global_norm) == 0.0


def test_second_moments_of_8_bits_follow_the_mean():
    """The random rounding: after 1500 steps of gradients of constant size the mean of v over many elements is the
    formula's g^2 (1 - b2^t) to 2 %; rounded to nearest it would stay near its first few steps' values (about
    16 of 1000 ways up). Noise: a step's rounding has a variance of about 1e-3 v^2 / 12, kept for 1 / (2 (1 - b2))
    steps: 0.2 of v, over 32768 elements 0.1 %; each block's largest element alone (1 of 128) is not rounded."""
    n, g = 32768, 0.25
    p = torch.zeros(n, device='cuda')
    opt = _adamw(state_bits=8, weight_decay=0.0)
    opt.build([p])
    rng = torch.Generator().manual_seed(0)
    sign = [(torch.randint(0, 2, (n,), generator=rng).float() * 2 - 1).cuda() * g for _ in range(8)]
    size = torch.where(torch.arange(n, device='cuda') % 128 == 0, 4.0, 1.0)     # the block's largest sets the scale
    for k in range(1500):
        opt.apply_gradients(sign[k % 8] * size)
    v = opt.slots()[1][0]
    want = g * g * (1 - B2 ** 1500)
    got = float(v[size == 1.0].double().mean())
    assert abs(got / want - 1) < 0.02, (got, want)


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_steps_count_on(bits):
    """Replays are steps of their own (bias corrections, random bits), with eager steps between them."""
    variables, grad, decay = _make([1000, 77, 4500])
    copies = [v.clone() for v in variables]
    a, b = (_adamw(state_bits=bits, global_clipnorm=1.0) for _ in range(2))
    a.build(variables, decay=decay)
    b.build(copies, decay=decay)
    parts = list(grad.split([1000, 77, 4500]))
    a.apply_gradients(grad)
    torch.cuda.synchronize()
    bucket, tensors = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(bucket):
        a.apply_gradients(grad)
    with torch.cuda.graph(tensors):
        a.apply_gradients(parts)
    for g in (bucket, None, tensors, bucket, None, bucket, tensors):
        g.replay() if g is not None else a.apply_gradients(grad)
        torch.cuda.synchronize()
    for _ in range(8):
        b.apply_gradients(grad)
    assert a.iterations == b.iterations == 8
    assert all(torch.equal(p, q) for p, q in zip(variables, copies))
    assert torch.equal(a.v.view(torch.uint8), b.v.view(torch.uint8))


def test_two_optimizers_on_two_streams():
    made = [_make([5000, 12, 900], seed=k) for k in (1, 2)]
    want = []
    for variables, grad, decay in made:
        c = [v.clone() for v in variables]
        opt = _adamw(state_bits=8, global_clipnorm=1.0)
        opt.build(c, decay=decay)
        for _ in range(5):
            opt.apply_gradients(grad)
        want.append(c)
    opts = []
    for variables, _, decay in made:
        opts.append(_adamw(state_bits=8, global_clipnorm=1.0))
        opts[-1].build(variables, decay=decay)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        for opt, st, (_, grad, _) in zip(opts, streams, made):
            with torch.cuda.stream(st):
                opt.apply_gradients(grad)
    torch.cuda.synchronize()
    for c, (variables, _, _) in zip(want, made):
        assert all(torch.equal(p, q) for p, q in zip(c, variables))


@pytest.mark.parametrize("bits", [32, 8])
def test_slots_round_trip(bits):
    sizes = [300, 7, 128]
    variables, grad, decay = _make(sizes)
    opt = _adamw(state_bits=bits)
    opt.build(variables, decay=decay)
    for _ in range(3):
        opt.apply_gradients(grad)
    m, v = opt.slots()
    other = _adamw(state_bits=bits)
    other.build([t.clone() for t in variables], decay=decay)
    other.set_slots([t.view(-1, 1) for t in m], v)
    m2, v2 = other.slots()
    if bits == 32:
        assert all(torch.equal(p, q) for p, q in zip(m + v, m2 + v2))
    else:
        # the same codes, with a scale that went through fl(fl(448 s) / 448): a slot, fl(code s), moves by 4 e at most
        assert torch.equal(opt.m.view(torch.uint8), other.m.view(torch.uint8))
        assert all(bool(((p - q).abs() <= 4 * E * p.abs()).all()) for p, q in zip(m, m2))
        # a block's largest v may have been rounded down, which moves the new scale by a code's step
        assert all(bool(((p - q).abs() <= 2.0 ** -4 * p + 1e-30).all()) for p, q in zip(v, v2))
    with pytest.raises(ValueError):
        other.set_slots(m[:2], v[:2])


def test_refusals_on_the_device():
    from realtime_style_transfer_amd import _lib as L
    variables, grad, _ = _make([10, 20])
    opt = _adamw()
    with pytest.raises(ValueError):
        opt.build([variables[0], variables[1].double()])
    with pytest.raises(ValueError):
        opt.build([variables[0], variables[1].view(4, 5).t()])
    opt.build(variables)
    with pytest.raises(ValueError, match="already has variables"):
        opt.build(variables)
    for bad in (grad[:-1], grad.double(), grad.cpu(), torch.cat([grad, grad])[::2], [grad[:10]], [grad[:10], None],
                [grad[:10], grad[10:].bfloat16()], [grad[:10], grad[:10]]):
        with pytest.raises(ValueError):
            opt.apply_gradients(bad)
    opt.beta_1 = 1.5
    with pytest.raises(ValueError):
        opt.apply_gradients(grad)
    assert opt.iterations == 0
    with pytest.raises(ValueError):
        opt.iterations = -1
    assert L.load().rst_adamw_num_blocks(opt._handle) == 2


def test_trains_a_normalised_layer():
    """Forward, gradients and step together, as a training loop runs them: three steps of the affine and the input of a
    group norm against the same loop in float64 (autograd, the formula). Each step's loss is the same to 1e-5 of its
    size, as 32-bit outputs with 64-bit statistics keep it; Adam's first steps divide by |g|, so that an element whose
    gradient is lost in rounding may go either way: variables are compared where |g| is not below 1e-3 of its rms."""
    from realtime_style_transfer_amd.styleTransfer import group_norm, group_norm_gradients
    g = torch.Generator().manual_seed(1)
    shape, G = (2, 12, 10, 32), 8
    x, scale, bias = (torch.randn(shape, generator=g).cuda(), 1 + 0.1 * torch.randn(32, generator=g).cuda(),
                      torch.randn(32, generator=g).cuda())
    target = torch.randn(shape, generator=g).cuda()
    ref = [t.double().clone() for t in (x, scale, bias)]
    state = [(torch.zeros_like(t), torch.zeros_like(t)) for t in ref]
    solid = [torch.ones_like(t, dtype=torch.bool) for t in ref]
    bucket = torch.empty(x.numel() + 64, device='cuda')
    opt = _adamw(global_clipnorm=5.0)
    opt.build([x, scale, bias], decay=[False, True, False])
    for t in range(1, 4):
        y, mean, rstd = group_norm(x, scale, bias, G, activation="swish", return_statistics=True)
        grads = group_norm_gradients(x, y - target, scale, bias, mean, rstd, G, activation="swish")
        torch.cat([d.reshape(-1) for d in grads], out=bucket)
        opt.apply_gradients(bucket)
        leaves = [t_.clone().requires_grad_() for t_ in ref]
        r = leaves[0].reshape(2, 120, G, 4)
        z = ((r - r.mean((1, 3), keepdim=True)) * (r.var((1, 3), unbiased=False, keepdim=True) + 1e-5).rsqrt()) \
            .reshape(shape) * leaves[1] + leaves[2]
        loss = 0.5 * ((z * torch.sigmoid(z) - target) ** 2).sum()
        loss.backward()
        loss = float(loss.detach())
        mine = 0.5 * float(((y.double() - target) ** 2).sum())
        assert abs(mine - loss) < 1e-5 * loss + (t > 1) * 1e-4 * loss
        norm = torch.sqrt(sum((l.grad ** 2).sum() for l in leaves))
        c = min(1.0, 5.0 / float(norm))
        for k, leaf in enumerate(leaves):
            m, v = state[k]
            gk = c * leaf.grad
            solid[k] &= gk.abs() > 1e-3 * gk.norm() / gk.numel() ** 0.5
            m.mul_(B1).add_((1 - B1) * gk)
            v.mul_(B2).add_((1 - B2) * gk * gk)
            ref[k] = ref[k] - LR * (m / (1 - B1 ** t) / (torch.sqrt(v / (1 - B2 ** t)) + EPS) + (WD if k == 1 else 0) * ref[k])
    for mine, want, at in zip((x, scale, bias), ref, solid):
        assert float(at.float().mean()) > 0.9
        assert float((mine.double() - want)[at].abs().max()) < 1e-2 * 3 * LR


def _training_model(optimizer, seed=2):
    from realtime_style_transfer_amd.stylePrediction import StylePredictionTrainer
    from realtime_style_transfer_amd.plan import network_plan
    from realtime_style_transfer_amd.styleTransferTrainingModel import StyleTransferTrainingModel
    ins, outs, br, bf = (32, 64, 17), (32, 64, 3), 8, 8
    P = network_plan(ins, outs, br, bf).num_style_params
    pr = StylePredictionTrainer((32, 64, 3), "MOBILE_NET", P, max_batch=2)
    return StyleTransferTrainingModel(ins, outs, br, bf, max_batch=2, seed=seed, style_predictor=pr,
                                      optimizer=optimizer)


def _batch(seed=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.rand(*s, generator=g).cuda()  # noqa: E731
    return ({'content': r(2, 32, 64, 17), 'style': r(2, 1, 32, 64, 3)},
            {'content': r(2, 32, 64, 3), 'style': r(2, 1, 32, 64, 3)})


@pytest.mark.parametrize("bits", [32, 8])
def test_training_model_steps_both_networks(bits):
    """compile(optimizer=AdamW): every trainable weight of the transfer network and the predictor takes the formula's
    step from the gradient bucket (one norm over both), kernels alone decay, BN moving statistics are left to the
    forward, and the transfer network's kernel images follow."""
    opt = _adamw(learning_rate=LR, global_clipnorm=1.0, state_bits=bits)
    tr = _training_model(None)
    tr.compile(optimizer=opt)
    pr = tr.style_predictor
    from realtime_style_transfer_amd.stylePrediction import trainable_mask
    mask = [not k for k in _moving(tr)] + list(trainable_mask(pr.spec))
    before = tr.get_weights() + pr.get_weights()
    x, y = _batch()
    tr.train_step(x, y)
    after = tr.get_weights() + pr.get_weights()
    flat = tr._grad_bucket.double().cpu().numpy()
    norm = np.sqrt((flat ** 2).sum())
    c, o = min(1.0, 1.0 / norm), 0
    assert abs(float(opt.global_norm) / norm - 1) < 1e-6
    for w0, w1, train in zip(before, after, mask):
        g = c * flat[o:o + w0.size].reshape(w0.shape)
        o += w0.size
        if not train:
            assert not g.any()
            continue
        q = g / (np.abs(g) + EPS)           # the first step: m / bc1 = g, sqrt(v / bc2) = |g|
        want = w0 - LR * (q + (WD if w0.ndim > 1 else 0.0) * w0.astype(np.float64))
        tol = LR * 16 * E * (np.abs(q) + 1) + 2 * E * np.abs(want)
        assert (np.abs(w1 - want) <= tol).all(), float((np.abs(w1 - want) - tol).max())
    assert o == flat.size and opt.iterations == tr.iterations == pr.iterations == 1
    # a model made anew from these weights gives the same losses: the kernels' images were re-packed
    other = _training_model(_adamw())
    other.set_weights(tr.get_weights())
    pr2 = other.style_predictor
    pr2.set_weights(pr.get_weights())
    for m in (tr, other):
        m.train_step(x, y)
    assert torch.equal(tr.style_losses['loss'], other.style_losses['loss'])


def _moving(tr):
    out = []
    for layer in tr.plan.layers:
        out += [False, False] + ([False, False, True, True] if layer.norm == 'bn' else [])
    return out


@pytest.mark.parametrize("bits", [32, 8])
def test_training_checkpoint_restores_the_moments(bits, tmp_path):
    x, y = _batch()
    a = _training_model(_adamw(state_bits=bits))
    for _ in range(3):
        a.train_step(x, y)
    a.save_weights(str(tmp_path / "ck"))
    a.optimizer.learning_rate = 5e-3
    a.save_weights(str(tmp_path / "ck"))
    b = _training_model(_adamw(state_bits=bits), seed=5)
    b.load_weights(str(tmp_path / "ck")).assert_nontrivial_match()
    assert b.iterations == b.optimizer.iterations == 3 and abs(b.optimizer.learning_rate - 5e-3) < 1e-9
    for p, q in zip(a.optimizer.slots()[0], b.optimizer.slots()[0]):      # 4 e: test_slots_round_trip
        assert torch.equal(p, q) if bits == 32 else bool(((p - q).abs() <= 4 * E * p.abs()).all())
    for p, q in zip(a.optimizer.slots()[1], b.optimizer.slots()[1]):
        assert torch.equal(p, q) if bits == 32 else bool(((p - q).abs() <= 2.0 ** -4 * p + 1e-30).all())
    if bits == 32:
        for m in (a, b):
            m.train_step(x, y)
        assert all(np.array_equal(p, q) for p, q in zip(a.get_weights(), b.get_weights()))
    # the moments are no RMSprop state: restored into an RMSprop model they are reported unused
    from realtime_style_transfer_amd.styleTransferTrainingModel import RMSprop
    c = _training_model(RMSprop())
    status = c.load_weights(str(tmp_path / "ck"))
    with pytest.raises(AssertionError):
        status.assert_consumed()


def test_training_model_refusals():
    tr = _training_model(_adamw())
    with pytest.raises(ValueError, match="train_step"):
        tr.apply_gradients(tr._grad)
    with pytest.raises(ValueError, match="already has variables"):
        _training_model(tr.optimizer)
    with pytest.raises(TypeError):
        tr.compile(optimizer=torch.optim.SGD([torch.zeros(1, requires_grad=True)], 0.1))
    with pytest.raises(ValueError, match="optimizer_slots"):
        tr.optimizer_slots()
    opt = tr.optimizer
    size = opt._bucket_size
    del tr
    import gc
    gc.collect()
    with pytest.raises(ValueError, match="no longer exists"):
        opt.apply_gradients(torch.zeros(size, device='cuda'))


def _bytes(opt):
    return [t.reshape(-1).view(torch.uint8) for t in (opt.m, opt.v, *((opt.m_scale, opt.v_scale) if opt.m_scale is not None else ()))]


@pytest.mark.parametrize("bits", [32, 8])
def test_without_clipping_a_bad_gradient_stays_with_its_element(bits):
    """Against the same steps with zeros in its place: no other element, code or scale differs (a bad moment counts for no
    scale, as a zero)."""
    (a, grad, decay), (b, _, _) = _make([300, 5000]), _make([300, 5000])
    at = torch.tensor([0, 17, 299, 300 + 1234, 300 + 4999], device='cuda')
    bad = torch.tensor([float('nan'), float('inf'), -float('inf'), float('inf'), float('nan')], device='cuda')
    x, y = _adamw(state_bits=bits, seed=5), _adamw(state_bits=bits, seed=5)
    x.build(a, decay=decay)
    y.build(b, decay=decay)
    for k in range(3):
        g = _make([300, 5000], seed=30 + k)[1]
        x.apply_gradients(g.index_copy(0, at, bad) if k == 0 else g)
        y.apply_gradients(g.index_fill(0, at, 0.0))
    other = torch.ones(5300, dtype=torch.bool, device='cuda')
    other[at] = False
    for p, q in ((torch.cat(a), torch.cat(b)), *zip(map(torch.cat, x.slots()), map(torch.cat, y.slots()))):
        assert torch.equal(p[other], q[other])
    assert bool(torch.cat(a)[at].isnan().all())
    assert bits == 32 or all(bool(torch.cat(s)[at].isnan().all()) for s in x.slots())


def test_a_gradient_past_8_bits_saturates():
    """(1 - b2) g^2 beyond 448 times the largest f32: v is that number, and nothing is NaN."""
    variables, grad, decay = _make([256])
    opt = _adamw(state_bits=8)
    opt.build(variables, decay=decay)
    grad[5] = -1e30
    for _ in range(2):
        opt.apply_gradients(grad)
        assert bool(variables[0].isfinite().all()) and bool(opt.m.float().isfinite().all())
        assert float(opt.v_scale[0]) == torch.finfo(torch.float32).max and float(opt.v.float()[0, 5]) == 448.0
        assert float(opt.m.float()[0, 5]) == -448.0 and float(opt.v_scale[1]) < 1.0


def test_slots_with_bad_values_and_tiny_blocks():
    variables, grad, decay = _make([256, 128])
    opt = _adamw(state_bits=8)
    opt.build(variables, decay=decay)
    m, v = [torch.randn(256), torch.full((128,), 1e-37)], [torch.rand(256) + 0.1, torch.full((128,), 1e-37)]
    for t in (m[0], v[0]):
        t[3], t[200] = float('nan'), float('inf')
    opt.set_slots(m, v)
    assert opt.m_scale[2] == 0 and opt.v_scale[2] == 0           # 1e-37 / 448 is below 2^-126: zeros
    for want, got in zip((m, v), opt.slots()):
        ok = want[0].isfinite()
        assert bool(got[0].cpu()[~ok].isnan().all()) and not got[1].any()
        # a code is within 2^-4 of its value, or half of the smallest, max / 448 2^-10 (v: all of it, 2^-9)
        off = (got[0].cpu() - want[0]).abs()[ok]
        assert bool((off <= (2.0 ** -4 + 4 * E) * want[0].abs()[ok] + 5 / 448 * 2.0 ** -9).all())
    before = _bytes(opt)[0].clone()
    with pytest.raises(ValueError, match="do not match"):
        opt.set_slots([t + 1 for t in m], v[:1])
    assert torch.equal(_bytes(opt)[0], before)                   # nothing is set by halves


@pytest.mark.parametrize("bits", [32, 8])
def test_empty_variables_among_others(bits):
    import ctypes
    from realtime_style_transfer_amd import _lib as L
    sizes = [0, 5, 0, 130, 0]
    (a, grad, decay), (b, _, _) = _make([5, 130]), _make([5, 130])
    empty = torch.empty(0, device='cuda')
    x, y = _adamw(state_bits=bits, global_clipnorm=1.0), _adamw(state_bits=bits, global_clipnorm=1.0)
    x.build([empty, a[0], empty, a[1], empty], decay=[True, decay[0], True, decay[1], False])
    y.build(b, decay=decay)
    x.apply_gradients(grad)
    x.apply_gradients(list(grad.split(sizes)))
    for _ in range(2):
        y.apply_gradients(grad)
    assert all(torch.equal(p, q) for p, q in zip(a, b)) and x.iterations == 2
    assert [t.numel() for t in x.slots()[0]] == sizes
    pointers = (ctypes.c_void_p * 5)(None, grad.data_ptr(), None, None, None)      # the fourth one's is missing
    rc = L.load().rst_adamw_step_tensors(x._handle, pointers, 5, 0, ctypes.byref(x._check_config()), L.stream_ptr())
    assert rc == L.RST_ERR_INVALID and x.iterations == 2


def test_memory_stays_when_its_names_are_given_away():
    variables, grad, decay = _make([300])
    opt = _adamw()
    opt.build(variables, decay=decay)
    v = variables[0]
    v.data, opt.m, opt.v = torch.zeros(300, device='cuda'), None, None
    variables.clear()
    torch.cuda.empty_cache()
    opt.apply_gradients(grad)
    assert not v.any() and opt.iterations == 1


def test_a_models_optimizer_steps_with_the_model_alone():
    from realtime_style_transfer_amd.styleTransferTrainingModel import RMSprop
    tr, (x, y) = _training_model(_adamw()), _batch()
    opt = tr.optimizer
    with pytest.raises(ValueError, match="train_step"):
        opt.apply_gradients(tr._grad_bucket)               # the kernels' weight images would not follow
    tr.train_step(x, y)
    tr.compile(optimizer=RMSprop(learning_rate=1e-3))
    tr.train_step(x, y)
    assert opt.iterations == 1 and len(tr.optimizer_slots()) == len(tr.get_weights())
    tr.compile(optimizer=opt)                              # its own AdamW again, with its moments
    tr.train_step(x, y)
    assert opt.iterations == 2 and tr.iterations == 3


def test_training_model_without_a_predictor(tmp_path):
    from realtime_style_transfer_amd.plan import network_plan, synthetic_style_params
    from realtime_style_transfer_amd.styleTransferTrainingModel import StyleTransferTrainingModel
    ins, outs, br, bf = (32, 64, 17), (32, 64, 3), 8, 8
    plan = network_plan(ins, outs, br, bf)
    x, y = _batch()
    x = {'content': x['content'],
         'style_params': torch.from_numpy(synthetic_style_params(2, 1, plan.num_style_params, plan, seed=1)).cuda()}
    models = [StyleTransferTrainingModel(ins, outs, br, bf, max_batch=2, seed=s, optimizer=_adamw(global_clipnorm=1.0))
              for s in (2, 3)]
    models[0].train_step(x, y)
    models[0].save_weights(str(tmp_path / "ck"))
    models[1].load_weights(str(tmp_path / "ck")).assert_nontrivial_match()
    for m in models:
        m.train_step(x, y)
    a, b = (np.concatenate([w.ravel() for w in m.get_weights()]) for m in models)
    assert np.array_equal(a, b) and models[1].optimizer.iterations == 2


def test_rmsprop_checkpoint_gives_an_adamw_model_its_weights_alone(tmp_path):
    from realtime_style_transfer_amd.styleTransferTrainingModel import RMSprop
    x, y = _batch()
    a, b = _training_model(RMSprop()), _training_model(_adamw(), seed=5)
    a.train_step(x, y)
    a.save_weights(str(tmp_path / "ck"))
    status = b.load_weights(str(tmp_path / "ck"))
    with pytest.raises(AssertionError):
        status.assert_consumed()
    assert all(np.array_equal(p, q) for p, q in zip(a.get_weights(), b.get_weights()))
    assert b.optimizer.iterations == 0 and b.optimizer.learning_rate == LR
    assert not any(t.any() for t in b.optimizer.slots()[0])


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_training_step_replays_as_the_next_one(bits):
    a, b = (_training_model(_adamw(state_bits=bits, global_clipnorm=1.0)) for _ in range(2))
    x, y = _batch()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a.train_step(x, y)
        b.train_step(x, y)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        b.train_step(x, y)
    for k in range(3):
        a.train_step(x, y)
        g.replay()
        torch.cuda.synchronize()
        wa, wb = (np.concatenate([q.ravel() for q in m.get_weights() + m.style_predictor.get_weights()]) for m in (a, b))
        assert np.array_equal(wa, wb) and a.optimizer.iterations == b.optimizer.iterations == k + 2
        assert torch.equal(a.style_losses['loss'], b.style_losses['loss'])


def _rank(rank, world, port, tmp):
    import os
    import torch.distributed as dist
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    torch.cuda.set_device(0)
    dist.init_process_group("gloo", rank=rank, world_size=world)
    try:
        tr = _training_model(_adamw(state_bits=8, global_clipnorm=1.0))
        x, y = _batch(seed=100 + rank)
        for _ in range(2):
            tr.train_step(x, y)
        w = np.concatenate([q.ravel() for q in tr.get_weights() + tr.style_predictor.get_weights()])
        np.save(os.path.join(tmp, f"w{rank}.npy"), np.append(w, float(tr.optimizer.global_norm)))
    finally:
        dist.destroy_process_group()


def test_ranks_stay_identical(tmp_path):
    import torch.multiprocessing as mp
    from realtime_style_transfer_amd.frames import free_port
    mp.spawn(_rank, args=(2, free_port(), str(tmp_path)), nprocs=2, join=True)
    a, b = (np.load(tmp_path / f"w{r}.npy") for r in range(2))
    assert np.array_equal(a, b) and np.isfinite(a).all()


@pytest.mark.parametrize("bits", [32, 8])
def test_the_smallest_epsilon(bits):
    """2^-126: an element without a gradient stays, the others step by their size; below it the C entry refuses, as for
    the other hyperparameters past 32 bits."""
    import ctypes
    from realtime_style_transfer_amd import _lib as L
    variables, grad, decay = _make([300, 5])
    opt = _adamw(state_bits=bits, epsilon=2.0 ** -126, weight_decay=0.0)
    opt.build(variables, decay=decay)
    grad[:130] = 0.0
    before = torch.cat(variables).double()
    opt.apply_gradients(grad)
    after = torch.cat(variables).double()
    assert bool(((after - (before - LR * grad.sign())).abs() <= LR * 16 * E + E * after.abs()).all())
    lib, kept = L.load(), after.clone()
    for change in (dict(epsilon=2.0 ** -127), dict(epsilon=1e-50), dict(epsilon=1e39), dict(learning_rate=1e39), dict(weight_decay=-1e39)):
        c = dict(learning_rate=LR, weight_decay=WD, beta_1=B1, beta_2=B2, epsilon=EPS, global_clipnorm=0.0, seed=0)
        cfg = L.RstAdamwConfig(*{**c, **change}.values())
        assert lib.rst_adamw_step(opt._handle, grad.data_ptr(), 0, ctypes.byref(cfg), L.stream_ptr()) == L.RST_ERR_INVALID
    assert opt.iterations == 1 and torch.equal(torch.cat(variables).double(), kept)


@pytest.mark.parametrize("bits", [32, 8])
def test_large_gradients_step_by_the_formula(bits):
    """v / bc2 past f32's range, and with 8-bit states v itself: the root is still inside. (32-bit states hold g up to
    sqrt(max / (1 - b2)) = 5.8e20.)"""
    sizes = [256, 384, 130]
    variables, grad, decay = _make(sizes)
    size = torch.logspace(5, 20 if bits == 32 else 37, 770, dtype=torch.float64).float().cuda()
    grad = grad.sign() * size
    opt = _adamw(state_bits=bits)
    opt.build(variables, decay=decay)
    ref = Reference(opt, variables, decay)
    for _ in range(3):
        want = ref.step(ref.read(opt, variables), grad.cpu().numpy())
        opt.apply_gradients(grad)
        off = np.abs(ref.read(opt, variables)["p"] - want["p"]) - want["dp"]
        assert (off <= 0).all(), (float(off.max()), int(off.argmax()))


def test_tiny_second_moments():
    """A v below f32's normal numbers still divides by its root (epsilon 1e-30 beside roots of 1e-20 to 1e-17). One step from
    given moments with a gradient of 0. v carries half a step of the subnormals, 2^-150, beside its 6 e: half of that,
    relative to v, is its root's."""
    n = 512
    p, g = torch.zeros(n, device='cuda'), torch.zeros(n, device='cuda')
    opt = _adamw(epsilon=1e-30)
    opt.build([p])
    v = torch.logspace(-40, -34, n, dtype=torch.float64).float()
    m = 0.5 * v.double().sqrt().float() * (1 - 2 * (torch.arange(n) % 2))
    opt.set_slots([m], [v])
    opt.iterations = 1000
    opt.apply_gradients(g)
    v1 = B2 * v.double()
    q = B1 * m.double() / (1 - B1 ** 1001) / (torch.sqrt(v1 / (1 - B2 ** 1001)) + 1e-30)
    tol = LR * q.abs() * (17 * E + 2.0 ** -150 / v1)
    off = (p.cpu().double() + LR * q).abs() - tol
    assert bool((off <= 0).all()), (float(off.max()), int(off.argmax()))


def test_a_second_moment_past_32_bits():
    """32-bit states: a v past f32 is infinite, its element decays and takes no step from there on; no other element differs."""
    (a, grad, decay), (b, _, _) = _make([300, 70]), _make([300, 70])
    decay = [True, False]
    x, y = _adamw(), _adamw()
    x.build(a, decay=decay)
    y.build(b, decay=decay)
    at = torch.tensor([11, 299, 300 + 64], device='cuda')
    before = torch.cat(a)[at].double()
    for k in range(2):
        x.apply_gradients(grad.index_copy(0, at, torch.tensor([1e30, -3e38, 1e25], device='cuda')) if k == 0 else grad)
        y.apply_gradients(grad)
    other = torch.ones(370, dtype=torch.bool, device='cuda')
    other[at] = False
    assert torch.equal(torch.cat(a)[other], torch.cat(b)[other]) and bool(x.v[at].isinf().all())
    want = before * torch.tensor([(1 - LR * WD) ** 2, (1 - LR * WD) ** 2, 1.0], device='cuda')
    assert bool(((torch.cat(a)[at].double() - want).abs() <= 8 * E * before.abs()).all())


def test_adamw_checkpoint_gives_an_rmsprop_model_its_weights_alone(tmp_path):
    """Its learning rate and step count go with its moments: none is taken over, and all are reported unused."""
    from realtime_style_transfer_amd.styleTransferTrainingModel import RMSprop
    x, y = _batch()
    a, b = _training_model(_adamw()), _training_model(RMSprop(learning_rate=2e-3, rho=0.8), seed=5)
    for _ in range(3):
        a.train_step(x, y)
    a.save_weights(str(tmp_path / "ck"))
    status = b.load_weights(str(tmp_path / "ck"))
    names = ("iter", "learning_rate", "weight_decay", "beta_1", "beta_2")
    assert all(any(k.startswith(f"optimizer/{n}/") for k in status.unused) for n in names)
    assert all(np.array_equal(p, q) for p, q in zip(a.get_weights(), b.get_weights()))
    assert (b.optimizer.learning_rate, b.optimizer.rho) == (2e-3, 0.8)
    assert b.iterations == b.style_predictor.iterations == 0
    assert not any(s.any() for s in b.optimizer_slots())
    b.train_step(x, y)
    b.save_weights(str(tmp_path / "rms"))                # and an RMSprop checkpoint restores as before
    c = _training_model(RMSprop())
    c.load_weights(str(tmp_path / "rms")).assert_consumed()
    assert c.iterations == 1 and abs(c.optimizer.learning_rate - 2e-3) < 1e-9 and abs(c.optimizer.rho - 0.8) < 1e-7


def test_autograd_sees_a_step():
    """Variables that a forward has saved are changed by the step: their backward is refused, as after any other change in
    place."""
    w = torch.randn(5, 4, device='cuda', requires_grad=True)
    b = torch.randn(4, device='cuda', requires_grad=True)
    x = torch.randn(3, 5, device='cuda', requires_grad=True)
    with torch.inference_mode():
        frozen = torch.ones(3, device='cuda')            # (has no version)
    buffer = torch.ones(9, device='cuda')
    opt = _adamw()
    opt.build([w, b, frozen, *buffer.split([2, 7])])
    loss = (x @ w + b).square().sum()
    versions = [t._version for t in (w, b, buffer)]
    opt.apply_gradients(torch.ones(36, device='cuda'))
    assert all(t._version > n for t, n in zip((w, b, buffer), versions))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    (x @ w + b).square().sum().backward()
    opt.apply_gradients([w.grad, b.grad, torch.zeros(3, device='cuda'), buffer[:2], buffer[2:]])
    assert opt.iterations == 2


def test_checkpoint_keeps_the_hyperparameters_bits(tmp_path):
    """In 32 bits a scheduled learning rate would come back rounded, and a beta_2 next to 1 as 1, which no step takes."""
    x, y = _batch()
    a = _training_model(_adamw(learning_rate=1e-3 / 3, weight_decay=0.1 / 7, beta_1=0.9 + 1e-9, beta_2=1 - 1e-9))
    a.train_step(x, y)
    a.save_weights(str(tmp_path / "ck"))
    b = _training_model(_adamw(), seed=5)
    b.load_weights(str(tmp_path / "ck"))
    names = ('learning_rate', 'weight_decay', 'beta_1', 'beta_2')
    assert [getattr(a.optimizer, n) for n in names] == [getattr(b.optimizer, n) for n in names]
    for m in (a, b):
        m.train_step(x, y)
    assert all(np.array_equal(p, q) for p, q in zip(a.get_weights(), b.get_weights()))
    tensors = {k: np.float32(v) if v.dtype == np.float64 else v for k, v in a._checkpoint_tensors().items()}
    tensors = {k: np.float32(0.999) if k.startswith('optimizer/beta_2') else v for k, v in tensors.items()}
    b._restore_tensors(tensors)                          # 32-bit variables: their shortest decimal
    assert b.optimizer.beta_2 == 0.999 and abs(b.optimizer.learning_rate / (1e-3 / 3) - 1) < 2.0 ** -24


def test_slots_of_saturated_states_are_finite():
    """448 times a scale can be past f32: a slot is its largest number then, and restored it is no infinity."""
    (variables, grad, decay), top = _make([256]), torch.finfo(torch.float32).max
    opt, other = _adamw(state_bits=8), _adamw(state_bits=8)
    opt.build(variables, decay=decay)
    other.build([v.clone() for v in variables], decay=decay)
    grad[5], grad[9], grad[200] = -1e30, 1e25, float('nan')
    opt.apply_gradients(grad)
    m, v = opt.slots()
    assert float(v[0][5]) == float(v[0][9]) == top and bool(v[0][200].isnan())
    other.set_slots(m, v)
    other.iterations = 1
    assert float(other.slots()[1][0][5]) == top
    for o in (opt, other):
        o.apply_gradients(torch.zeros_like(grad))
    finite = torch.arange(256, device='cuda') != 200
    assert bool(other.slots()[1][0][finite].isfinite().all()) and bool(other._variables[0][finite].isfinite().all())
