"""Linear cross entropy and its gradient on the GPU against their definitions in 64 bits."""
import pytest
import torch

import hiptensor_b200 as ht
import training_helpers as ref

pytestmark = pytest.mark.gpu
KIND = {v: k for k, v in ref.TYPES.items()}
IGNORE = -100


@pytest.fixture(scope="module")
def h():
    return ht.Handle()


def desc(h, x):
    return h.tensor_descriptor(x.shape, x.stride(), KIND[x.dtype])


def inputs(t, v, d, kind, seed=5, ignored=0.2, ldpad=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    H = torch.randn(t, d + ldpad, generator=g, device="cuda").to(kind)[:, :d]
    W = (torch.randn(v, d + ldpad, generator=g, device="cuda") * 2 / d ** 0.5).to(kind)[:, :d]
    y = torch.randint(0, v, (t,), generator=g, device="cuda")
    y[torch.rand(t, generator=g, device="cuda") < ignored] = IGNORE
    gl = torch.rand(t, generator=g, device="cuda") * (100.0 if kind == torch.float16 else 1.0) / t
    return H, W, y, gl


class Call:
    """One plan with its buffers, forward and backward."""

    def __init__(self, h, H, W, y, gl, modes=((0, 2), (1, 2)), alpha=1.0, ignore=IGNORE, pref=ht.WORKSPACE_RECOMMENDED):
        self.h, self.H, self.W, self.y, self.gl, self.alpha, self.ignore = h, H, W, y, gl, alpha, ignore
        self.plan = h.cross_entropy_plan(desc(h, H), modes[0], desc(h, W), modes[1], ignore)
        sizes = [h.cross_entropy_workspace_size(self.plan, g, pref) for g in (False, True)]
        self.ws = [torch.full((n,), 0xFF, device="cuda", dtype=torch.uint8) for n in sizes]  # NaN in every type
        t = y.numel()
        self.loss, self.lse = torch.full((t,), 9.0, device="cuda"), torch.full((t,), 9.0, device="cuda")
        self.dH, self.dW = torch.empty_strided(H.shape, H.stride(), dtype=H.dtype, device="cuda"), torch.empty_strided(
            W.shape, W.stride(), dtype=W.dtype, device="cuda")

    def forward(self, stream=None):
        self.h.cross_entropy(self.plan, self.alpha, self.H, self.W, self.y, self.loss, self.lse, self.ws[0], self.ws[0].numel(), stream)

    def backward(self, stream=None, want=(True, True)):
        self.h.cross_entropy_gradient(self.plan, self.alpha, self.H, self.W, self.y, self.lse, self.gl, self.dH if want[0] else None,
                                      self.dW if want[1] else None, self.ws[1], self.ws[1].numel(), stream)

    def check(self, H2=None, W2=None):
        """Against 64 bits; H2 / W2: H and W as matrices where they are not."""
        H, W = self.H if H2 is None else H2, self.W if W2 is None else W2
        within(*ref.loss(H, W, self.y, self.alpha, self.ignore), self.loss, self.lse)

    def check_gradient(self, dH=None, dW=None, H2=None, W2=None):
        H, W = self.H if H2 is None else H2, self.W if W2 is None else W2
        a, b, ea, eb = ref.gradient(H, W, self.y, self.lse, self.gl, self.alpha, self.ignore)
        within(a, b, ea, eb, self.dH if dH is None else dH, self.dW if dW is None else dW)


def within(a, b, ea, eb, x, y):
    for want, bound, got in ((a, ea, x), (b, eb, y)):
        off = (got.double() - want).abs()
        assert bool((off <= bound).all()), float((off - bound).nan_to_num(nan=9e9).max())


ALL = [torch.bfloat16, torch.float16, torch.float32]


@pytest.mark.parametrize("pref", [ht.WORKSPACE_MIN, ht.WORKSPACE_MAX])
@pytest.mark.parametrize("kind", ALL)
@pytest.mark.parametrize("t,v,d", [(1, 1, 1), (1, 1000, 64), (2, 257, 8), (17, 1031, 136), (130, 2000, 72), (300, 777, 260),
                                   (513, 513, 64), (700, 4100, 520), (40, 700, 2100), (300, 600, 4200),
                                   (129, 3000, 40), (400, 1500, 1100), (65, 9000, 24)])
def test_sizes(h, t, v, d, kind, pref):
    c = Call(h, *inputs(t, v, d, kind), pref=pref)
    c.forward()
    c.check()
    c.backward()
    c.check_gradient()
    assert h.device_status() == 0


@pytest.mark.parametrize("kind", ALL)
@pytest.mark.parametrize("t,v,d,ldpad", [(5, 300, 33, 0), (260, 700, 101, 0), (260, 700, 101, 3), (64, 1000, 64, 8)])
def test_odd_widths_and_padded_rows(h, t, v, d, ldpad, kind):
    c = Call(h, *inputs(t, v, d, kind, ldpad=ldpad))
    c.forward()
    c.check()
    c.backward()
    c.check_gradient()


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float32])
def test_tokens_in_several_modes_and_weights_the_other_way_round(h, kind):
    """The hidden states without the last position of every sequence (modes that do not fold), W stored [d, v]."""
    full, W, _, _ = inputs(7 * 21, 600, 64, kind)
    H = full.view(7, 21, 64)[:, :-1]
    y = torch.randint(0, 600, (140,), device="cuda")
    gl = torch.rand(140, device="cuda") / 140
    Wt = W.T.contiguous()
    c = Call(h, H, Wt, y, gl, modes=((5, 0, 2), (2, 1)))
    c.dH = torch.full_like(full, 3.0).view(7, 21, 64)[:, :-1]
    c.forward()
    c.check(H.reshape(140, 64), W)
    c.backward()
    c.check_gradient(c.dH.reshape(140, 64), c.dW.T, H.reshape(140, 64), W)
    assert bool((c.dH._base.view(7, 21, 64)[:, -1] == 3).all())


@pytest.mark.parametrize("kind", ALL)
@pytest.mark.parametrize("t,v,d,ldpad", [(20, 40, 4100, 4), (300, 700, 101, 3), (150, 900, 1026, 2), (130, 300, 60, 68)])
def test_what_lies_between_the_rows_of_dw_stays(h, t, v, d, ldpad, kind):
    c = Call(h, *inputs(t, v, d, kind, ldpad=ldpad))
    wide = torch.full((v, d + ldpad), 7.0, device="cuda", dtype=kind)
    c.dW = wide[:, :d]
    c.forward()
    c.backward()
    c.check_gradient()
    assert bool((wide[:, d:] == 7).all())


@pytest.mark.parametrize("kind", ALL)
def test_what_ignored_tokens_hold_counts_for_nothing(h, kind):
    H, W, y, gl = inputs(200, 900, 128, kind)
    H[y == IGNORE] = float("nan")
    H[torch.nonzero(y == IGNORE)[0]] = float("inf")
    gl[y == IGNORE] = float("nan")
    c = Call(h, H, W, y, gl)
    c.forward()
    keep = y != IGNORE
    assert bool((c.loss[~keep] == 0).all()) and bool(c.loss[keep].isfinite().all())
    c.backward()
    assert bool((c.dH[~keep] == 0).all())
    gz = torch.where(keep, gl, torch.zeros_like(gl))
    a, b, ea, eb = ref.gradient(H, W, y, c.lse, gz, 1.0, IGNORE)
    within(a, b, ea, eb, c.dH, c.dW)


@pytest.mark.parametrize("kind", ALL)
@pytest.mark.parametrize("t", [9, 40, 200])
@pytest.mark.parametrize("poison", [1e30, float("inf"), float("nan")])
def test_what_the_losses_gradients_of_tokens_that_do_not_count_hold(h, t, poison, kind):
    """Probabilities of about 1e-5 times a factor next to factors of ignored and out-of-range tokens that dwarf it. Logits are
    made by alpha = 1 / 64, so that small entries of P make gradients of ordinary size."""
    H, W, y, _ = inputs(t, 900, 128, kind)
    y[0], y[1], y[2:4] = IGNORE, 900, y[2:4].clamp(min=0)
    gl = torch.full((t,), 2.0 ** -6, device="cuda") * (1 + torch.arange(t, device="cuda") % 3)
    keep = (y >= 0) & (y < 900)
    gl[~keep] = poison
    c = Call(h, H * 64, W, y, gl, alpha=1 / 64)
    c.forward()
    torch.cuda.synchronize()
    with pytest.raises(ht.HiptensorError):  # the forward pass met the target that is no class
        c.backward()
    c.backward()
    torch.cuda.synchronize()
    with pytest.raises(ht.HiptensorError):
        c.forward()
    assert bool((c.dH[~keep] == 0).all())
    c.check_gradient()


@pytest.mark.parametrize("t", [9, 40, 200])
def test_one_infinite_loss_gradient_leaves_the_other_tokens_theirs(h, t):
    H, W, y, _ = inputs(t, 900, 128, torch.float16, ignored=0)
    gl = torch.full((t,), 2.0 ** -6, device="cuda")
    gl[t // 2] = float("inf")
    c = Call(h, H * 64, W, y, gl, alpha=1 / 64)
    c.forward()
    c.backward()
    rows = torch.arange(t, device="cuda") != t // 2
    want, _, bound, _ = ref.gradient(c.H[rows], W, y[rows], c.lse[rows], gl[rows], 1 / 64, IGNORE)
    assert bool(((c.dH[rows].double() - want).abs() <= bound).all())


@pytest.mark.parametrize("kind", ALL)
@pytest.mark.parametrize("t", [3, 8, 9, 40, 200])
@pytest.mark.parametrize("value", [float("inf"), -float("inf"), float("nan")])
def test_tokens_that_do_not_count_get_zeros_whatever_the_weights_hold(h, t, value, kind):
    H, W, y, gl = inputs(t, 600, 64, kind, ignored=0)
    W[17], W[400, 3] = value, value
    y[0], y[t // 2] = IGNORE, 600
    c = Call(h, H, W, y, gl)
    c.lse.fill_(1.0)
    c.backward()
    torch.cuda.synchronize()
    with pytest.raises(ht.HiptensorError):
        c.forward()
    dead = (y < 0) | (y >= 600)
    assert bool((c.dH[dead] == 0).all()) and bool(c.dH[~dead].isnan().any())


@pytest.mark.parametrize("kind", ALL)
@pytest.mark.parametrize("t", [1, 4, 9, 40, 300])
def test_the_loss_of_the_only_class_is_nothing(h, t, kind):
    H, W, _, gl = inputs(t, 1, 64, kind)
    H = H.abs() * (1 + 5 * torch.rand(t, 1, device="cuda")).to(kind)
    c = Call(h, H, W.abs() + 1, torch.zeros(t, device="cuda", dtype=torch.int64), gl, alpha=0.37)
    c.forward()
    assert bool((c.loss == 0).all()) and bool((c.lse > 1).all())


@pytest.mark.parametrize("kind", ALL)
@pytest.mark.parametrize("t,v", [(1, 300), (4, 700), (9, 300), (40, 700), (300, 4100)])
def test_no_loss_is_below_nothing(h, t, v, kind):
    """Every target is the class of the largest logit, about 100 to 1500, by margins from none to much."""
    H, W, y, gl = inputs(t, v, 64, kind, ignored=0)
    H, W = H.abs() + 1, W.abs() * 4 + 1
    W[v // 2] = W.amax(0) + (torch.arange(64, device="cuda") % 3).to(kind)
    y[:] = v // 2
    c = Call(h, H, W, y, gl)
    c.forward()
    assert bool((c.loss >= 0).all())
    c.check()


@pytest.mark.parametrize("kind,t", [(torch.bfloat16, 1), (torch.bfloat16, 40), (torch.bfloat16, 300), (torch.float16, 40), (torch.float32, 5),
                                    (torch.float32, 9), (torch.float32, 40), (torch.float32, 300)])
def test_classes_masked_by_the_lowest_value(h, kind, t):
    """The last column of W is the lowest value of the type for masked classes and H's is 1: they take no part."""
    H, W, y, gl = inputs(t, 600, 64, kind, ignored=0)
    low, open_ = torch.finfo(kind).min, 450
    H[:, 63], W[:, 63], W[open_:, 63], y[:] = 1, 0, low, y % open_
    c = Call(h, H, W, y, gl)
    c.forward()
    within(*ref.loss(H, W[:open_], y, 1.0, IGNORE), c.loss, c.lse)
    c.backward()
    a, b, ea, eb = ref.gradient(H, W[:open_], y, c.lse, gl, 1.0, IGNORE)
    within(a, b, ea, eb, c.dH, c.dW[:open_])
    assert bool((c.dW[open_:] == 0).all())
    y[0] = open_ + 7  # a target that is masked: as far away as the mask is
    c.forward()
    assert abs(float(c.loss[0]) / -low - 1) < 2.0 ** -10


@pytest.mark.parametrize("kind,t", [(torch.bfloat16, 1), (torch.bfloat16, 40), (torch.bfloat16, 300), (torch.float16, 40), (torch.float32, 5),
                                    (torch.float32, 9), (torch.float32, 40), (torch.float32, 300)])
def test_a_token_whose_every_class_is_masked_by_the_lowest_value(h, kind, t):
    H, W, y, gl = inputs(t, 600, 64, kind, ignored=0)
    low = torch.finfo(kind).min
    H[:, 63], W[:, 63], H[t // 2, 63] = 0, low, 1
    c = Call(h, H, W, y, gl)
    c.forward()
    others = torch.arange(t, device="cuda") != t // 2
    near = abs(low) * 2.0 ** -20  # the other terms of the sum (60 at most) are lost next to the mask
    assert abs(float(c.lse[t // 2]) - low) <= near + 60 and abs(float(c.loss[t // 2])) <= near + 60
    a, b, ea, eb = ref.loss(H[others], W, y[others], 1.0, IGNORE)
    within(a, b, ea, eb, c.loss[others], c.lse[others])


def test_the_longest_rows(h):
    """2^26 columns: more of them than a grid has blocks in its second dimension. All but a few columns are zeros."""
    d = 1 << 26
    H, W = torch.zeros(9, d, device="cuda", dtype=torch.bfloat16), torch.zeros(5, d, device="cuda", dtype=torch.bfloat16)
    some = torch.tensor([0, 1, 8191, d // 3, d - 1000, d - 2, d - 1], device="cuda")
    h0, w0, y, gl = inputs(9, 5, 7, torch.bfloat16, ignored=0)
    H[:, some], W[:, some] = h0, w0
    c = Call(h, H, W, y, gl, pref=ht.WORKSPACE_MIN)
    c.forward()
    c.backward()
    within(*ref.loss(h0, w0, y, 1.0, IGNORE), c.loss, c.lse)
    a, b, ea, eb = ref.gradient(h0, w0, y, c.lse, gl, 1.0, IGNORE)
    within(a, b, ea, eb, c.dH[:, some], c.dW[:, some])
    c.dH[:, some], c.dW[:, some] = 0, 0
    assert not bool(c.dH.any()) and not bool(c.dW.any())


@pytest.mark.parametrize("pref", [ht.WORKSPACE_MIN, ht.WORKSPACE_MAX])
@pytest.mark.parametrize("kind", ALL)
@pytest.mark.parametrize("times", [1, 3, 16])
@pytest.mark.parametrize("t,v,d", [(40, 300, 64), (65, 300, 64), (130, 2000, 72), (300, 1031, 101), (700, 4100, 260), (1500, 9000, 24)])
def test_the_targets_entries_are_not_rounded(h, t, v, d, times, kind, pref):
    """An lse far above every logit leaves -gradLoss alone in each row of P; `times` tokens have the same class (of up to 16 the
    entries are kept whole). dW and dH are then off by their own rounding alone, and dW by that of its f32 sum."""
    H, W, y, gl = inputs(t, v, d, kind, ignored=0)
    y[:] = torch.arange(t, device="cuda") % -(-t // times) * 11 % v  # (no v is a multiple of 11)
    y[t // 2] = IGNORE
    gl[:] = (1 + torch.rand(t, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")) * (1 - 2 * (torch.arange(t, device="cuda") % 2))
    c = Call(h, H, W, y, gl, pref=pref)
    c.lse.fill_(1e4)
    c.backward()
    P = torch.zeros(t, v, device="cuda", dtype=torch.float64)
    keep = y >= 0
    P[torch.arange(t, device="cuda")[keep], y[keep]] = -gl[keep].double()
    step = ref.half_step(kind) if kind != torch.float32 else 2.0 ** -22  # (f32: products of three-part sums, one more rounding)
    for got, p, x in ((c.dH, P, W.double()), (c.dW, P.T, H.double())):
        want, mag = p @ x, p.abs() @ x.abs()
        assert bool(((got.double() - want).abs() <= 1.01 * step * want.abs() + (times + 8) * 2.0 ** -23 * mag + 2.0 ** -25).all())


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("t,v,d", [(3, 20000, 512), (40, 9000, 256), (300, 20000, 256), (1000, 9000, 520)])
def test_gradients_are_off_by_their_own_rounding_in_the_mean(h, t, v, d, kind):
    """A bound for each element has room for the worst of thousands of classes; the norm of the whole error has not. A rounding is
    off by a step over the root of 12 in the mean, relative to a number at least step / (2 half_step): at most 2 / sqrt(12) half
    steps. The entries of P that are not targets' are rounded once more. f32 sums: 2^-18 is far above their error."""
    H, W, y, gl = inputs(t, v, d, kind)
    c = Call(h, H, W, y, gl)
    c.forward()
    c.backward()
    keep = y >= 0
    P = torch.exp(H.double() @ W.double().T - c.lse.double()[:, None]) * torch.where(keep, gl, torch.zeros_like(gl)).double()[:, None]
    full = P.clone()
    full[torch.arange(t, device="cuda")[keep], y[keep]] -= gl[keep].double()
    P[torch.arange(t, device="cuda")[keep], y[keep]] = 0
    for got, whole, others in ((c.dH, full @ W.double(), P @ W.double()), (c.dW, full.T @ H.double(), P.T @ H.double())):
        share = float(others.norm() / whole.norm())
        off = float((got.double() - whole).norm() / whole.norm())
        assert off <= 2 / 12 ** 0.5 * ref.half_step(kind) * (1 + share) + 2.0 ** -18, off / ref.half_step(kind)


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float16])
def test_a_class_of_very_many_tokens(h, kind):
    H, W, y, gl = inputs(900, 700, 136, kind, ignored=0.1)
    y[y >= 0] = torch.where(torch.arange(900, device="cuda") % 5 < 4, 333, y)[y >= 0]
    c = Call(h, H, W, y, gl)
    c.forward()
    c.backward()
    c.check_gradient()
    first = c.dW.clone()
    for _ in range(3):
        c.dW.fill_(9)
        c.backward()
        assert torch.equal(c.dW, first)


@pytest.mark.parametrize("kind", ALL)
def test_every_token_ignored(h, kind):
    H, W, y, gl = inputs(70, 300, 64, kind)
    y[:] = IGNORE
    c = Call(h, H, W, y, gl)
    c.forward()
    c.backward()
    assert bool((c.loss == 0).all()) and bool((c.dH == 0).all()) and bool((c.dW == 0).all())


@pytest.mark.parametrize("kind", ALL)
@pytest.mark.parametrize("t", [1, 2, 3, 4, 5, 8, 9])
@pytest.mark.parametrize("v,d,ldpad", [(1, 8, 0), (3, 4100, 4), (1201, 98, 0), (1500, 33, 3), (4001, 1026, 2), (700, 2048, 8), (2, 8200, 0)])
def test_few_tokens(h, v, d, ldpad, t, kind):
    c = Call(h, *inputs(t, v, d, kind, ldpad=ldpad))
    wide = torch.full((v, d + ldpad), 7.0, device="cuda", dtype=kind)
    c.dW = wide[:, :d]
    c.forward()
    c.check()
    c.backward()
    c.check_gradient()
    assert bool((wide[:, d:] == 7).all())
    both = c.dH.clone(), c.dW.clone()
    for want in ((True, False), (False, True)):
        c.dH.fill_(5), c.dW.fill_(5)
        c.backward(want=want)
        for got, before, wanted in zip((c.dH, c.dW), both, want):
            assert torch.equal(got, before) if wanted else bool((got == 5).all())
    assert h.device_status() == 0


@pytest.mark.parametrize("kind", ALL)
@pytest.mark.parametrize("t", [1, 3, 4, 8])
def test_few_tokens_some_of_which_count_for_nothing(h, t, kind):
    H, W, y, gl = inputs(t, 900, 130, kind, ignored=0)
    if t > 3:
        H = H.view(2, t // 2, 130).transpose(0, 1)  # tokens in two modes that do not fold: the second token is row t / 2
    y[0], gl[0] = IGNORE, float("nan")
    if t > 3:
        H[0, 0], H[0, 1] = float("nan"), float("inf")
    else:
        H[0], H[1:2] = float("nan"), float("inf")
    if t > 1:
        y[1] = 900
    c = Call(h, H, W, y, gl, modes=((0, 5, 2), (1, 2)) if t > 3 else ((0, 2), (1, 2)))
    c.forward()
    torch.cuda.synchronize()
    rows = c.H.reshape(t, 130)
    bad = y == 900
    assert float(c.loss[0]) == 0 and torch.equal(c.loss.isnan(), bad)
    keep = (y >= 0) & ~bad
    if bool(bad.any()):
        assert h.device_status() == 7
        with pytest.raises(ht.HiptensorError):
            c.backward()
    lse = torch.where(keep, c.lse, torch.full_like(c.lse, float("nan")))
    c.lse = lse
    c.backward()
    torch.cuda.synchronize()
    if bool(bad.any()):
        assert h.device_status() == 7
        with pytest.raises(ht.HiptensorError):
            c.forward()
    dH = c.dH.reshape(t, 130)
    assert bool((dH[~keep] == 0).all())
    a, b, ea, eb = ref.gradient(rows, W, y, lse, gl, 1.0, IGNORE)
    within(a, b, ea, eb, dH, c.dW)


def test_few_tokens_and_infinite_weights(h):
    H, W, y, gl = inputs(3, 600, 64, torch.float32, ignored=0)
    H[:], y[:] = H.abs() + 0.1, 5
    W[17], W[400] = -float("inf"), -float("inf")
    c = Call(h, H, W, y, gl)
    c.forward()
    keep = [i for i in range(600) if i not in (17, 400)]
    lse = torch.logsumexp(H.double() @ W[keep].double().T, 1)
    assert bool(((c.lse.double() - lse).abs() < 2.0 ** -17 * (1 + lse.abs())).all())
    W[17] = float("inf")
    c.forward()
    assert bool((c.lse == float("inf")).all())
    W[17] = float("nan")
    c.forward()
    assert bool(c.lse.isnan().all()) and bool(c.loss.isnan().all())


def test_an_ignored_index_inside_the_vocabulary(h):
    H, W, y, gl = inputs(100, 300, 64, torch.bfloat16, ignored=0)
    y[::3] = 0
    c = Call(h, H, W, y, gl, ignore=0)
    c.forward()
    c.check()
    c.backward()
    c.check_gradient()


def test_a_target_outside_the_vocabulary(h):
    H, W, y, gl = inputs(100, 300, 64, torch.bfloat16, ignored=0)
    y[3], y[50] = 300, -1
    c = Call(h, H, W, y, gl)
    c.forward()
    torch.cuda.synchronize()
    assert h.device_status() == 7
    assert torch.equal(c.loss.isnan(), (y < 0) | (y >= 300))
    with pytest.raises(ht.HiptensorError) as e:
        c.backward()
    assert e.value.status == ht.STATUS_EXECUTION_FAILED
    c.backward()
    c.check_gradient()
    assert bool((c.dH[3] == 0).all())
    with pytest.raises(ht.HiptensorError):
        c.forward()


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("alpha", [-0.5, 30.0])
def test_alpha_and_large_logits(h, kind, alpha):
    H, W, y, gl = inputs(150, 1300, 96, kind)
    c = Call(h, H, W, y, gl, alpha=alpha)
    c.forward()
    c.check()
    c.backward()
    c.check_gradient()


@pytest.mark.parametrize("kind", ALL)
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("t,v", [(1, 40), (3, 700), (40, 700), (300, 9000)])
def test_every_logit_far_from_zero(h, t, v, sign, kind):
    """Logits of about 130 to 2000, all of one sign: nothing is taken relative to zero."""
    H, W, y, gl = inputs(t, v, 64, kind)
    c = Call(h, (H.abs() + 1) * sign, W.abs() * 8 + 2, y, gl)
    c.forward()
    c.check()
    c.backward()
    c.check_gradient()


def test_infinite_logits(h):
    H, W, y, gl = inputs(40, 600, 64, torch.bfloat16, ignored=0)
    H[:], y[:] = H.abs() + 0.1, 5
    W[17], W[400] = -float("inf"), -float("inf")
    c = Call(h, H, W, y, gl)
    c.forward()
    keep = [i for i in range(600) if i not in (17, 400)]
    lse = torch.logsumexp(H.double() @ W[keep].double().T, 1)
    assert bool(((c.lse.double() - lse).abs() < 2.0 ** -12 * (1 + lse.abs())).all())
    W[17] = float("inf")
    c.forward()
    assert bool((c.lse == float("inf")).all())
    W[17] = float("nan")
    c.forward()
    assert bool(c.lse.isnan().all()) and bool(c.loss.isnan().all())


@pytest.mark.parametrize("want", [(True, False), (False, True)])
def test_one_gradient_alone(h, want):
    H, W, y, gl = inputs(300, 900, 128, torch.bfloat16)
    c = Call(h, H, W, y, gl)
    c.forward()
    c.backward()
    both = c.dH.clone(), c.dW.clone()
    c.dH.fill_(7), c.dW.fill_(7)
    c.backward(want=want)
    for got, before, wanted in zip((c.dH, c.dW), both, want):
        assert torch.equal(got, before) if wanted else bool((got == 7).all())


@pytest.mark.parametrize("kind", ALL)
def test_no_tokens(h, kind):
    H, W, y, gl = inputs(0, 300, 64, kind)
    c = Call(h, H, W, y, gl)
    c.dW.fill_(5)
    c.forward()
    c.backward()
    assert bool((c.dW == 0).all())


def test_too_little_workspace(h):
    H, W, y, gl = inputs(100, 3000, 64, torch.bfloat16)
    c = Call(h, H, W, y, gl, pref=ht.WORKSPACE_MIN)
    for k, call in enumerate((c.forward, c.backward)):
        full = c.ws[k]
        c.ws[k] = full[:-1]
        with pytest.raises(ht.HiptensorError) as e:
            call()
        assert e.value.status == ht.STATUS_INSUFFICIENT_WORKSPACE
        c.ws[k] = full
        call()


def test_unaligned_workspace_and_refused_pointers(h):
    H, W, y, gl = inputs(100, 3000, 64, torch.bfloat16)
    c = Call(h, H, W, y, gl, pref=ht.WORKSPACE_MIN)
    c.ws = [torch.empty(w.numel() + 3, device="cuda", dtype=torch.uint8)[3:] for w in c.ws]
    c.forward()
    c.check()
    c.backward()
    c.check_gradient()
    c.H = torch.empty(100 * 64 + 1, device="cuda", dtype=torch.bfloat16)[1:]
    for call in (c.forward, c.backward):
        with pytest.raises(ht.HiptensorError) as e:
            call()
        assert e.value.status == ht.STATUS_INVALID_VALUE


@pytest.mark.parametrize("kind", ALL)
def test_the_gradient_is_the_loss_s_slope(h, kind):
    """Differences of the loss along a direction, in f32 from the operator itself, against the gradient's product with it."""
    H, W, y, gl = inputs(60, 500, 64, torch.float32)
    H, W = H.to(kind).float(), W.to(kind).float()
    c = Call(h, H.to(kind), W.to(kind), y, torch.ones_like(gl))
    c.forward()
    c.backward()
    u, v = torch.randn_like(H), torch.randn_like(W) * 0.1
    f = Call(h, H, W, y, torch.ones_like(gl))
    e, ends = 2.0 ** -6, []
    for s in (e, -e):
        f.H, f.W = H + s * u, W + s * v
        f.forward()
        ends.append(f.loss.double().sum())
    slope = float((ends[0] - ends[1]) / (2 * e))
    exact = float((c.dH.double() * u).sum() + (c.dW.double() * v).sum())
    # third derivatives times e^2 / 6 (logits move by about 2 a unit), and the gradient's own rounding over its terms
    size = float((c.dH.double() * u).norm() + (c.dW.double() * v).norm())
    assert abs(slope - exact) <= 60 * 8 * e * e / 6 + 8 * ref.half_step(kind) * size + 60 * 2.0 ** -16 / e


def test_twice_the_same_and_two_captured_graphs(h):
    H, W, y, gl = inputs(333, 5000, 256, torch.bfloat16)
    one, two = Call(h, H, W, y, gl), Call(h, H.flip(0).contiguous(), W, y.flip(0).contiguous(), gl)
    for c in (one, two):
        c.forward()
        c.backward()
    first = [x.clone() for x in (one.loss, one.dH, one.dW, two.loss, two.dH, two.dW)]
    graphs = []
    for c in (one, two):
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            c.forward(torch.cuda.current_stream())
            c.backward(torch.cuda.current_stream())
        graphs.append((g, side))
    for c in (one, two):
        for x in (c.loss, c.lse, c.dH, c.dW):
            x.fill_(0)
    torch.cuda.synchronize()
    for _ in range(3):
        for g, side in graphs:  # at the same time: each has its own workspace
            with torch.cuda.stream(side):
                g.replay()
    torch.cuda.synchronize()
    for x, want in zip((one.loss, one.dH, one.dW, two.loss, two.dH, two.dW), first):
        assert torch.equal(x, want)


def test_a_training_step_in_8_bits(h):
    """Activations and weights quantised, a linear layer, the head's loss and gradient, and the layer's two gradient products."""
    t, k, n, v = 300, 512, 384, 2000
    E4, E5 = ht.R_8F_E4M3, ht.R_8F_E5M2
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(t, k, generator=g, device="cuda").to(torch.bfloat16)
    w = torch.randn(n, k, generator=g, device="cuda") / k ** 0.5
    head = (torch.randn(v, n, generator=g, device="cuda") / n ** 0.5).to(torch.bfloat16)
    y = torch.randint(0, v, (t,), generator=g, device="cuda")
    kinds = {E4: torch.float8_e4m3fn, E5: torch.float8_e5m2}
    kind_of = lambda z: {torch.bfloat16: ht.R_16BF, torch.float32: ht.R_32F, torch.float8_e4m3fn: E4, torch.float8_e5m2: E5}[z.dtype]  # noqa: E731
    d = lambda z: h.tensor_descriptor(z.shape, z.stride(), kind_of(z))  # noqa: E731

    def quant(z, block, to, turned=False):
        ld = -(-(z.shape[0] if turned else z.shape[1]) // 16) * 16
        q = torch.zeros(z.shape[1] if turned else z.shape[0], ld, device="cuda", dtype=kinds[to])
        q = q[:, :z.shape[0]] if turned else q[:, :z.shape[1]]
        s = torch.empty([-(-a // b) for a, b in zip(z.shape, block)], device="cuda")
        h.block_quantize(z, d(z), (0, 1), block, q, d(q), (1, 0) if turned else (0, 1), s, d(s))
        return (q, s.T, block[::-1]) if turned else (q, s, block)

    def product(A, B, out, c=None):
        (a, sa, ba), (b, sb, bb) = A, B
        plan = h.scaled_contraction_plan(d(a), (0, 2), d(sa), ba, d(b), (1, 2), d(sb), bb, None if c is None else d(out), d(out), (0, 1))
        h.scaled_contraction(plan, 1.0, a, sa, b, sb, 0.0 if c is None else 1.0, c, out)
        want, bound = ref.scaled(a, sa, ba, b, sb, bb, 1.0, 1.0, c)
        tail = 1.01 * 2.0 ** -8 if out.dtype == torch.bfloat16 else 2.0 ** -23
        return want, bound + tail * want.abs()

    hidden = torch.empty(t, n, device="cuda", dtype=torch.bfloat16)
    master = torch.randn(n, k, device="cuda") * 1e-3
    before = master.clone()
    want, bound = product(quant(x, (1, 128), E4), quant(w, (128, 128), E4), hidden)
    assert bool(((hidden.double() - want).abs() <= bound).all())
    c = Call(h, hidden, head, y, torch.full((t,), 1.0 / t, device="cuda"))
    c.forward()
    c.check()
    c.backward()
    c.check_gradient()
    dx = torch.empty_like(x)
    want, bound = product(quant(c.dH, (1, 128), E5), quant(w, (128, 128), E4, turned=True), dx)
    assert bool(((dx.double() - want).abs() <= bound).all())
    want, bound = product(quant(c.dH, (128, 1), E5, turned=True), quant(x, (128, 1), E4, turned=True), master, before)
    assert bool(((master.double() - want).abs() <= bound).all())
