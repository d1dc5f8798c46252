"""Fine-tuning operators (prosim_amd.finetune) against plain implementations in 64 bits.

Tolerances, with u = 2^-24 (half a step of float32):
* an exponential e^d, d = x - max <= 0, is off by at most (|d| + |d| / 2 + 2) u * 2 relative (rounding of d, of its product with log2 e and of that
  constant, one step of the exponential); a row's sum is added in 64 bits.
  Weighted with p = e^d / s, sum p |d| = H - ln s <= ln K, so ln s is off by at most u (3 ln K + 4), and a stored log-probability by
  u (|logp| + 3 ln K + 4); the end of a row (its 64-bit logarithm) is far below the 4 u left.
* a gradient element coef (one-hot - p): half a step of its type, plus |coef| p u (3 |d| + 8 + the sum's error) and the one-hot difference's 2 u |coef|,
  plus the error of coef: its own rounding and the log-probability's error times d coef / d logp.
"""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
U = 2.0 ** -24


@pytest.fixture(scope="module")
def ft():
    from prosim_amd import finetune
    return finetune


def dev():
    return torch.device("cuda", torch.cuda.current_device())


def rand(*shape, seed=0, dtype=torch.float32):
    g = torch.Generator()
    g.manual_seed(seed + 7919 * len(shape) + sum(shape))
    return torch.randn(*shape, generator=g).to(dtype)


def row_slack(k):
    return U * (3.0 * math.log(k) + 8.0)


def plain_logp(x, c):
    x = x.double()
    return torch.log_softmax(x, -1).gather(-1, c.long().clamp(0, x.shape[-1] - 1)[..., None])[..., 0]


def plain_grad(x, c, coef):
    """coef (one-hot - softmax) in 64 bits."""
    p = torch.softmax(x.double(), -1)
    g = -p * coef.double()[..., None]
    return g.scatter_add(-1, c.long()[..., None], coef.double()[..., None])


def grad_tol(x, c, coef, dcoef, dtype):
    """Element-wise bound for coef (one-hot - p); dcoef: the error of coef."""
    xd = x.double()
    p = torch.softmax(xd, -1)
    d = (xd - xd.max(-1, keepdim=True).values).abs().clamp(max=1.0e4)
    d = torch.where(p == 0, torch.zeros_like(d), d)
    hot = torch.zeros_like(p).scatter_(-1, c.long()[..., None], 1.0)
    a = coef.double().abs()[..., None]
    k = x.shape[-1]
    t = a * (p * U * (3.0 * d + 8.0 + 3.0 * math.log(k) + 8.0) + hot * 2 * U) + dcoef[..., None] * (hot + p)
    out = plain_grad(x, c, coef).abs()
    tiny = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -25}[dtype]
    return t * 1.01 + out * (torch.finfo(dtype).eps / 2) * 1.01 + tiny


def close(got, want, tol, what=""):
    got, want = got.double(), want.double()
    same = (got == want) | (got.isnan() & want.isnan())
    bad = ~same & ~((got - want).abs() <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float(((got - want).abs() - tol)[bad].max())} beyond its bound"


ROWS_CHOICES = [(130, 70001), (129, 131080), (40000, 30), (30000, 4), (257, 5), (9000, 8), (1000, 9), (7000, 16), (70, 250), (90, 600), (60, 2048), (1, 1), (5, 1), (1, 2), (3, 3), (1025, 3), (17, 7), (64, 16), (65, 17), (31, 64), (33, 65), (9, 127), (10, 128), (7, 255), (5, 257), (130, 511), (4, 513),
                (3, 1000), (6, 1024), (5, 2049), (2, 4096), (3, 4099), (2, 8191), (3, 16387), (2, 32768), (1, 50021), (2, 65537), (1, 131072), (2, 131071), (1, 200003),
                (300, 1111), (2500, 40), (70, 9001)]


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("rows,k", ROWS_CHOICES)
def test_choice_logp_and_gradient(ft, rows, k, dtype):
    x = (rand(rows, k, seed=1) * 3.0).to(dtype).to(dev())
    c = torch.randint(0, k, (rows,), generator=torch.Generator().manual_seed(k)).to(dev())
    c[-1] = k - 1
    want = plain_logp(x, c)
    got = ft.choice_logp(x, c)
    assert got.dtype == torch.float32 and got.shape == (rows,)
    close(got, want, U * want.abs() + row_slack(k), "logp")
    g = rand(rows, seed=3).to(dev())
    leaf = x.clone().requires_grad_(True)
    out = ft.choice_logp(leaf, c.int())
    assert torch.equal(out, got)
    grad, = torch.autograd.grad(out, leaf, g)
    assert grad.dtype == dtype
    close(grad, plain_grad(x, c, g), grad_tol(x, c, g, 2 * U * g.double().abs(), dtype), "gradient")


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("rows,k", [(60000, 4), (40000, 30), (8192, 600), (2048, 5000), (512, 70001)])
def test_log_probabilities_are_off_by_their_own_rounding_only(ft, rows, k, dtype):
    """Over many rows the errors of the exponentials average out, so what is left of the error is the result's own rounding: a step of s spread evenly
    gives s / sqrt(12) rms, s <= |logp| 2^-23, plus that of a row's own sum -- single exponentials of half a step each, at most 2 u p_i (1 + |d_i|) added in
    squares: 4 u^2 sum p_i^2 (1 + |d_i|)^2 -- and no mean beyond three standard errors of that plus the exponential's mean error, taken as a tenth of u.
    (Adding in 32 bits, or log2 e cut to 24 bits, moves the mean by 0.2 u to 0.4 u or doubles the spread.)"""
    x = rand(rows, k, seed=3, dtype=dtype).to(dev())
    c = torch.arange(rows, device=x.device) % k
    want = plain_logp(x, c)
    err = (ft.choice_logp(x, c).double() - want)
    xd = x.double()
    p = torch.softmax(xd, -1)
    d = (xd.max(-1, keepdim=True).values - xd)
    var = (want.abs() * 2 * U) ** 2 / 12 + 4 * U * U * (p * p * (1 + d) ** 2).sum(-1)
    assert float((err ** 2).mean()) <= 1.1 * float(var.mean())
    assert abs(float(err.mean())) <= 3 * math.sqrt(float(var.mean()) / rows) + 0.1 * U, (float(err.mean()) / U, float((err ** 2).mean().sqrt()) / U)


def policy_plain(x, c, old, adv, ref, mask, lo, hi, beta, mean, scale):
    """Loss, logp, kl, share, gradient and its coefficient's derivative, in 64 bits."""
    logp = plain_logp(x, c)
    v = torch.ones_like(logp) if mask is None else mask.double()
    n = float(v.sum()) if float(v.sum()) > 0 else 1.0
    w = scale / (n if mean else 1.0)
    r, a = torch.exp(logp - old.double()), adv.double().expand_as(logp)
    s1, s2 = r * a, r.clamp(1.0 - lo, 1.0 + hi) * a
    hold = s2 < s1
    loss, slope, curve = -torch.minimum(s1, s2), torch.where(hold, 0.0, -s1), torch.where(hold, 0.0, s1.abs())
    kl = torch.zeros_like(r)
    if ref is not None:
        d = ref.double() - logp
        kl = torch.exp(d) - d - 1.0
        loss, slope, curve = loss + beta * kl, slope + beta * (1.0 - torch.exp(d)), curve + beta * torch.exp(d)
    loss, kl, slope, curve, logp = (torch.where(v > 0, t, 0.0) for t in (loss, kl, slope, curve, logp))
    coef = slope * w
    return loss.sum() * w, logp, kl.sum() / n, (hold & (v > 0)).sum() / n, plain_grad(torch.where((v > 0)[..., None], x.double(), 0.0), c, coef), coef, curve * abs(w)


def policy_inputs(rows, k, dtype, seed):
    x = (rand(rows, k, seed=seed) * 2.0).to(dtype).to(dev())
    g = torch.Generator().manual_seed(seed)
    c = torch.randint(0, k, (rows,), generator=g).to(dev())
    x.scatter_(1, c[:, None], (math.log(k) + 1.0 + rand(rows, 1, seed=seed + 1).to(dev())).to(dtype))
    now = plain_logp(x, c).float()
    old = now + 0.2 * rand(rows, seed=seed + 2).to(dev())
    ref = now + 0.5 * rand(rows, seed=seed + 3).to(dev())
    # no ratio within 1e-4 of a border of the clipping range: there the two sides may rightly differ
    ratio = torch.exp(now.double() - old.double())
    for border in (0.8, 1.3):
        old = torch.where((ratio - border).abs() < 1e-4, old + 1e-3, old)
    return x, c, old, rand(rows, seed=seed + 4).to(dev()), ref


def check_policy(ft, x, c, old, adv, ref, mask, beta, reduction, scale, gain=1.0):
    dtype, k = x.dtype, x.shape[-1]
    leaf = x.clone().requires_grad_(True)
    out = ft.policy_loss(leaf, c, old, adv, ref_logp=ref, mask=mask, clip_low=0.2, clip_high=0.3, kl_coef=beta, reduction=reduction, scale=scale)
    grad, = torch.autograd.grad(out.loss * gain if gain != 1.0 else out.loss, leaf)
    loss, logp, kl, frac, dx, coef, curve = policy_plain(x, c, old, adv, ref, mask, 0.2, 0.3, beta, reduction == "mean", scale)
    slack = row_slack(k)
    close(out.logp, logp, U * logp.abs() + slack, "logp")
    n = max(1, int(mask.sum()) if mask is not None else c.numel())
    bound = float(curve.sum())          # sum of |d loss_i / d logp_i| bounds, weighted
    close(out.loss, loss, 2 * U * loss.abs() + bound * slack + 1e-12, "loss")
    kl_slope = 0.0 if ref is None else float(torch.exp(ref.double() - logp).add(1.0).mean())
    close(out.kl, kl, 2 * U * kl.abs() + kl_slope * slack + 1e-12, "kl")
    close(out.clip_frac, frac, U * 2, "clip_frac")
    masked_x = x if mask is None else torch.where(mask[..., None], x, torch.zeros_like(x))
    coef, curve = coef * gain, curve * abs(gain)
    close(grad, dx * gain, grad_tol(masked_x, c, coef, 4 * U * coef.abs() + curve * slack, dtype), "gradient")
    # without a gradient: the same numbers
    with torch.no_grad():
        again = ft.policy_loss(leaf, c, old, adv, ref_logp=ref, mask=mask, clip_low=0.2, clip_high=0.3, kl_coef=beta, reduction=reduction, scale=scale)
    for a, b in zip(again, out):
        assert torch.equal(a, b.detach())


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("rows,k", [(1, 1), (1, 2), (7, 3), (1025, 3), (31, 64), (130, 65), (9, 513), (300, 1111), (5, 2049), (2, 8191), (1, 50021), (3, 65537), (2, 131071), (1, 200003)])
@pytest.mark.parametrize("masked", [False, True])
def test_policy_loss(ft, rows, k, dtype, masked):
    x, c, old, adv, ref = policy_inputs(rows, k, dtype, seed=rows + k)
    mask = None
    if masked:
        mask = torch.rand(rows, generator=torch.Generator().manual_seed(5)).to(dev()) < 0.7
        c = torch.where(mask, c, torch.zeros_like(c))
    check_policy(ft, x, c, old, adv, ref, mask, 0.05, "mean", 1.0)
    check_policy(ft, x, c, old, adv, None, mask, 0.0, "sum", 0.25)


# every way rows are laid out over threads (groups of 8 .. 64 lanes, 2 .. 16 waves, two passes, split rows), at its borders
BORDERS = [32, 33, 40, 63, 64, 65, 100, 127, 128, 129, 255, 256, 257, 511, 512, 513, 1023, 1024, 1025, 2047, 2048, 2050, 4096, 4103, 8192, 8199, 16390, 32775, 65543]


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("pad,offset", [(0, 0), (0, 1), (5, 3), (64, 0)])
def test_row_lengths_at_odd_addresses(ft, dtype, pad, offset):
    """Rows of every length class, beginning at any element, dense or with a gap behind each (then the gradient's rows are aligned otherwise than the logits')."""
    rows = 70
    for k in BORDERS:
        n = rows if k < 20000 else 3
        flat = (rand(n * (k + pad) + offset, seed=k) * 2).to(dtype).to(dev())
        x = flat[offset:].view(n, k + pad)[:, :k]
        c = torch.randint(0, k, (n,), generator=torch.Generator().manual_seed(k)).to(dev())
        c[0], c[1] = 0, k - 1
        now = plain_logp(x, c)
        old = (now + 0.1).float()
        adv = rand(n, seed=1).to(dev())
        mask = torch.ones(n, dtype=torch.bool, device=dev())
        mask[-1] = False
        check_policy(ft, x, c, old, adv, None, mask, 0.0, "sum", 1.0)
        leaf = x.detach().requires_grad_(True)
        out = ft.choice_logp(leaf, c, mask=mask)
        close(out, torch.where(mask, now, 0.0), U * now.abs() + row_slack(k), f"logp of {k}")
        g = rand(n, seed=3).to(dev())
        grad, = torch.autograd.grad(out, leaf, g)
        g = torch.where(mask, g, 0.0)
        close(grad, plain_grad(x, c, g), grad_tol(x, c, g, 2 * U * g.double().abs(), dtype), f"gradient of {k}")


@pytest.mark.parametrize("dtype,k", [(torch.float32, 66001), (torch.bfloat16, 140003), (torch.float16, 131080)])
def test_rows_no_block_can_hold(ft, dtype, k):
    """More than 64 rows longer than 256 KB: statistics by parts, the end of a row, the gradient, a launch each -- from C also without the caller's statistics."""
    from prosim_amd.engine import PsDecisions, PsPolicyTerms, load_library
    rows = 67
    x, c, old, adv, ref = policy_inputs(rows, k, dtype, seed=12)
    mask = torch.rand(rows, generator=torch.Generator().manual_seed(6)).to(dev()) < 0.7
    check_policy(ft, x, c, old, adv, ref, mask, 0.1, "mean", 1.0)
    leaf = x.detach().requires_grad_(True)
    o = ft.policy_loss(leaf, c, old, adv, ref_logp=ref, mask=mask, kl_coef=0.1)
    want, = torch.autograd.grad(o.loss, leaf)
    lib = load_library()
    d = PsDecisions(x.data_ptr(), rows, k, k, {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}[dtype], 64, c.data_ptr(), mask.data_ptr())
    q = PsPolicyTerms(old.data_ptr(), adv.data_ptr(), ref.data_ptr(), 0.2, 0.2, 0.1, 1.0, 1)
    nums, logp, grad = torch.empty(3, device=dev()), torch.empty(rows, device=dev()), torch.empty_like(x)
    space = torch.empty(lib.ps_choice_workspace(d), dtype=torch.uint8, device=dev())
    at = nums.data_ptr()
    rc = lib.ps_policy_loss(d, q, at, at + 4, at + 8, logp.data_ptr(), None, None, grad.data_ptr(), space.data_ptr(), space.numel(), torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    assert torch.equal(grad, want) and torch.equal(logp, o.logp) and torch.equal(nums[0], o.loss.detach()) and torch.equal(nums[1], o.kl)


def test_more_blocks_than_one_grid_dimension(ft):
    """70001 rows of a block each, and ten stretches of the gradient per row: samples around the ends and the 65536th block."""
    rows, k = 70001, 9001
    x = torch.zeros((rows, k), dtype=torch.bfloat16, device=dev())
    pick = torch.tensor([0, 1, 6553, 6554, 65534, 65535, 65536, 65537, 69999, 70000], device=dev())
    x[pick] = (rand(len(pick), k, seed=2) * 2).to(torch.bfloat16).to(dev())
    c = torch.full((rows,), k - 1, dtype=torch.int32, device=dev())
    leaf = x.requires_grad_(True)
    out = ft.choice_logp(leaf, c)
    want = plain_logp(x.detach()[pick], c[pick])
    close(out.detach()[pick], want, U * want.abs() + row_slack(k), "logp")
    g, = torch.autograd.grad(out, leaf, torch.ones(rows, device=dev()))
    one = torch.ones_like(want)
    close(g[pick], plain_grad(x.detach()[pick], c[pick], one), grad_tol(x.detach()[pick], c[pick], one, one * 0, torch.bfloat16), "gradient")
    rest = torch.ones(rows, dtype=torch.bool, device=dev())
    rest[pick] = False
    assert (out.detach()[rest] - out.detach()[2]).abs().max() == 0 and abs(float(out.detach()[2]) + math.log(k)) < 1e-5
    same = g[2].clone()
    for a in range(0, rows, 10000):
        assert (g[a:a + 10000][rest[a:a + 10000]] == same).all()
    mask = torch.rand(rows, generator=torch.Generator().manual_seed(1)).to(dev()) < 0.5
    mask[pick] = True
    o = ft.policy_loss(leaf, c, out.detach(), one[:1].float(), mask=mask, reduction="mean")
    assert abs(float(o.loss.detach()) + 1.0) < 1e-5
    gp, = torch.autograd.grad(o.loss, leaf)
    coef = -one / float(mask.sum())
    close(gp[pick], plain_grad(x.detach()[pick], c[pick], coef), grad_tol(x.detach()[pick], c[pick], coef, coef.abs() * (8 * U + row_slack(k)), torch.bfloat16), "policy gradient")
    assert not gp[~mask][:2000].any()


@pytest.mark.parametrize("rows,k", [(1500, 5000), (20000, 40), (300, 700), (40000, 3), (30000, 30), (513, 4), (512, 4), (511, 5)])
def test_the_mean_counts_valid_rows_in_every_layout(ft, rows, k):
    x, c, old, adv, ref = policy_inputs(rows, k, torch.float16, seed=3)
    mask = torch.rand(rows, generator=torch.Generator().manual_seed(6)).to(dev()) < 0.5
    check_policy(ft, x, c, old, adv, ref, mask, 0.1, "mean", 1.0)
    check_policy(ft, x, c, old, adv, ref, mask.to(torch.uint8) * 255 != 0, 0.1, "sum", 1e-4)
    leaf = x.clone().requires_grad_(True)
    a = ft.policy_loss(leaf, c, old, adv, mask=mask)
    b = ft.policy_loss(leaf, c, old, adv, mask=mask.to(torch.uint8) * 200)       # (any byte but 0 is valid)
    assert torch.equal(a.loss, b.loss) and torch.equal(a.logp, b.logp)


@pytest.mark.parametrize("rows", [1, 15, 33, 5000, 16401, 70003])
@pytest.mark.parametrize("off", [1, 3, 16])
def test_a_mask_at_any_address(ft, rows, off):
    x, c, old, adv, ref = policy_inputs(rows, 9, torch.bfloat16, seed=8)
    mask = (torch.rand(off + rows + 64, generator=torch.Generator().manual_seed(rows)).to(dev()) < 0.5)      # (valid and masked bytes around it, too)
    check_policy(ft, x, c, old, adv, ref, mask[off:off + rows], 0.1, "mean", 1.0)
    steps = rows // 3
    if steps:
        m = mask[off:off + 3 * steps].view(3, steps)
        w = rand(3, steps, seed=9).to(dev()).requires_grad_(True)
        a, b = ft.preference_loss(w, w * 0.5, better_mask=m, worse_mask=m), ft.preference_loss(w, w * 0.5, better_mask=m.clone(), worse_mask=m.clone())
        assert torch.equal(a.loss, b.loss) and torch.equal(a.margin, b.margin)
        assert torch.equal(torch.autograd.grad(a.loss, w)[0], torch.autograd.grad(b.loss, w)[0])


def test_mean_loss_of_many_rows_counts_its_mask(ft):
    rows, k = 70001, 6
    x, c, old, adv, ref = policy_inputs(rows, k, torch.float32, seed=3)
    mask = torch.rand(rows, generator=torch.Generator().manual_seed(6)).to(dev()) < 0.5
    check_policy(ft, x, c, old, adv, ref, mask, 0.1, "mean", 3.0)
    check_policy(ft, x, c, old, adv, ref, mask.to(torch.uint8).bool(), 0.1, "sum", 1e-4)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("k", [5, 700, 40001])
def test_a_gradient_that_arrives_with_another_factor_and_twice(ft, dtype, k):
    """loss * 1024 (a scaler's factor: the gradient must not have been rounded before it), then two passes over a retained graph."""
    x, c, old, adv, ref = policy_inputs(11, k, dtype, seed=9)
    check_policy(ft, x, c, old, adv, ref, None, 0.05, "mean", 1.0, gain=1024.0)
    leaf = x.clone().requires_grad_(True)
    out = ft.policy_loss(leaf, c, old, adv)
    one, = torch.autograd.grad(out.loss, leaf, retain_graph=True)
    keep = one.clone()
    one.zero_()                                     # (what a caller does with its gradient must not reach the next pass)
    two, = torch.autograd.grad(out.loss, leaf, retain_graph=True)
    half, = torch.autograd.grad(out.loss, leaf, torch.full((), 0.5, device=dev()))
    if k < 600:
        assert torch.equal(two, keep)
    close(two, keep.double(), keep.double().abs() * torch.finfo(dtype).eps + 2 * U * keep.double().abs().max() + (2.0 ** -24 if dtype == torch.float16 else 0), "second pass")
    close(half, keep.double() / 2, keep.double().abs() * torch.finfo(dtype).eps + 2 * U * keep.double().abs().max() + (2.0 ** -24 if dtype == torch.float16 else 0), "half")


def test_gradient_against_differences(ft):
    """Central differences of the loss itself (float32: the step is large enough that its rounding, u |loss| / h, stays below 1e-4; h^2 / 6 times the third
    derivative, of order 1 / rows times a few, below 1e-3)."""
    x, c, old, adv, ref = policy_inputs(6, 9, torch.float32, seed=21)
    leaf = x.clone().requires_grad_(True)
    kw = dict(ref_logp=ref, kl_coef=0.1)
    grad, = torch.autograd.grad(ft.policy_loss(leaf, c, old, adv, **kw).loss, leaf)
    h = 2.0 ** -6
    ratio = torch.exp(plain_logp(x, c) - old.double())
    free = ((ratio - 0.8).abs() > 0.1) & ((ratio - 1.2).abs() > 0.1)       # (rows whose ratio crosses a border within the step have no derivative there)
    for j in range(9):
        v = torch.zeros_like(x)
        v[free, j] = h
        if not free.any():
            break
        diff = (ft.policy_loss(x + v, c, old, adv, **kw).loss.double() - ft.policy_loss(x - v, c, old, adv, **kw).loss.double()) / (2 * h)
        assert abs(float(diff) - float(grad[free, j].double().sum())) < 2e-3
    assert free.any()
    logp_leaf = x.clone().requires_grad_(True)
    g, = torch.autograd.grad(ft.choice_logp(logp_leaf, c).sum(), logp_leaf)
    for j in range(9):
        v = torch.zeros_like(x)
        v[:, j] = h
        diff = (ft.choice_logp(x + v, c).double().sum() - ft.choice_logp(x - v, c).double().sum()) / (2 * h)
        assert abs(float(diff) - float(g[:, j].double().sum())) < 2e-3


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("k", [3, 70, 1500, 70001])
def test_masked_rows_may_hold_anything(ft, dtype, k):
    rows = 8
    x, c, old, adv, ref = policy_inputs(rows, k, dtype, seed=2)
    mask = torch.tensor([1, 0, 1, 0, 0, 1, 0, 1], dtype=torch.bool, device=dev())
    check_policy(ft, x, c, old, adv, ref, mask, 0.05, "mean", 1.0)
    clean = [t.clone() for t in (x, c, old, adv, ref)]
    x[1], x[3, 0], x[4] = float("nan"), float("inf"), -float("inf")
    c[1], c[3], c[4] = -1, k, 1 << 40
    old[1], adv[3], ref[4] = float("nan"), float("inf"), float("nan")
    outs = []
    for a in (clean, (x, c, old, adv, ref)):
        leaf = a[0].clone().requires_grad_(True)
        o = ft.policy_loss(leaf, a[1], a[2], a[3], ref_logp=a[4], mask=mask, kl_coef=0.05)
        g, = torch.autograd.grad(o.loss, leaf, retain_graph=True)
        g2, = torch.autograd.grad(o.loss, leaf)
        l = ft.choice_logp(leaf, a[1], mask=mask.to(torch.uint8))
        g3, = torch.autograd.grad(l, leaf, torch.ones(rows, device=dev()))
        assert not g[~mask].any() and not g2[~mask].any() and not g3[~mask].any() and not l[~mask].any() and not o.logp[~mask].any()
        outs.append((*[t.detach() for t in o], g, g2, l.detach(), g3))
    for a, b in zip(*outs):
        assert torch.equal(a, b) and torch.isfinite(a).all()


@pytest.mark.parametrize("k", [4, 900, 70001])
def test_no_valid_row(ft, k):
    x, c, old, adv, ref = policy_inputs(3, k, torch.bfloat16, seed=2)
    leaf = x.fill_(float("nan")).requires_grad_(True)
    o = ft.policy_loss(leaf, c, old, adv, ref_logp=ref, mask=torch.zeros(3, dtype=torch.bool, device=dev()), kl_coef=0.1)
    assert float(o.loss.detach()) == 0.0 and float(o.kl) == 0.0 and float(o.clip_frac) == 0.0
    assert not torch.autograd.grad(o.loss, leaf)[0].any()


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("k", [4, 64, 900, 5000, 70001])
def test_infinities_and_bad_choices(ft, dtype, k):
    """Logits of -inf are choices that cannot be drawn; NaN, +inf, a row of -inf alone and a choice outside the row give NaN in that row alone."""
    x = (rand(8, k, seed=4) * 2.0).to(dtype).to(dev())
    c = torch.zeros(8, dtype=torch.int64, device=dev())
    x[0, 1:3] = -float("inf")
    x[1, 0] = -float("inf")                      # the chosen one: log-probability -inf
    x[2, k - 1] = float("nan")
    x[3, k // 2] = float("inf")
    x[4] = -float("inf")
    c[5], c[6] = k, -1
    x[7] = torch.finfo(dtype).min                # the type's lowest value everywhere: a uniform row
    leaf = x.clone().requires_grad_(True)
    out = ft.choice_logp(leaf, c)
    g, = torch.autograd.grad(out, leaf, torch.ones(8, device=dev()))
    o = out.detach()
    close(o[[0, 7]], plain_logp(x, c)[[0, 7]], U * 20 + row_slack(k), "logp")
    assert o[1] == -float("inf")
    assert o[2:7].isnan().all() and g[2:7].isnan().any(1).all()
    assert torch.isfinite(g[[0, 1, 7]]).all() and (g[0, 1:3] == 0).all() and g[1, 0] == 1.0
    old, adv = torch.full((8,), -1.0, device=dev()), torch.ones(8, device=dev())
    p = ft.policy_loss(leaf, c, old, adv, reduction="sum")
    assert p.loss.isnan()
    gp, = torch.autograd.grad(p.loss, leaf)
    assert gp[5:7].isnan().all() and torch.isfinite(gp[[0, 1, 7]]).all() and (gp[1] == 0).all()


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("k", [24, 300, 3000, 9001, 70001])
def test_infinities_at_every_place_of_a_piece(ft, dtype, k):
    """One special element per row, at 20 neighbouring columns in turn (both halves of a word, pieces' borders, the row's ends): +inf and NaN make the row
    and its gradient NaN, -inf is a choice that cannot be drawn, the type's lowest value is one that never is."""
    n = 20
    cols = torch.cat([torch.arange(n), torch.arange(k - n, k)]).to(dev())
    base, c = rand(2 * n, k, seed=12).to(dtype).to(dev()), (cols + 1) % k
    at = torch.arange(2 * n, device=base.device)
    for value in (math.inf, math.nan, -math.inf, torch.finfo(dtype).min):
        x = base.clone()
        x[at, cols] = value
        leaf = x.clone().requires_grad_(True)
        logp = ft.choice_logp(leaf, c)
        grad, = torch.autograd.grad(logp.sum(), leaf)
        if value in (-math.inf, torch.finfo(dtype).min):
            want = plain_logp(x, c)
            close(logp.detach(), want, U * want.abs() + row_slack(k))
            coef = torch.ones(2 * n, device=base.device)
            close(grad, plain_grad(x, c, coef), grad_tol(x, c, coef, torch.zeros_like(coef, dtype=torch.float64), dtype))
            assert (grad[at, cols] == 0).all()
        else:
            assert logp.isnan().all() and grad.isnan().all()
    x = torch.full((4, k), -math.inf, dtype=dtype, device=base.device)        # the type's lowest value everywhere; -inf everywhere; one element that is left
    x[0] = torch.finfo(dtype).min
    x[2, k // 2] = torch.finfo(dtype).min
    x[3, 1] = torch.finfo(dtype).max
    c = torch.tensor([k - 1, 0, k // 2, 1], device=base.device)
    logp = ft.choice_logp(x, c)
    assert abs(float(logp[0]) + math.log(k)) <= U * (math.log(k) + 8) and bool(logp[1].isnan()) and float(logp[2]) == 0.0 and float(logp[3]) == 0.0


def test_layouts_and_shapes(ft):
    """[replans, agents, K] logits as slices of larger tensors, transposed, unaligned, expanded; a single decision; no rows at all."""
    base = (rand(6, 10, 40, seed=8) * 2).to(dev())
    for dtype in DTYPES:
        big = base.to(dtype)
        views = [big, big[:, :, 3:36], big[:, 2, 1:], big[1:5], big[:, ::2], big.transpose(0, 1), big.transpose(1, 2), big[0, 0].expand(6, 10, 40), big[..., ::3], big[:, 3:4, :7],
                 big.reshape(-1)[1:1 + 59 * 40].view(59, 40), big.reshape(-1)[3:3 + 300 * 7].view(300, 7), big[2, 3], big[..., :1]]
        for v in views:
            assert v.dtype == dtype
            c = torch.randint(0, v.shape[-1], v.shape[:-1], generator=torch.Generator().manual_seed(1)).to(dev())
            want = plain_logp(v, c)
            close(ft.choice_logp(v, c), want, U * want.abs() + row_slack(40), "logp")
            leaf = v.detach().requires_grad_(True)
            out = ft.choice_logp(leaf, c)
            g, = torch.autograd.grad(out.sum(), leaf)           # (the incoming gradient is an expanded scalar)
            close(g, plain_grad(v, c, torch.ones_like(want)), grad_tol(v, c, torch.ones_like(want), torch.zeros_like(want), dtype), "gradient")
            old = want.float() + 0.05
            adv = torch.full((), 0.7, device=dev())             # broadcast
            o = ft.policy_loss(leaf, c, old, adv)
            gp, = torch.autograd.grad(o.loss, leaf)
            n = max(1, c.numel())
            coef = -torch.exp(want - old.double()) * 0.7 / n
            close(gp, plain_grad(v, c, coef), grad_tol(v, c, coef, coef.abs() * (4 * U + row_slack(40)), dtype), "policy gradient")
    cc = torch.zeros(4, 12, dtype=torch.int64, device=dev())[:, ::2]     # choices, masks with strides of their own
    mk = torch.ones(6, 4, dtype=torch.bool, device=dev()).t()
    x = base[:4, :6, :9].contiguous()
    close(ft.choice_logp(x, cc, mask=mk), plain_logp(x, cc), 20 * U + row_slack(9), "strided choice")
    e = torch.zeros(0, 5, device=dev(), requires_grad=True)
    none = torch.zeros(0, dtype=torch.int64, device=dev())
    assert ft.choice_logp(e, none).shape == (0,)
    o = ft.policy_loss(e, none, torch.zeros(0, device=dev()), torch.zeros(0, device=dev()))
    assert float(o.loss) == 0.0 and torch.autograd.grad(o.loss, e)[0].shape == (0, 5)


def test_offsets_beyond_32_bits(ft):
    """4.3 G elements of bfloat16: the last rows lie behind 2^32 elements and 2^33 bytes."""
    rows, k = 32800, 131071
    x = torch.zeros((rows, k), dtype=torch.bfloat16, device=dev())
    c = torch.full((rows,), k - 1, dtype=torch.int64, device=dev())
    x[-3:, -1], x[0, -1] = 5.0, 5.0
    got = ft.choice_logp(x, c)
    want = -math.log(k)
    up = 5.0 - math.log(k - 1 + math.exp(5.0))
    assert torch.allclose(got[[0, -3, -2, -1]].double(), torch.full((4,), up, dtype=torch.float64, device=dev()), atol=1e-5, rtol=0)
    assert ((got[1:-3].double() - want).abs() < 1e-5).all()
    leaf = x.requires_grad_(True)
    o = ft.policy_loss(leaf, c, got, torch.ones(rows, device=dev()), reduction="sum")
    g, = torch.autograd.grad(o.loss, leaf)
    assert abs(float(g[-1, -1]) + 1.0 - math.exp(up)) < 2.0 ** -8 and abs(float(g[-1, 0]) - math.exp(up - 5.0)) < 1e-7 and float(g[-4, -1]) == pytest.approx(-1.0, abs=2.0 ** -8)


@pytest.mark.parametrize("pairs,steps,steps_w", [(1, 1, 1), (3, 0, 2), (2, 5, 0), (16, 8, 8), (65, 33, 31), (300, 257, 300), (5, 4096, 4093), (2100, 3, 3), (1, 70001, 70000)])
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("with_ref", [False, True])
def test_preference_loss(ft, pairs, steps, steps_w, masked, with_ref):
    shapes = {"b": (pairs, steps), "w": (pairs, steps_w)}
    t = {k: (-2.0 + rand(*s, seed=ord(k))).to(dev()) for k, s in shapes.items()}
    ref = {k: (-2.0 + rand(*s, seed=ord(k) + 1)).to(dev()) if with_ref else None for k, s in shapes.items()}
    mask = {k: (torch.rand(s, generator=torch.Generator().manual_seed(ord(k))) < 0.6).to(dev()) if masked else None for k, s in shapes.items()}
    want = {}
    for k in shapes:
        d = t[k].double() - (ref[k].double() if with_ref else 0.0)
        want[k] = torch.where(mask[k], d, 0.0).sum(1) if masked else d.sum(1)
        if masked:                          # (a masked step may hold anything)
            t[k] = torch.where(mask[k], t[k], float("nan"))
    beta, eps = 0.1, 0.1
    z = beta * (want["b"] - want["w"])
    ls = torch.nn.functional.logsigmoid
    loss = -(1 - eps) * ls(z) - eps * ls(-z)
    slope = beta * (torch.sigmoid(z) - (1 - eps))
    for reduction, n in (("mean", pairs), ("sum", 1)):
        b, w = t["b"].clone().requires_grad_(True), t["w"].clone().requires_grad_(True)
        o = ft.preference_loss(b, w, ref["b"], ref["w"], better_mask=mask["b"], worse_mask=mask["w"], beta=beta, label_smoothing=eps, reduction=reduction, scale=2.0)
        close(o.margin, z, U * z.abs() + 1e-12, "margin")
        total = loss.sum() * 2.0 / n
        close(o.loss, total, U * total.abs() + 1e-12, "loss")
        gb, gw = torch.autograd.grad(o.loss, (b, w), retain_graph=True)
        for g, k, sign in ((gb, "b", 1.0), (gw, "w", -1.0)):
            e = (sign * 2.0 / n * slope)[:, None].expand(shapes[k])
            e = torch.where(mask[k], e, 0.0) if masked else e
            close(g, e, 2 * U * e.abs(), "gradient")
        gb2, = torch.autograd.grad(o.loss * -3.0, b)
        close(gb2, gb.double() * -3.0, 2 * U * 3 * gb.double().abs(), "gradient of a multiple")
    with torch.no_grad():
        assert torch.equal(ft.preference_loss(t["b"], t["w"], ref["b"], ref["w"], better_mask=mask["b"], worse_mask=mask["w"], beta=beta).margin, o.margin)


def test_preference_extremes(ft):
    """Saturated pairs stay finite, sums given as [pairs], one-sided gradients, NaN in a valid step."""
    b = torch.tensor([1e4, -1e4, 0.0, 3e38], device=dev()).requires_grad_(True)
    w = torch.zeros(4, device=dev())
    o = ft.preference_loss(b, w, beta=1.0, reduction="sum")
    assert float(o.loss) == pytest.approx(1e4 + math.log(2.0), rel=1e-6)
    g, = torch.autograd.grad(o.loss, b)
    assert g.tolist() == [0.0, -1.0, -0.5, 0.0]
    bad = torch.tensor([[1.0, float("nan")]], device=dev())
    assert ft.preference_loss(bad, bad[:, :1]).loss.isnan()


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("sizes", [[1], [3, 0, 7], [5000], [100003], [1, 2, 3, 65536, 65537, 32767, 9], [17] * 700, [1 << 20, 5, (1 << 20) + 1]])
@pytest.mark.parametrize("max_norm", [0.5, 1e6])
def test_clip_grads(ft, dtype, sizes, max_norm):
    gs = [(rand(n, seed=i) * 0.1).to(dtype).to(dev()) for i, n in enumerate(sizes)]
    want = [g.double() for g in gs]
    norm = torch.sqrt(sum((g * g).sum() for g in want))
    got = ft.clip_grads_(gs, max_norm)
    assert got.dtype == torch.float32 and got.shape == ()
    close(got, norm, U * 1.01 * norm, "norm")
    c = min(1.0, max_norm / (float(norm) + 1e-6))
    for g, w in zip(gs, want):
        assert g.dtype == dtype
        if c == 1.0:
            assert torch.equal(g.double(), w)
        else:
            close(g, w * c, (w * c).abs() * (torch.finfo(dtype).eps / 2 + 3 * U) + (2.0 ** -25 if dtype == torch.float16 else 0.0), "scaled")


def test_clip_grads_beyond_32_bits(ft):
    """One tensor of more than 2^31 elements (a table takes 2^31 of a range at most), its values at both ends and around the seam."""
    n = (1 << 31) + 12347
    g = torch.zeros(n, dtype=torch.bfloat16, device=dev())
    at = torch.tensor([0, 1, 4095, (1 << 31) - 1, 1 << 31, (1 << 31) + 1, n - 2, n - 1], device=dev())
    g[at] = 3.0
    other = torch.full((5,), 4.0, device=dev())
    norm = math.sqrt(8 * 9.0 + 5 * 16.0)
    assert float(ft.clip_grads_([g, other], 1.0)) == pytest.approx(norm, rel=1e-7)
    assert (g[at].double() - 3.0 / norm).abs().max() < 3.0 / norm * 2.0 ** -8 and (other.double() - 4.0 / norm).abs().max() < 1e-6
    assert int(torch.count_nonzero(g)) == 8


def test_clip_grads_mixed_lists(ft):
    """Types mixed, views of one buffer at odd offsets, other orders of dimensions, None entries, neighbours left as they were."""
    flat = rand(100000, seed=5).to(dev())
    keep = flat.clone()
    half = rand(5001, seed=6).to(torch.bfloat16).to(dev())
    gs = [flat[1:78], flat[79:1079], half[1:], None, flat[2000:2000 + 35 * 21].view(35, 21).t(), rand(3, 4, 5, 6, seed=7).half().to(dev()).permute(0, 2, 3, 1), torch.zeros(0, device=dev()), flat[99999:]]
    before = [None if g is None else g.double().clone() for g in gs]
    norm = math.sqrt(sum(float((b * b).sum()) for b in before if b is not None))
    got = ft.clip_grads_(gs, 1.0)
    assert float(got) == pytest.approx(norm, rel=1e-6)
    for g, b in zip(gs, before):
        if g is not None:
            w = b / (norm + 1e-6)
            close(g, w, w.abs() * (torch.finfo(g.dtype).eps / 2 + 3 * U) + 2.0 ** -25, "scaled")
    touched = torch.zeros(100000, dtype=torch.bool, device=dev())
    for a, e in ((1, 78), (79, 1079), (2000, 2735), (99999, 100000)):
        touched[a:e] = True
    assert torch.equal(flat[~touched], keep[~touched])


def test_clip_grads_extremes(ft):
    one = lambda v, n=5, dt=torch.float32: torch.full((n,), v, dtype=dt, device=dev())
    g = [one(3e37)]
    assert float(ft.clip_grads_(g, 1.0)) == pytest.approx(3e37 * math.sqrt(5), rel=1e-6) and float(g[0][0]) == pytest.approx(1 / math.sqrt(5), rel=1e-6)
    g = [one(1e-30)]
    assert float(ft.clip_grads_(g, 1.0)) == pytest.approx(1e-30 * math.sqrt(5), rel=1e-6) and torch.equal(g[0], one(1e-30))
    g = [one(0.0)]
    assert float(ft.clip_grads_(g, 1.0)) == 0.0 and torch.equal(g[0], one(0.0))
    g = [one(2.0), one(float("nan"), 1)]
    assert ft.clip_grads_(g, 1.0).isnan() and g[0].isnan().all()
    g = [one(2.0), one(float("inf"), 1)]
    assert ft.clip_grads_(g, 1.0) == float("inf") and (g[0] == 0).all() and g[1].isnan().all()
    g = [one(2.0)]
    assert float(ft.clip_grads_(g, float("inf"))) == pytest.approx(2 * math.sqrt(5)) and torch.equal(g[0], one(2.0))
    assert float(ft.clip_grads_(g, 0.0)) > 0 and torch.equal(g[0], one(0.0))


def test_refusals(ft):
    x, c = torch.zeros(2, 3, device=dev()), torch.zeros(2, dtype=torch.int64, device=dev())
    f = torch.zeros(2, device=dev())
    for bad in (lambda: ft.choice_logp(x.double(), c), lambda: ft.choice_logp(x, c.float()), lambda: ft.choice_logp(x, c, mask=f), lambda: ft.policy_loss(x, c, f.half(), f)):
        with pytest.raises(TypeError):
            bad()
    for bad in (lambda: ft.choice_logp(x, c[:1]), lambda: ft.choice_logp(x, c.cpu()), lambda: ft.choice_logp(x[:, :0], c), lambda: ft.choice_logp(x.sum(), c[0]),
                lambda: ft.choice_logp(x, c, mask=torch.ones(3, dtype=torch.bool, device=dev())), lambda: ft.policy_loss(x, c, f[:1], f), lambda: ft.policy_loss(x, c, f, torch.zeros(3, device=dev())),
                lambda: ft.policy_loss(x, c, f, f, kl_coef=0.1), lambda: ft.policy_loss(x, c, f, f, clip_low=2.0), lambda: ft.policy_loss(x, c, f, f, reduction="none"),
                lambda: ft.policy_loss(x, c, f, f, kl_coef=-1.0), lambda: ft.policy_loss(x, c, f, f, scale=float("nan")),
                lambda: ft.preference_loss(x, x[:1]), lambda: ft.preference_loss(x, x, x[:, :2]), lambda: ft.preference_loss(x, x, label_smoothing=2.0), lambda: ft.preference_loss(x[:0], x[:0]),
                lambda: ft.clip_grads_([], 1.0), lambda: ft.clip_grads_([x, x], 1.0), lambda: ft.clip_grads_([x, x[1]], 1.0), lambda: ft.clip_grads_([x[:, :2]], 1.0),
                lambda: ft.clip_grads_([f[:1].expand(4)], 1.0), lambda: ft.clip_grads_([x], -1.0), lambda: ft.clip_grads_([x], float("nan")), lambda: ft.clip_grads_([x.cpu()], 1.0),
                lambda: ft.clip_grads_([torch.zeros(2, device=dev(), requires_grad=True)], 1.0)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        ft.clip_grads_([x.double()], 1.0)
    leaf = x.clone().requires_grad_(True)            # a gradient of a gradient
    g, = torch.autograd.grad((ft.choice_logp(leaf, c) ** 2).sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
    with pytest.raises(RuntimeError):                # changed between the passes: autograd's own check
        leaf = (x + 1).requires_grad_(True)
        y = ft.choice_logp(leaf * 1.0, c)
        z = leaf * 1.0
        out = ft.choice_logp(z, c)
        z.add_(1.0)
        out.sum().backward()
    assert y is not None


def test_tensors_whose_memory_is_not_their_value(ft):
    """The imaginary part of a conjugate is a view with a flag for its sign, torch's efficient zeros have no memory: refused as inputs, right as incoming
    gradients."""
    x, c, f = rand(6, 5, seed=4).to(dev()), torch.arange(6, device=dev()) % 5, rand(6, seed=5).to(dev())
    neg = lambda t: torch.complex(t, -t).conj().imag          # = t
    zero = lambda *s: torch._efficientzerotensor(s, device=dev(), dtype=torch.float32)
    assert neg(x).is_neg() and zero(6)._is_zerotensor()
    for bad in (lambda: ft.choice_logp(neg(x), c), lambda: ft.choice_logp(zero(6, 5), c), lambda: ft.policy_loss(x, c, neg(f), f), lambda: ft.policy_loss(x, c, f, zero(6)),
                lambda: ft.policy_loss(x, c, f, f, ref_logp=zero(6)), lambda: ft.preference_loss(f, neg(f)), lambda: ft.preference_loss(f, f, zero(6)), lambda: ft.clip_grads_([f, neg(x)], 1.0),
                lambda: ft.clip_grads_([zero(6)], 1.0)):
        with pytest.raises(ValueError):
            bad()
    a, b = x.clone().requires_grad_(True), f.clone().requires_grad_(True)
    one = torch.full((), 0.75, device=dev())
    for out, leaf, g, none in ((lambda: ft.choice_logp(a, c), a, f, zero(6)), (lambda: ft.policy_loss(a, c, f, f).loss, a, one, zero()), (lambda: ft.preference_loss(b, f * 2).loss, b, one, zero())):
        want, = torch.autograd.grad(out(), leaf, g)
        got, = torch.autograd.grad(out(), leaf, neg(g))
        assert torch.equal(got, want) and want.abs().max() > 0
        assert (torch.autograd.grad(out(), leaf, none)[0] == 0).all()


def test_calls_from_several_threads(ft):
    """Four host threads, each on a stream of its own, at once."""
    from concurrent.futures import ThreadPoolExecutor
    inputs = [policy_inputs(33, 1500 + 100 * i, torch.float16, seed=i) for i in range(4)]
    def once(a):
        x, c, old, adv, ref = a
        leaf = x.detach().requires_grad_(True)
        o = ft.policy_loss(leaf, c, old, adv, ref_logp=ref, kl_coef=0.1)
        g, = torch.autograd.grad(o.loss, leaf)
        return [o.loss.detach(), o.logp, g, ft.clip_grads_([g.clone(), old.clone()], 0.1)]
    want = [once(a) for a in inputs]
    torch.cuda.synchronize()
    def loop(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            got = [once(inputs[i]) for _ in range(20)]
            torch.cuda.current_stream().synchronize()
        return got
    with ThreadPoolExecutor(4) as pool:
        for i, got in enumerate(pool.map(loop, range(4))):
            for r in got:
                for a, b in zip(r, want[i]):
                    assert torch.equal(a, b)


def test_equal_inputs_give_equal_bits_on_any_stream(ft):
    x, c, old, adv, ref = policy_inputs(97, 3001, torch.bfloat16, seed=31)
    leaf = x.requires_grad_(True)
    def once():
        o = ft.policy_loss(leaf, c, old, adv, ref_logp=ref, kl_coef=0.02)
        g, = torch.autograd.grad(o.loss, leaf)
        gs = [g.float(), old.clone()]
        return [o.loss.detach(), o.kl, o.logp, g, ft.clip_grads_(gs, 0.1), *gs]
    first = once()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    results = []
    for _ in range(4):
        for s in streams:                   # three calls in flight at once
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                results.append(once())
    torch.cuda.synchronize()
    for r in results:
        for a, b in zip(r, first):
            assert torch.equal(a, b)


def test_captured_step(ft):
    """The whole step in a graph, replayed on new inputs with eager calls between, each replay against the eager result; and a second graph of the same kind."""
    rows, k = 40, 777
    xs = [policy_inputs(rows, k, torch.bfloat16, seed=s) for s in range(4)]
    mask = torch.rand(rows, generator=torch.Generator().manual_seed(5)).to(dev()) < 0.8
    def step(x, c, old, adv, ref):
        leaf = x.detach().requires_grad_(True)
        o = ft.policy_loss(leaf, c, old, adv, ref_logp=ref, mask=mask, kl_coef=0.02)
        g, = torch.autograd.grad(o.loss, leaf)
        lp = ft.choice_logp(leaf, c, mask=mask)
        pref = ft.preference_loss(lp[:20].view(4, 5), lp[20:].view(4, 5), ref[:20].view(4, 5), ref[20:].view(4, 5))
        g2, = torch.autograd.grad(pref.loss, leaf)
        norm = ft.clip_grads_([g, g2], 0.01)
        return [o.loss.detach(), o.logp, o.kl, o.clip_frac, pref.loss.detach(), g, g2, norm]
    want = [[t.clone() for t in step(*x)] for x in xs]
    graphs = []
    for _ in range(2):
        static = [t.clone() for t in xs[0]]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(*static)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(*static)
        graphs.append((graph, static, out))
    for turn in range(6):
        for (graph, static, out), i in zip(graphs, (turn % 4, (turn + 1) % 4)):
            for s, t in zip(static, xs[i]):
                s.copy_(t)
            graph.replay()
            step(*xs[(turn + 2) % 4])                    # eager work between
            torch.cuda.synchronize()
            for a, b in zip(out, want[i]):
                assert torch.equal(a, b)


def test_a_fine_tuning_run_on_engine_rollouts(ft):
    """The operators as they are used: a head over the engine's policy embeddings draws the motion mode of every replan and agent, M replicas of a scene roll out
    with the drawn modes, the device metric scores them, and the losses' gradients update the head.  Checked: the run, its numbers and gradients against the
    same step in 64 bits."""
    from prosim_amd import synth, weights
    from prosim_amd.engine import Engine
    from prosim_amd.spec import SMALL_SPEC
    spec = SMALL_SPEC.replace(motion_k=3, rollout_top_k=3)
    M, N, K = 4, 6, spec.motion_k
    scene = synth.make_scene(spec, N, 24, batch=1, seed=3, replay=0.3)
    eng = Engine(spec, weights.init_weights(spec, 0))
    try:
        eng.set_replicas(M)
        eng.set_scene(scene)
        eng.encode_scene()
        eng.generate_policy()
        eng.sync()
        A, R = eng.num_agents, spec.n_replans
        emd = torch.from_numpy(eng.get("policy_emd").astype(np.float32)).to(dev())          # [A, hidden], replica-major
        valid = torch.from_numpy(eng.policy_rows.astype(bool)).to(dev())[None].expand(R, A)
        head = (rand(R, emd.shape[1], K, seed=2) * 0.1).to(dev()).requires_grad_(True)
        logits = torch.bmm(emd[None].expand(R, -1, -1).contiguous(), head)
        drawn = torch.distributions.Categorical(logits=logits.detach().cpu()).sample().to(torch.int32)       # [R, A]
        old = ft.choice_logp(logits.detach(), drawn.to(dev()), mask=valid)
        table = np.zeros((R, M, N), np.int32)
        slots = np.asarray(eng.row_slots)
        table.reshape(R, M * N)[:, slots] = drawn.numpy()
        eng.set_mode_choice(table)
        eng.rollout()
        score = torch.zeros(A, 2, device=dev())
        torch.cuda.synchronize()
        eng.rollout_metric(score.data_ptr())
        eng.sync()
        reward = -torch.nan_to_num(score[:, 0]).view(M, -1)
        adv = ((reward - reward.mean(0)) / (reward.std(0) + 1e-3)).reshape(-1)               # [A]: one score per rollout, over all replans
        assert torch.isfinite(adv).all()
        ref = old - 0.1
        out = ft.policy_loss(logits, drawn.to(dev()), old, adv, ref_logp=ref, mask=valid, kl_coef=0.1)
        policy_grad, = torch.autograd.grad(out.loss, head, retain_graph=True)
        lp = ft.choice_logp(logits, drawn.to(dev()), mask=valid)
        half = A // 2
        pref = ft.preference_loss(lp[:, :half].t(), lp[:, half:2 * half].t(), ref[:, :half].t(), ref[:, half:2 * half].t(), better_mask=valid[:, :half].t(),
                                  worse_mask=valid[:, half:2 * half].t())
        pref_grad, = torch.autograd.grad(pref.loss, head)
        # the same step in 64 bits
        h64 = head.detach().double().requires_grad_(True)
        l64 = torch.bmm(emd[None].expand(R, -1, -1).double().contiguous(), h64)
        lp64 = torch.log_softmax(l64, -1).gather(-1, drawn.to(dev()).long()[..., None])[..., 0]
        ratio = torch.exp(lp64 - old.double())
        a64 = adv.double()[None].expand(R, A)
        per = -torch.minimum(ratio * a64, ratio.clamp(0.8, 1.2) * a64) + 0.1 * (torch.exp(ref.double() - lp64) - (ref.double() - lp64) - 1.0)
        v = valid.double()
        loss64 = (per * v).sum() / v.sum()
        g64, = torch.autograd.grad(loss64, h64, retain_graph=True)
        d64 = (lp64 - ref.double()) * v
        hp = d64[:, :half].sum(0) - d64[:, half:2 * half].sum(0)
        p64 = -torch.nn.functional.logsigmoid(0.1 * hp).mean()
        gp64, = torch.autograd.grad(p64, h64)
        # float32 products over 128 terms and sums over A rows: a few hundred roundings of the largest entries
        tol = lambda g: 600 * U * float(g.abs().max()) + 1e-9
        assert float(out.clip_frac) == 0.0 and abs(float(out.loss) - float(loss64)) < 1e-5 and abs(float(pref.loss) - float(p64)) < 1e-5
        assert float((policy_grad.double() - g64).abs().max()) < tol(g64) and float((pref_grad.double() - gp64).abs().max()) < tol(gp64)
        grads = [policy_grad, pref_grad]
        norm = ft.clip_grads_(grads, 1e-3)
        n64 = math.sqrt(float((g64 ** 2).sum() + (gp64 ** 2).sum()))
        assert float(norm) == pytest.approx(n64, rel=1e-4) and n64 > 1e-3
        with torch.no_grad():
            head -= grads[0] + grads[1]
        assert torch.isfinite(head).all()
    finally:
        eng.close()
