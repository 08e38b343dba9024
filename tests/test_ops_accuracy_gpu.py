"""Where the operators of dream_go_amd.ops could lose digits that their formulas keep, against 64 bits, on a GPU.

Every tolerance counts half steps of fp32 (ULP) along the longest run of roundings that the form under test has, and the one rounding of the result."""
import math

import pytest

from test_ops_gpu import TYPES, ULP, close, gen, group_norm64, group_norm_case

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def ops(api):
    from dream_go_amd import ops as module
    return module


# ---- group norm ---------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("n,p,c,groups,dtype", [(512, 65536, 64, 8, "fp16"), (512, 32768, 64, 8, "fp32"), (1, 1 << 24, 64, 32, "bf16")])
def test_group_norm_of_flat_maps_behind_a_border(ops, n, p, c, groups, dtype):
    """The first rows lie far from all others, which are equal, and a thread adds up a thousand of them: what each of them adds to the variance is
    rounded the same way every time.  The moments are joined eight rows at a time, at most 2048 / 8 = 256 joins, each within a few half steps."""
    x = torch.full((n, p, c), 0.123, dtype=TYPES[dtype], device="cuda")
    border, edge, flat = 64, 1000.0, float(x[0, 0, 0])
    x[:, :border] = edge
    y = ops.group_norm(x, groups, eps=0.0)
    f = border / p
    mean, sd = f * edge + (1 - f) * flat, (edge - flat) * math.sqrt(f * (1 - f))
    for part, value in ((y[:, :border], edge), (y[:, border:], flat)):
        want = (value - mean) / sd
        slack = 512 * ULP * (abs(want) + (abs(value) + abs(mean)) / sd)
        bound = torch.finfo(y.dtype).eps / 2 * (abs(want) + slack) + slack
        low, high = float(part.min()), float(part.max())
        assert abs(low - want) <= bound and abs(high - want) <= bound, (value, low, high, want, bound)


@pytest.mark.parametrize("shape,groups", [((1, 40000, 64), 8), ((2, 33333, 24), 3), ((1, 70001, 8), 1)])
def test_group_norm_of_huge_values_that_differ_little(ops, shape, groups):
    """Around 2^70 the square of a value is no number of fp32 any more; differences from the mean of at most 2^56 have squares of which half a million add
    up to less than 2^128.  The last share of the positions has threads without a row."""
    step = torch.finfo(torch.float32).eps * 2.0 ** 70
    x = (2.0 ** 70 + step * torch.randint(0, 500, shape, generator=gen(5)).double()).float()
    pre, _ = group_norm64(x, groups, None, None, None, 0.0)
    n, p, c = shape
    v = x.double().reshape(n, p, groups, c // groups)
    scale = (1 / v.std((1, 3), unbiased=False, keepdim=True)).expand_as(v).reshape(shape)
    # the mean is off by 64 half steps of its size at most, the variance by the square of that beside itself
    off = 64 * ULP * 2.0 ** 70 * scale
    close(ops.group_norm(x.cuda(), groups, eps=0.0), pre, off + (64 * ULP + off * off) * pre.abs(), (shape, groups))


@pytest.mark.parametrize("shape,groups", [((2, 361, 64), 8), ((3, 7, 30), 3), ((1, 1000, 90), 9), ((1, 50000, 16), 4), ((2, 20000, 40), 4)])
def test_group_norm_keeps_the_variance_of_values_far_from_zero(ops, shape, groups):
    """A mean fifteen hundred away: squares of values differ in their last bits only.  No thread here adds up more than 8 rows of 8 values one after the
    other, trees join the rest: 96 half steps are more than either form has."""
    serial = 96
    n, p, c = shape
    x = (torch.randn(shape, generator=gen(3)) + 1500.0).float()
    v = x.double().reshape(n, p, groups, c // groups)
    d = v - v.mean((1, 3), keepdim=True)
    var = (d * d).mean((1, 3), keepdim=True)
    y = ops.group_norm(x.cuda(), groups, eps=0.0).cpu()
    off = serial * ULP * 1500.0 / var.sqrt()                                   # of the mean, in standard deviations
    got = y.double().reshape(v.shape)
    assert ((got - d / var.sqrt()).abs() <= off + (serial * ULP + off * off) * (d / var.sqrt()).abs()).all()
    spread = got.var((1, 3), unbiased=False)
    assert ((spread - 1).abs() <= 2 * serial * ULP + (off * off).reshape(spread.shape)).all(), spread


def test_group_norm_of_nearly_two_to_the_31_channels(ops):
    """The last vector of a row begins eight channels in front of 2^31 and ends inside it."""
    c, pad = 2147483646, 16
    buffer = torch.empty(c + pad, dtype=torch.bfloat16, device="cuda").normal_(generator=torch.Generator(device="cuda").manual_seed(1))
    buffer[c:] = math.nan
    x, bias = buffer[:c].view(1, 1, c), torch.empty(c, dtype=torch.bfloat16, device="cuda").fill_(0.5)
    out = torch.full((c + pad,), 3.0, dtype=torch.bfloat16, device="cuda")
    y = out[:c].view(1, 1, c)
    assert ops.group_norm(x, c // 2, None, bias, out=y) is y
    for begin in (0, (1 << 30) - 4, c - (1 << 20)):                            # pairs of channels: each is half their difference from the mean
        pair = x[0, 0, begin:begin + (1 << 20)].double().view(-1, 2)
        d = (pair - pair.mean(1, keepdim=True))
        want = (d / torch.sqrt((d * d).mean(1, keepdim=True) + 1e-5) + 0.5).flatten()
        got = y[0, 0, begin:begin + (1 << 20)].double()
        slack = 32 * ULP * (1 + want.abs())
        assert ((got - want).abs() <= 2.0 ** -8 * (want.abs() + slack) + slack).all()
    assert not y.isnan().any() and (out[c:] == 3.0).all()


@pytest.mark.parametrize("shape,groups", [((96, 43, 195), 65), ((192, 43, 189), 63), ((96, 72, 455), 65)])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_group_norm_with_all_the_lds_it_may_ask_for(ops, shape, groups, dtype):
    """1024 threads with one number for each of eight channels: 66048 bytes are the most that a call asks for."""
    group_norm_case(ops, shape, groups, TYPES[dtype], "relu", affine=TYPES[dtype], residual=True, seed=groups)


# ---- dense: the activations -----------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype,out", [("fp16", "fp32"), ("bf16", "fp32"), ("bf16", "bf16")])
def test_gelu_keeps_its_digits(ops, dtype, out):
    """x * 1 is exact, so what shows is the activation alone.  v Phi(v), with the tail Phi(-|v|) = exp(-v^2 / 2) P: the exponent is off by 2.5 half steps of its
    size (the square, the factor log2(e) / 2 and the product with it), exp2 and the reciprocal by a step each, P and the products by 12 half steps, beside
    2.5 of the polynomial itself; 1 - tail and the last product by 1.5."""
    t = TYPES[dtype]
    v = torch.cat([torch.linspace(-12.5, 12.5, 40001, dtype=torch.float64), torch.logspace(-6, 1, 4001, dtype=torch.float64), -torch.logspace(-6, 1, 4001, dtype=torch.float64)]).to(t)
    y = ops.dense(v[:, None].cuda(), torch.ones(1, 1, dtype=t, device="cuda"), activation="gelu", out_dtype=TYPES[out])[:, 0]
    d = v.double()
    tail = 0.5 * torch.special.erfc(d.abs() / math.sqrt(2.0))
    slack = ULP * d.abs() * (tail * (1.25 * d * d + 20) + torch.where(d < 0, tail * 0, 1.5 + tail * 0))
    close(y, torch.where(d < 0, d * tail, d * (1 - tail)), slack, (dtype, out))


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_tanh_keeps_its_digits(ops, dtype):
    """Up to 0.7 an odd polynomial: the square, its products with the coefficients and the last two roundings, 3 half steps. Beyond, 1 - w with w = 2 / (exp(2 |x|) + 1):
    w is off by 2 |x| half steps of the exponent, two each of exp2 and the reciprocal and one of the sum; the difference is what is rounded to the result."""
    t = TYPES[dtype]
    v = torch.cat([torch.linspace(-12, 12, 40001, dtype=torch.float64), torch.logspace(-6, 1, 4001, dtype=torch.float64), -torch.logspace(-6, 1, 4001, dtype=torch.float64)]).to(t)
    y = ops.dense(v[:, None].cuda(), torch.ones(1, 1, dtype=t, device="cuda"), activation="tanh", out_dtype=torch.float32)[:, 0]
    d = v.double()
    w = 2 / (torch.exp(2 * d.abs()) + 1)
    close(y, torch.tanh(d), ULP * torch.where(d.abs() < 0.7, 2 * d.abs(), w * (2 * d.abs() + 5)), dtype)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_silu_keeps_its_digits(ops, dtype):
    """v / d with d = 1 + exp(-v) = 1 + exp2(v log2(e)): the exponent is off by one half step of its size for the product and by 0.23 of one for the factor, whose
    nearest number of fp32 is 1.93e-8 below 1.442695, a relative 1.34e-8 = 0.23 * 2^-24; exp2 by a step.  Of d that is the part 1 - 1 / d; the sum is rounded once,
    and the quotient once, which is the result's own rounding."""
    t = TYPES[dtype]
    v = torch.cat([torch.linspace(-60, 60, 40001, dtype=torch.float64), torch.logspace(-6, 1, 4001, dtype=torch.float64), -torch.logspace(-6, 1, 4001, dtype=torch.float64)]).to(t)
    one = torch.ones(1, 1, dtype=t, device="cuda")
    y = ops.dense(v[:, None].cuda(), one, activation="silu", out_dtype=torch.float32)[:, 0]
    d = v.double()
    ref, part = d / (1 + torch.exp(-d)), 1 - 1 / (1 + torch.exp(-d))
    close(y, ref, ULP * ref.abs() * (part * (1.23 * d.abs() + 2.5) + 1), dtype)
    # as 16 bits, and of infinities: v / (1 + exp(-v)) is infinite, and of minus infinity no number
    assert torch.equal(ops.dense(v[:, None].cuda(), one, activation="silu")[:, 0].isnan().cpu(), v.isnan())
    x = torch.tensor([[math.inf], [-math.inf], [math.nan], [100.0], [-100.0], [0.0], [-3e4]], dtype=t, device="cuda")
    for out in (torch.float32, t):
        got = ops.dense(x, one, activation="silu", out_dtype=out)[:, 0].float().cpu()
        assert got[0] == math.inf and got[1].isnan() and got[2].isnan() and got[3] == 100 and (got[4:].abs() < 1e-30).all(), got


# ---- logits -----------------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("b,v", [(3, 362), (5, 20011)])
def test_a_repetition_divides(ops, b, v):
    """One rounding, that of l / repetition or l * repetition: the bits are those of the one operation."""
    g = gen(8)
    logits = torch.randn(b, v, generator=g) * 5
    history = torch.arange(v, dtype=torch.int32).expand(b, v).contiguous()
    r = torch.rand(b, generator=g) + 0.7
    want = torch.where(logits > 0, logits / r[:, None], logits * r[:, None])
    assert torch.equal(ops.adjust_logits(logits.cuda(), history=history.cuda(), repetition=r.cuda()).cpu(), want)
    # where 1 / repetition is no number of fp32, l / repetition may be one
    tiny = torch.full((b,), 2.0 ** -130)
    small = logits * 2.0 ** -100
    got = ops.adjust_logits(small.cuda(), history=history.cuda(), repetition=tiny.cuda()).cpu()
    assert torch.equal(got[small > 0], (small / tiny[:, None])[small > 0])


# ---- what a call leaves behind, and what it refuses ---------------------------------------------------------------------------------------

def test_forward_mode_tangents_are_refused(ops, api):
    """A dual tensor does not ask for gradients; its tangent would be lost all the same."""
    import torch.autograd.forward_ad as forward
    h = torch.ones(4, 16, dtype=torch.float16, device="cuda")
    maps, logits, history = h.view(2, 2, 16), h.float(), torch.zeros(4, 3, dtype=torch.int32, device="cuda")
    with forward.dual_level():
        def dual(t): return forward.make_dual(t, torch.ones_like(t))           # noqa: E306,E704
        calls = [lambda: ops.dense(dual(h), h), lambda: ops.dense(h, dual(h)), lambda: ops.dense(h, h, dual(h[0, :4].contiguous())),
                 lambda: ops.dense(h, h, residual=dual(h[:, :4].contiguous())), lambda: ops.group_norm(dual(maps), 4), lambda: ops.group_norm(maps, 4, dual(h[0])),
                 lambda: ops.group_norm(maps, 4, residual=dual(maps)), lambda: ops.adjust_logits(dual(logits)), lambda: ops.adjust_logits(logits, bias=dual(logits)),
                 lambda: ops.adjust_logits(logits, history=history, frequency=dual(logits[:, 0].contiguous()))]
        for run in calls:
            for mode in (torch.enable_grad, torch.no_grad):                    # (no_grad does not stop tangents: torch's own operators carry them on)
                with mode(), pytest.raises(api.Error) as e:
                    run()
                assert e.value.status == api.UNSUPPORTED
        assert ops.dense(h, h).shape == (4, 4)                                 # nothing here has a tangent
        assert ops.dense(forward.unpack_dual(dual(h)).primal, h).shape == (4, 4)
    assert ops.dense(h, h).shape == (4, 4)


def test_a_result_written_over_a_saved_tensor_is_noticed(ops):
    """What autograd keeps for a backward pass and an operator then writes over: the backward pass says so, as behind torch's own operators."""
    h = torch.ones(4, 4, dtype=torch.float16, device="cuda")
    maps = torch.ones(2, 2, 4, device="cuda")
    logits = torch.ones(4, 4, device="cuda")
    for out, run in ((h.clone(), lambda o: ops.dense(h, h, out=o)), (maps.clone(), lambda o: ops.group_norm(maps, 2, out=o)), (logits.clone(), lambda o: ops.adjust_logits(logits, out=o))):
        leaf = torch.ones_like(out, requires_grad=True)
        loss = (leaf * out).sum()
        before = out._version
        assert run(out) is out and out._version > before
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
    with torch.inference_mode():
        buffer = torch.empty(4, 4, dtype=torch.float16, device="cuda")
        assert ops.dense(h, h, out=buffer) is buffer


def test_numbers_that_are_none_are_refused(ops, api):
    h = torch.ones(4, 16, dtype=torch.float16, device="cuda")
    maps, logits, history = h.view(2, 2, 16), h.float(), torch.zeros(4, 3, dtype=torch.int32, device="cuda")
    learned = torch.tensor(0.5, device="cuda", requires_grad=True)
    bad = [lambda: ops.dense(h, h, alpha2="2"), lambda: ops.dense(h, h, alpha1=None), lambda: ops.dense(h, h, alpha1=learned),
           lambda: ops.dense(h, h, residual=h[:, :4].contiguous(), alpha2=learned), lambda: ops.group_norm(maps, 4, eps=1e39), lambda: ops.group_norm(maps, 4, eps=None),
           lambda: ops.group_norm(maps, 4, eps=learned), lambda: ops.group_norm(maps, 4.0), lambda: ops.group_norm(maps, None), lambda: ops.group_norm(maps[..., :0], 1 << 70),
           lambda: ops.adjust_logits(logits, repetition=1e39), lambda: ops.adjust_logits(logits, history=history, presence=None),
           lambda: ops.adjust_logits(logits, history=history, frequency="much"), lambda: ops.adjust_logits(logits, history=history, frequency=learned)]
    for n, run in enumerate(bad):
        with pytest.raises(api.Error) as e:
            run()
        assert e.value.status in (api.BAD_ARGUMENT, api.UNSUPPORTED), n
    with torch.no_grad():
        assert torch.equal(ops.dense(h, h, alpha1=learned), ops.dense(h, h, alpha1=0.5))


def test_operands_that_are_no_tensors_are_refused(ops, api):
    h, f = torch.ones(4, 16, dtype=torch.float16, device="cuda"), torch.ones(4, 16, device="cuda")
    bad = [lambda: ops.dense(h, h, out=5), lambda: ops.dense(h, h, out=h.cpu().numpy()), lambda: ops.dense(h, h, activation=["relu"]), lambda: ops.dense([h], h),
           lambda: ops.dense(h, h, out_dtype="fp16"), lambda: ops.dense(h, None), lambda: ops.dense(h, h, residual=0.0), lambda: ops.group_norm(f, 4, out=5),
           lambda: ops.group_norm(f, 4, 1.0), lambda: ops.group_norm(f, 4, activation={}), lambda: ops.adjust_logits(f, out=5), lambda: ops.adjust_logits(f, mask=[1]),
           lambda: ops.adjust_logits(f, bias=1.0), lambda: ops.adjust_logits(f, history=[[1]]), lambda: ops.adjust_logits(f, history=torch.zeros(4, 1, dtype=torch.int32, device="cuda"), lengths=1)]
    for n, run in enumerate(bad):
        with pytest.raises(api.Error) as e:
            run()
        assert e.value.status in (api.BAD_ARGUMENT, api.UNSUPPORTED), n
