"""The operators of dream_go_amd.ops against their formulas in 64 bits, on a GPU.

Tolerances.  A result is rounded once, by at most half a step of its type.  In front of that:
  dense         with small whole numbers every product and every sum is a whole number (or a half) below 2^24: exact in fp32, in any order, so
                the outputs have to be THE rounded values.  Activations add the error of their fp32 evaluation: ACT steps of fp32.
  group_norm    mean and variance are sums of at most SERIAL values in a row joined by trees: each is off by SERIAL + 16 steps of fp32
                relative to the sum of the magnitudes, and (x - mean) * scale * weight + bias + z by a handful more.
  adjust_logits six operations in fp32, each off by half a step of its result.
"""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

ULP = 2.0 ** -24            # half a step of fp32, relative
ACT = 16                    # half steps of fp32 within which an activation's own evaluation stays
SERIAL = 512
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -140}   # half a step among the subnormals (fp32: and what is flushed)
ACTIVATIONS = ("identity", "relu", "tanh", "gelu", "silu")


@pytest.fixture(scope="module")
def ops(api):
    from dream_go_amd import ops as module
    return module


def gen(seed):
    return torch.Generator().manual_seed(seed)


def act64(v, name):
    if name == "relu":
        return torch.where(v < 0, torch.zeros_like(v), v)
    if name == "tanh":
        return torch.tanh(v)
    if name == "gelu":
        return 0.5 * v * torch.special.erfc(-v / math.sqrt(2.0))
    if name == "silu":
        return v / (1.0 + torch.exp(-v))
    return v


def close(out, ref, slack, what):
    """|out - ref| <= half a step of out's type + slack, and the same infinities and NaNs."""
    o, r = out.double().cpu(), ref
    limit = torch.finfo(out.dtype).max
    half = torch.finfo(out.dtype).eps / 2
    r = torch.where(r.isfinite() & (r.abs() > limit * (1 + half)), torch.sign(r) * math.inf, r)
    fine = r.isfinite()
    assert torch.equal(o.isnan(), r.isnan()), what
    assert torch.equal(o[~fine & ~r.isnan()], r[~fine & ~r.isnan()]), what
    slack = slack if isinstance(slack, torch.Tensor) else torch.full_like(r, slack)
    bound = half * (r.abs() + slack) + slack + TINY[out.dtype]
    bad = ((o - r).abs() > bound) & fine
    assert not bad.any(), (what, int(bad.sum()), (o - r)[bad][:4], r[bad][:4], bound[bad][:4], bad.nonzero()[:4])


def act_slack(pre, slack, name):
    """An error of `slack` in front of an activation, and the activation's own: none of them is steeper than 1.13."""
    if name in ("identity", "relu"):
        return slack
    return 1.13 * slack + ACT * ULP * (1.0 if name == "tanh" else 1.0 + pre.abs().clamp(max=1e30))


# ---- dense --------------------------------------------------------------------------------------------------------------------------

def whole(shape, g, dtype, low=-4, high=5):
    return torch.randint(low, high, shape, generator=g).to(dtype)


def dense_case(ops, m, n, k, dtype, out_dtype, activation, bias, residual, seed, alpha1=0.5, alpha2=2.0, small=False):
    g = gen(seed)
    # (activations that saturate are looked at where they do not: values of a few units)
    x, w = whole((m, k), g, dtype), whole((n, k), g, dtype) * (torch.rand(n, k, generator=g) < (4.0 / max(k, 4) if small else 1.0)).to(dtype)
    b = whole((n,), g, torch.float32 if bias == "fp32" else dtype) if bias else None
    z = whole((m, n), g, out_dtype) if residual else None
    pre = alpha1 * (x.double() @ w.double().t())
    if z is not None:
        pre = pre + alpha2 * z.double()
    if b is not None:
        pre = pre + b.double()
    y = ops.dense(x.cuda(), w.cuda(), None if b is None else b.cuda(), None if z is None else z.cuda(), alpha1=alpha1, alpha2=alpha2,
                  activation=activation, out_dtype=out_dtype)
    assert y.shape == (m, n) and y.dtype == out_dtype
    ref = act64(pre, activation)
    if activation in ("identity", "relu"):
        assert torch.equal(y.cpu(), ref.to(torch.float32).to(out_dtype)), (m, n, k)
    else:
        close(y, ref, act_slack(pre, 0.0, activation), (m, n, k, activation))


SIZES = [(1, 1, 1), (1, 362, 2888), (1, 1, 722), (2, 3, 5), (3, 17, 31), (7, 64, 64), (15, 16, 33), (16, 48, 256), (17, 15, 8), (16, 1000, 520),
         (31, 33, 1031), (32, 96, 96), (33, 200, 40), (63, 65, 127), (64, 64, 64), (65, 129, 200), (100, 362, 722), (127, 255, 511), (128, 128, 128),
         (129, 130, 1000), (255, 257, 65), (256, 256, 512), (256, 362, 2888), (257, 300, 72), (300, 1, 722), (512, 512, 96), (600, 520, 1032),
         (1000, 999, 333), (2049, 77, 24), (5000, 9, 9), (9, 5000, 9), (1, 9000, 40), (4, 4100, 2048), (1024, 1024, 1024), (769, 1025, 2056),
         # shares of k, copies of unaligned rows, the largest tile with ragged edges, many rows on one side only
         (16, 512, 8192), (8, 100, 20001), (33, 40, 16384), (700, 900, 1001), (2100, 1030, 515), (3500, 3700, 200), (3600, 3500, 263), (70000, 16, 72), (40, 30000, 80)]


@pytest.mark.parametrize("m,n,k", SIZES)
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_dense_sizes(ops, m, n, k, dtype):
    t = TYPES[dtype]
    dense_case(ops, m, n, k, t, t, "identity", "same", True, m * 7 + n * 3 + k)
    dense_case(ops, m, n, k, t, torch.float32, "relu", None, False, m * 5 + n + k)


@pytest.mark.parametrize("activation", ACTIVATIONS)
@pytest.mark.parametrize("dtype,out", [("fp16", "fp16"), ("fp16", "fp32"), ("bf16", "bf16"), ("bf16", "fp32")])
@pytest.mark.parametrize("m,n,k", [(5, 70, 64), (130, 67, 33), (260, 264, 64)])
def test_dense_epilogues(ops, activation, dtype, out, m, n, k):
    for i, (bias, residual) in enumerate([(None, False), ("same", False), ("fp32", True), (None, True)]):
        dense_case(ops, m, n, k, TYPES[dtype], TYPES[out], activation, bias, residual, 100 * m + i, small=True)


@pytest.mark.parametrize("m,n,k", [(1, 40, 64), (16, 40, 136), (70, 72, 136), (300, 264, 200)])
def test_dense_strides_alignments_and_places(ops, m, n, k):
    """Row strides of every kind, operands that start at odd elements, a residual row for all, results into columns and in place."""
    g = gen(m)
    for pad, first in ((0, 0), (8, 0), (8, 8), (1, 0), (3, 1), (5, 7)):
        bx, bw, by = (torch.full((r, c + 16 + pad), 7.0, dtype=torch.float16) for r, c in ((m, k), (n, k), (m, n)))
        bx[:, first:first + k], bw[:, first:first + k], by[:, first:first + n] = whole((m, k), g, torch.float16), whole((n, k), g, torch.float16), whole((m, n), g, torch.float16)
        dx, dw, dy = bx.cuda(), bw.cuda(), by.cuda()
        x, w, y = dx[:, first:first + k], dw[:, first:first + k], dy[:, first:first + n]
        want = (bx[:, first:first + k].double() @ bw[:, first:first + k].double().t())
        for z, expect in ((y, want + by[:, first:first + n].double()), (dy[0, first:first + n].clone(), want + by[0, first:first + n].double())):
            dy.copy_(by)
            assert ops.dense(x, w, residual=z, out=y) is y
            assert torch.equal(y.cpu(), expect.to(torch.float16))
            keep = torch.ones_like(by, dtype=torch.bool)
            keep[:, first:first + n] = False
            assert torch.equal(dy.cpu()[keep], by[keep])                      # what lies between the rows is left as it was
    # x and y as columns of one buffer; the same rows read again and again; windows that overlap
    whole_row = torch.zeros(m, k + n, dtype=torch.float16, device="cuda")
    whole_row[:, :k] = x
    ops.dense(whole_row[:, :k], w, out=whole_row[:, k:])
    assert torch.equal(whole_row[:, k:].cpu(), want.to(torch.float16))
    one = x[:1].expand(m, k)
    assert torch.equal(ops.dense(one, w), ops.dense(x[:1].contiguous(), w).expand(m, n))
    line = whole((m + k,), g, torch.float16)
    windows = line.cuda().as_strided((m, k), (1, 1))
    assert torch.equal(ops.dense(windows, w).cpu(), (line.as_strided((m, k), (1, 1)).double() @ bw[:, first:first + k].double().t()).to(torch.float16))


def test_dense_shapes_of_other_ranks(ops):
    g = gen(1)
    x, w, z = whole((3, 5, 24), g, torch.bfloat16).cuda(), whole((10, 24), g, torch.bfloat16).cuda(), whole((3, 5, 10), g, torch.bfloat16).cuda()
    flat = ops.dense(x.view(15, 24), w, residual=z.view(15, 10))
    assert torch.equal(ops.dense(x, w, residual=z).view(15, 10), flat)
    assert torch.equal(ops.dense(x[1, 2], w, residual=z[1, 2]), flat[7])
    assert ops.dense(x[:0], w).shape == (0, 5, 10) and ops.dense(x, w[:0]).shape == (3, 5, 0)
    empty = ops.dense(x[..., :0], w[:, :0], residual=z, alpha2=0.5)            # nothing to sum
    assert torch.equal(empty, z * 0.5)


@pytest.mark.parametrize("m,n,k", [(1, 33, 64), (16, 64, 40), (40, 40, 40), (256, 256, 256), (300, 260, 264)])
def test_dense_infinities_stay_in_their_rows_and_columns(ops, m, n, k):
    g = gen(4)
    x, w = whole((m, k), g, torch.bfloat16), whole((n, k), g, torch.bfloat16)
    x[m // 2, k - 1], w[n - 1, 0] = math.inf, math.nan
    y = ops.dense(x.cuda(), w.cuda()).cpu()
    want = (x.double() @ w.double().t()).to(torch.bfloat16)
    assert torch.equal(y.isnan(), want.isnan()) and torch.equal(y.nan_to_num(7), want.nan_to_num(7))
    # a padded buffer: what lies behind the rows is not read into a sum
    pad = torch.full((m + 1, k + 8), math.nan, dtype=torch.bfloat16, device="cuda")
    pad[:m, :k] = x[0].cuda()
    assert torch.equal(ops.dense(pad[:m, :k], w[:1].cuda().contiguous()).cpu(), (x[:1].double() @ w[:1].double().t()).to(torch.bfloat16).expand(m, 1))


def test_dense_random_values_beside_a_sum_in_64_bits(ops):
    """Real numbers: the sum's own error is at most k half steps of the sum of the magnitudes, and about their root here."""
    g = gen(9)
    for m, n, k in ((64, 362, 2888), (300, 260, 4096), (3, 70, 8191), (1021, 515, 1027)):
        x, w = torch.randn(m, k, generator=g).bfloat16(), (torch.randn(n, k, generator=g) / math.sqrt(k)).bfloat16()
        ref = x.double() @ w.double().t()
        slack = 16 * math.sqrt(k) * ULP * (x.double().abs() @ w.double().abs().t()) / math.sqrt(k)
        close(ops.dense(x.cuda(), w.cuda(), out_dtype=torch.float32), ref, slack, (m, n, k))
        close(ops.dense(x.cuda(), w.cuda()), ref, slack, (m, n, k))


def test_dense_rounds_large_sums_to_infinity_in_fp16(ops):
    x = torch.full((2, 64), 1000.0, dtype=torch.float16, device="cuda")
    assert torch.equal(ops.dense(x, x).cpu(), torch.full((2, 2), math.inf, dtype=torch.float16))
    assert torch.equal(ops.dense(x, x, out_dtype=torch.float32).cpu(), torch.full((2, 2), 64e6))


# ---- group norm ---------------------------------------------------------------------------------------------------------------------

def group_norm64(x, groups, weight, bias, z, eps):
    """(value in front of the activation, bound of its error) in 64 bits."""
    n, c = x.shape[0], x.shape[-1]
    v = x.double().reshape(n, -1, groups, c // groups)
    mean = v.mean((1, 3), keepdim=True)
    d = v - mean
    scale = 1.0 / torch.sqrt((d * d).mean((1, 3), keepdim=True) + eps)
    shape = x.shape
    w = torch.ones(c, dtype=torch.float64) if weight is None else weight.double()
    pre = (d * scale).reshape(shape) * w
    off = (SERIAL + 16) * ULP * (v.abs().mean((1, 3), keepdim=True) + v.abs()) * scale + (SERIAL + 32) * ULP * (d * scale).abs()
    off = off.reshape(shape) * w.abs()
    if bias is not None:
        pre = pre + bias.double()
    if z is not None:
        pre = pre + z.double()
    return pre, off + 4 * ULP * (pre.abs() + (0 if bias is None else bias.double().abs()) + (0 if z is None else z.double().abs()))


def group_norm_case(ops, shape, groups, dtype, activation="identity", affine=None, residual=False, eps=1e-5, shift=0.5, seed=0):
    g = gen(seed)
    c = shape[-1]
    x = (torch.randn(shape, generator=g) * (1 + torch.rand(c, generator=g)) + shift).to(dtype)
    weight, bias = ((torch.randn(c, generator=g).to(affine), torch.randn(c, generator=g).to(affine)) if affine else (None, None))
    z = torch.randn(shape, generator=g).to(dtype) if residual else None
    pre, off = group_norm64(x, groups, weight, bias, z, eps)
    cuda = [None if t is None else t.cuda() for t in (weight, bias, z)]
    y = ops.group_norm(x.cuda(), groups, *cuda, eps=eps, activation=activation)
    assert y.shape == x.shape and y.dtype == dtype
    close(y, act64(pre, activation), act_slack(pre, off, activation), (shape, groups, dtype, activation))


GN_SHAPES = [((1, 1, 1), 1), ((1, 1, 8), 8), ((2, 1, 6), 3), ((1, 2, 64), 4), ((3, 5, 7), 7), ((2, 361, 64), 8), ((5, 19, 19, 32), 4), ((1, 361, 256), 32),
             ((4, 361, 128), 1), ((2, 100, 90), 9), ((3, 77, 320), 32), ((2, 33, 10), 1), ((1, 4096, 16), 4), ((1, 5000, 24), 2), ((2, 2049, 48), 3),
             ((1, 3, 4096), 1), ((2, 40, 1030), 2), ((1, 17, 2048), 4), ((1, 20000, 8), 1), ((1, 70000, 4), 4), ((1, 9000, 320), 32), ((2, 128, 128, 64), 32),
             ((70, 10, 40), 5), ((1, 1000, 513), 27), ((600, 3, 16), 2), ((1, 40000, 33), 3)]


@pytest.mark.parametrize("shape,groups", GN_SHAPES)
@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
def test_group_norm_sizes(ops, shape, groups, dtype):
    t = TYPES[dtype]
    group_norm_case(ops, shape, groups, t, affine=t, seed=len(shape) + groups)
    group_norm_case(ops, shape, groups, t, "relu", affine=torch.float32, residual=True, shift=-3.0, seed=1)


# where one way of cutting a call up ends and another begins: slabs that may be halved or not, short maps and long ones, one share and many, more
# groups than the waves that join them, lines and vectors that groups end inside
GN_CUTS = [((1, p, c), g) for p in (63, 64, 65, 1024, 1025, 2048, 2049, 4096, 4097) for c, g in ((64, 8), (80, 8), (96, 16))] + [
    ((193, 9, 64), 8), ((191, 9, 64), 8), ((97, 33, 80), 8), ((3, 5241, 180), 9), ((1, 6193, 320), 32), ((2, 4500, 512), 512), ((2, 3000, 36), 9), ((7, 1515, 27), 9),
    ((300, 15, 128), 16), ((2, 5000, 1100), 2), ((260, 513, 24), 3), ((64, 361, 90), 9), ((193, 700, 20), 2)]


@pytest.mark.parametrize("shape,groups", GN_CUTS)
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_group_norm_where_the_cut_changes(ops, shape, groups, dtype):
    t = TYPES[dtype]
    group_norm_case(ops, shape, groups, t, "silu", affine=t, residual=True, seed=shape[1])


@pytest.mark.parametrize("activation", ACTIVATIONS)
@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("shape,groups", [((3, 50, 40), 5), ((2, 361, 64), 8), ((1, 30000, 16), 2)])
def test_group_norm_activations(ops, activation, dtype, shape, groups):
    for i, (affine, residual) in enumerate([(None, False), (torch.float32, False), (TYPES[dtype], True)]):
        group_norm_case(ops, shape, groups, TYPES[dtype], activation, affine, residual, seed=i)


@pytest.mark.parametrize("shape,groups", [((2, 361, 64), 8), ((1, 50000, 16), 4), ((3, 7, 30), 3)])
def test_group_norm_far_from_zero(ops, shape, groups):
    """A mean a thousand standard deviations away: a variance from a difference of sums would be noise."""
    group_norm_case(ops, shape, groups, torch.float32, shift=1500.0, seed=3)
    x = torch.full(shape, 3.0, dtype=torch.float32)                            # no variance at all: the bias alone
    bias = torch.randn(shape[-1], generator=gen(2))
    y = ops.group_norm(x.cuda(), groups, None, bias.cuda())
    assert torch.equal(y.cpu(), bias.expand(shape))


@pytest.mark.parametrize("shape,groups", [((3, 50, 40), 5), ((2, 361, 64), 8), ((2, 20000, 16), 2)])
def test_group_norm_infinities_and_nan_stay_in_their_group(ops, shape, groups):
    n, p, c = shape
    x = torch.randn(shape, generator=gen(5)).half()
    clean = ops.group_norm(x.cuda(), groups).cpu()
    per = c // groups
    x[0, p // 2, 0], x[n - 1, p - 1, c - 1] = math.inf, math.nan
    y = ops.group_norm(x.cuda(), groups).cpu()
    hit = torch.zeros(shape, dtype=torch.bool)
    hit[0, :, :per] = True
    hit[n - 1, :, c - per:] = True
    assert y[hit].isnan().all() and torch.equal(y[~hit], clean[~hit])


@pytest.mark.parametrize("shape,groups", [((3, 50, 40), 5), ((2, 361, 64), 8), ((2, 20000, 16), 2), ((1, 100, 33), 3)])
def test_group_norm_strides_and_places(ops, shape, groups):
    n, p, c = shape
    x = torch.randn(shape, generator=gen(6)).half()
    want = ops.group_norm(x.cuda(), groups, activation="relu").cpu()
    for pad, first in ((8, 0), (8, 8), (3, 0), (5, 3)):
        buffer = torch.full((n, p + 2, c + 16 + pad), 9.0, dtype=torch.float16)
        buffer[:, 1:p + 1, first:first + c] = x
        before = buffer.clone()
        dev = buffer.cuda()
        view = dev[:, 1:p + 1, first:first + c]
        assert torch.equal(ops.group_norm(view, groups, activation="relu").cpu(), want)
        assert ops.group_norm(view, groups, activation="relu", out=view) is view                   # in place
        before[:, 1:p + 1, first:first + c] = want
        assert torch.equal(dev.cpu(), before)                                                      # and nothing beside it
    z = torch.randn(shape, generator=gen(7)).half().cuda()
    both = ops.group_norm(x.cuda(), groups, residual=z)
    assert torch.equal(ops.group_norm(x.cuda(), groups, residual=z, out=z), both)                  # into the residual
    row = torch.randn(1, 1, c, generator=gen(8)).half().cuda()
    assert torch.equal(ops.group_norm(x.cuda(), groups, residual=row.expand(shape)), ops.group_norm(x.cuda(), groups, residual=row.expand(shape).contiguous()))
    assert torch.equal(ops.group_norm(x.cuda()[:1].expand(shape), groups, activation="relu").cpu(), want[:1].expand(shape))
    nchw = x.cuda().transpose(1, 2).contiguous().transpose(1, 2)                                   # channels not innermost
    if c > 1:
        with pytest.raises(Exception, match="contiguous in its channels"):
            ops.group_norm(nchw, groups)


def test_group_norm_of_nothing(ops):
    for shape in ((0, 5, 8), (3, 0, 8), (2, 4, 0)):
        assert ops.group_norm(torch.empty(shape, device="cuda"), 1).shape == shape


# ---- logits -------------------------------------------------------------------------------------------------------------------------

def logits_case(ops, b, v, t, dtype, out=None, mask="row", bias="row", bias_type=torch.float32, history=torch.int32, lengths=True, prompts=True,
                per_row=True, seed=0, spread=None):
    g = gen(seed)
    logits = (torch.randn(b, v, generator=g) * 4).to(dtype)
    kw, words = {}, (v + 31) // 32
    allowed = torch.ones(b, v, dtype=torch.bool)
    if mask:
        rows = b if mask == "row" else 1
        bits = torch.rand(rows, words * 32, generator=g) < 0.6
        if rows > 1:
            bits[rows - 1] = False                                             # this row keeps nothing
        packed = (bits.view(rows, words, 32).long() << torch.arange(32)).sum(-1)
        packed = torch.where(packed >= 1 << 31, packed - (1 << 32), packed).to(torch.int32)
        kw["mask"] = (packed if mask == "row" else packed[0]).cuda()
        allowed = bits[:, :v].expand(b, v)
    shift = torch.zeros(b, v, dtype=torch.float64)
    if bias:
        values = torch.randn((b, v) if bias == "row" else (v,), generator=g).to(bias_type)
        kw["bias"] = values.cuda()
        shift = values.double().expand(b, v)
    seen, count = torch.zeros(b, v, dtype=torch.bool), torch.zeros(b, v, dtype=torch.float64)
    r, pr, fr = (torch.full((b,), x, dtype=torch.float64) for x in (1.3, 0.25, 0.125))
    if history is not None:
        tokens = torch.randint(-3, min(v, spread or v) + 3, (b, t), generator=g).to(history)
        n = torch.randint(-2, t + 4, (b,), generator=g) if lengths else torch.full((b,), t)
        q = torch.randint(-2, t + 4, (b,), generator=g) if prompts else torch.zeros(b, dtype=torch.long)
        kw["history"] = tokens.cuda()
        if lengths:
            kw["lengths"] = n.to(torch.int32).cuda()
        if prompts:
            kw["prompt_lengths"] = q.to(torch.int32).cuda()
        for i in range(b):
            for j in range(max(0, min(int(n[i]), t))):
                token = int(tokens[i, j])
                if 0 <= token < v:
                    seen[i, token] = True
                    count[i, token] += j >= int(q[i])
        if per_row:
            r, pr, fr = (torch.rand(b, generator=g) + s for s in (0.5, -0.5, -0.5))
            kw.update(repetition=r.cuda(), presence=pr.cuda(), frequency=fr.cuda())
            r, pr, fr = r.double(), pr.double(), fr.double()
        else:
            kw.update(repetition=1.3, presence=0.25, frequency=0.125)
            r = torch.full((b,), float(np.float32(1.3)), dtype=torch.float64)
    l = logits.double()
    ref = torch.where(seen, torch.where(l > 0, l / r[:, None], l * r[:, None]), l)
    ref = ref - fr[:, None] * count - pr[:, None] * (count > 0) + shift
    slack = 6 * ULP * (l.abs() * torch.maximum(r, 1 / r)[:, None] + fr[:, None].abs() * count + pr[:, None].abs() + shift.abs())
    ref = ref.masked_fill(~allowed, -math.inf)
    to = None if out is None else torch.empty(b, v, dtype=out, device="cuda")
    got = ops.adjust_logits(logits.cuda(), **kw, out=to)
    assert got.dtype == (out or dtype) and got.shape == (b, v) and (to is None or got is to)
    close(got, ref, slack, (b, v, t))


@pytest.mark.parametrize("b,v,t", [(1, 1, 1), (1, 362, 3), (2, 31, 5), (3, 32, 0), (2, 33, 40), (5, 362, 100), (1, 1000, 2000), (3, 4096, 17), (2, 4097, 64),
                                   (1, 8191, 1), (4, 20011, 300), (2, 40000, 1111), (1, 70001, 50), (33, 100, 20), (300, 64, 9)])
@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
def test_logits_sizes(ops, b, v, t, dtype):
    logits_case(ops, b, v, t, TYPES[dtype], seed=v + t)
    logits_case(ops, b, v, t, TYPES[dtype], out=torch.float32, mask="shared", bias="vocabulary", bias_type=TYPES[dtype], history=torch.int64, lengths=False,
                per_row=False, seed=v, spread=5)


@pytest.mark.parametrize("mask", [None, "row", "shared"])
@pytest.mark.parametrize("bias", [None, "row", "vocabulary"])
@pytest.mark.parametrize("history", [None, torch.int32, torch.int64])
def test_logits_parts(ops, mask, bias, history):
    logits_case(ops, 4, 515, 37, torch.bfloat16, mask=mask, bias=bias, history=history, seed=1)
    logits_case(ops, 3, 4200, 37, torch.float16, mask=mask, bias=bias, history=history, prompts=False, per_row=False, seed=2)


def test_logits_one_token_again_and_again(ops):
    """The same index thousands of times: counts are whole numbers and exact."""
    v, t = 5000, 70000
    history = torch.full((2, t), 4321, dtype=torch.int32, device="cuda")
    logits = torch.zeros(2, v, device="cuda")
    out = ops.adjust_logits(logits, history=history, lengths=torch.tensor([t, 65537], dtype=torch.int32, device="cuda"), frequency=1.0).cpu()
    want = torch.zeros(2, v)
    want[0, 4321], want[1, 4321] = -t, -65537
    assert torch.equal(out, want)
    padded = torch.full((1, 50), -1, dtype=torch.int64, device="cuda")
    assert torch.equal(ops.adjust_logits(logits[:1], history=padded, frequency=1.0, presence=1.0, repetition=2.0), logits[:1])
    far = torch.tensor([[2 ** 31 + 5, -2 ** 33, 2 ** 32 + 7, v]], dtype=torch.int64, device="cuda")
    assert torch.equal(ops.adjust_logits(logits[:1], history=far, frequency=1.0, presence=1.0, repetition=2.0), logits[:1])


def test_logits_special_values(ops):
    lowest = torch.finfo(torch.bfloat16).min
    row = torch.tensor([[math.inf, -math.inf, math.nan, lowest, 0.0, 1.0, math.nan, math.inf]], dtype=torch.bfloat16, device="cuda")
    history = torch.arange(6, dtype=torch.int32, device="cuda")[None]
    mask = torch.tensor([[0b00111111]], dtype=torch.int32, device="cuda")
    got = ops.adjust_logits(row, mask=mask, history=history, repetition=2.0).float().cpu()[0]
    assert got[0] == math.inf and got[1] == -math.inf and got[2].isnan() and got[3] == -math.inf and got[4] == 0 and got[5] == 0.5
    assert got[6] == -math.inf and got[7] == -math.inf                        # masked: whatever it was
    nothing = ops.adjust_logits(row, mask=torch.zeros(1, 1, dtype=torch.int32, device="cuda"), bias=torch.full((8,), math.inf, device="cuda"))
    assert (nothing == -math.inf).all()


@pytest.mark.parametrize("v", [362, 4096, 9001])
def test_logits_strides_and_places(ops, v):
    b, words = 5, (v + 31) // 32
    g = gen(3)
    logits = torch.randn(b, v, generator=g).half().cuda()
    mask = torch.randint(-(1 << 31), 1 << 31, (b, words), generator=g).to(torch.int32).cuda()
    bias = torch.randn(b, v, generator=g).cuda()
    history = torch.randint(0, v, (b, 30), generator=g).to(torch.int32).cuda()
    want = ops.adjust_logits(logits, mask=mask, bias=bias, history=history, repetition=1.5, frequency=0.5)
    for pad, first in ((8, 0), (1, 1), (3, 2)):
        big = torch.full((b, v + pad + first), 5.0, dtype=torch.float16, device="cuda")
        view = big[:, first:first + v]
        view.copy_(logits)
        wide = [torch.zeros(b, t.shape[1] + 3, dtype=t.dtype, device="cuda") for t in (mask, bias, history)]
        parts = [w[:, 1:1 + t.shape[1]] for w, t in zip(wide, (mask, bias, history))]
        for p, t in zip(parts, (mask, bias, history)):
            p.copy_(t)
        kw = dict(mask=parts[0], bias=parts[1], history=parts[2], repetition=1.5, frequency=0.5)
        assert torch.equal(ops.adjust_logits(view, **kw), want)
        assert ops.adjust_logits(view, **kw, out=view) is view
        assert torch.equal(view, want)
        big[:, first:first + v] = 5.0
        assert (big == 5.0).all()
    assert torch.equal(ops.adjust_logits(logits[:1].expand(b, v), mask=mask), ops.adjust_logits(logits[:1].expand(b, v).contiguous(), mask=mask))


def test_logits_rows_beyond_two_to_the_31_elements(ops):
    stride = (1 << 30) + 3
    base = torch.empty(2 * stride + 400, dtype=torch.float16, device="cuda")
    rows = base.as_strided((3, 362), (stride, 1))
    values = torch.randn(3, 362, generator=gen(1)).half()
    rows.copy_(values)
    ops.adjust_logits(rows, bias=torch.ones(362, device="cuda"), out=rows)
    assert torch.equal(rows.cpu(), (values.float() + 1).half())


def test_dense_and_group_norm_beyond_two_to_the_31_elements(ops):
    stride = (1 << 30) + 8
    base = torch.empty(2 * stride + 4096, dtype=torch.float16, device="cuda")
    g = gen(2)
    x, w = whole((3, 64), g, torch.float16), whole((72, 64), g, torch.float16)
    rows = base.as_strided((3, 64), (stride, 1))
    rows.copy_(x)
    out = base[2048:].as_strided((3, 72), (stride, 1))
    ops.dense(rows, w.cuda(), out=out)
    assert torch.equal(out.cpu(), (x.double() @ w.double().t()).half())
    maps, ref = base.as_strided((3, 16, 32), (stride, 32, 1)), torch.randn(3, 16, 32, generator=g).half()
    maps.copy_(ref)
    want = ops.group_norm(ref.cuda(), 4)
    assert torch.equal(ops.group_norm(maps, 4, out=maps), want)


def test_more_work_than_one_grid_holds(ops):
    """Loops behind a capped grid: rows, samples, slabs and sequences beyond what one launch numbers."""
    g = gen(11)
    x, w = whole((16_800_000, 8), g, torch.float16).cuda(), whole((3, 8), g, torch.float16).cuda()
    assert torch.equal(ops.dense(x, w), (x[:, None, :].float() * w.float()).sum(-1).half())
    group_norm_case(ops, (40000, 3, 16), 2, torch.float16, "relu", torch.float32, True)
    group_norm_case(ops, (1, 2, 64 * 66000), 66000, torch.float16, "identity", torch.float16)
    logits = torch.randn(70000, 40, generator=g).cuda()
    assert torch.equal(ops.adjust_logits(logits, bias=torch.ones(40, device="cuda")), logits + 1)
    history = torch.arange(70000, dtype=torch.int32, device="cuda")[:, None] % 40
    want = logits.scatter_add(1, history.long(), torch.full((70000, 1), -0.5, device="cuda"))
    assert torch.equal(ops.adjust_logits(logits, history=history, frequency=0.5), want)


def test_an_error_of_the_runtime_is_told_once(ops, api):
    x = torch.ones(4, 8, dtype=torch.float16, device="cuda")
    y = torch.empty(4, 4, dtype=torch.float16, device="cuda")
    block = ops._DENSE.pack(x.data_ptr(), x.data_ptr(), 0, 0, y.data_ptr(), 0, 0, 4, 4, 8, 8, 8, 0, 4, 1.0, 1.0, 0, 0, 0, 0)
    assert ops.lib.dgnn_dense(1 << 20, None, block) == api.HIP_ERROR and ops.lib.dgnn_ops_last_hip_error() != 0
    assert torch.equal(torch.relu(x), x)                                       # torch asks the runtime after its launches
    assert ops.lib.dgnn_dense(0, None, block) == api.OK
    torch.cuda.synchronize()
    assert (y == 8).all()


# ---- refusals -----------------------------------------------------------------------------------------------------------------------

def test_refusals_of_the_python_mirror(ops, api):
    h = lambda *s: torch.zeros(*s, dtype=torch.float16, device="cuda")      # noqa: E731
    i = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")        # noqa: E731
    f = lambda *s: torch.zeros(*s, device="cuda")                           # noqa: E731
    x, w, maps, l = h(4, 16), h(8, 16), h(2, 9, 16), h(3, 100)
    grad = torch.zeros(4, 16, dtype=torch.float16, device="cuda", requires_grad=True)
    bad = [
        (api.BAD_ARGUMENT, lambda: ops.dense(x, h(8, 15))), (api.BAD_ARGUMENT, lambda: ops.dense(x, h(16))), (api.UNSUPPORTED, lambda: ops.dense(x, w.bfloat16())),
        (api.UNSUPPORTED, lambda: ops.dense(f(4, 16), f(8, 16))), (api.BAD_ARGUMENT, lambda: ops.dense(x, w.cpu())), (api.BAD_ARGUMENT, lambda: ops.dense(x, w, h(7))),
        (api.UNSUPPORTED, lambda: ops.dense(x, w, h(8).bfloat16())), (api.BAD_ARGUMENT, lambda: ops.dense(x, w, residual=h(4, 7))),
        (api.UNSUPPORTED, lambda: ops.dense(x, w, residual=f(4, 8))), (api.BAD_ARGUMENT, lambda: ops.dense(x, w, activation="swish")),
        (api.BAD_ARGUMENT, lambda: ops.dense(x, w, out=h(4, 9))), (api.UNSUPPORTED, lambda: ops.dense(x, w, out_dtype=torch.bfloat16)),
        (api.UNSUPPORTED, lambda: ops.dense(h(16, 4).t(), w)), (api.UNSUPPORTED, lambda: ops.dense(x, h(16, 8).t())), (api.UNSUPPORTED, lambda: ops.dense(x, w, h(16)[::2])),
        (api.UNSUPPORTED, lambda: ops.dense(grad, w)), (api.UNSUPPORTED, lambda: ops.dense(x, w, out=h(8, 4).t())), (api.BAD_ARGUMENT, lambda: ops.dense(x, w, out=h(1, 8).expand(4, 8))),
        (api.BAD_ARGUMENT, lambda: ops.dense(x, h(16, 16), out=x)), (api.UNSUPPORTED, lambda: ops.dense(h(4, 3, 16).transpose(0, 1), w)),
        (api.BAD_ARGUMENT, lambda: ops.group_norm(maps, 5)), (api.BAD_ARGUMENT, lambda: ops.group_norm(maps, 0)), (api.BAD_ARGUMENT, lambda: ops.group_norm(h(16), 4)),
        (api.BAD_ARGUMENT, lambda: ops.group_norm(maps, 4, h(15))), (api.UNSUPPORTED, lambda: ops.group_norm(maps, 4, f(16), h(16))), (api.UNSUPPORTED, lambda: ops.group_norm(maps, 4, residual=f(2, 9, 16))),
        (api.BAD_ARGUMENT, lambda: ops.group_norm(maps, 4, residual=h(2, 8, 16))), (api.BAD_ARGUMENT, lambda: ops.group_norm(maps, 4, eps=-1.0)), (api.UNSUPPORTED, lambda: ops.group_norm(maps.double(), 4)),
        (api.BAD_ARGUMENT, lambda: ops.group_norm(maps, 4, out=h(2, 9, 15))), (api.BAD_ARGUMENT, lambda: ops.group_norm(maps, 4, activation=None)), (api.UNSUPPORTED, lambda: ops.group_norm(grad, 4)),
        (api.BAD_ARGUMENT, lambda: ops.group_norm(h(3, 9, 16)[:2], 4, out=h(1, 9, 16).expand(2, 9, 16))),
        (api.BAD_ARGUMENT, lambda: ops.adjust_logits(h(100))), (api.BAD_ARGUMENT, lambda: ops.adjust_logits(l, mask=i(3, 3))), (api.UNSUPPORTED, lambda: ops.adjust_logits(l, mask=f(3, 4))),
        (api.BAD_ARGUMENT, lambda: ops.adjust_logits(l, mask=i(2, 4))), (api.BAD_ARGUMENT, lambda: ops.adjust_logits(l, bias=f(99))), (api.UNSUPPORTED, lambda: ops.adjust_logits(l, bias=l.bfloat16())),
        (api.BAD_ARGUMENT, lambda: ops.adjust_logits(l, history=i(2, 4))), (api.BAD_ARGUMENT, lambda: ops.adjust_logits(l, history=i(3))), (api.UNSUPPORTED, lambda: ops.adjust_logits(l, history=f(3, 4))),
        (api.BAD_ARGUMENT, lambda: ops.adjust_logits(l, lengths=i(3))), (api.BAD_ARGUMENT, lambda: ops.adjust_logits(l, history=i(3, 4), lengths=i(2))),
        (api.UNSUPPORTED, lambda: ops.adjust_logits(l, history=i(3, 4), lengths=i(3).long())), (api.BAD_ARGUMENT, lambda: ops.adjust_logits(l, history=i(3, 4), repetition=0.0)),
        (api.BAD_ARGUMENT, lambda: ops.adjust_logits(l, history=i(3, 4), repetition=f(2))), (api.BAD_ARGUMENT, lambda: ops.adjust_logits(l, history=i(3, 4), presence=math.nan)),
        (api.UNSUPPORTED, lambda: ops.adjust_logits(l, out=l.bfloat16())), (api.BAD_ARGUMENT, lambda: ops.adjust_logits(l, out=h(1, 100).expand(3, 100))),
    ]
    for n, (status, run) in enumerate(bad):
        with pytest.raises(api.Error) as e:
            run()
        assert e.value.status == status, (n, str(e.value))
    with torch.no_grad():
        assert ops.dense(grad, w).shape == (4, 8)                              # evaluating: nothing to record


# ---- streams, graphs, threads -------------------------------------------------------------------------------------------------------

class Net:
    """A small network of another shape than the reference's: dense layers on points, group norm, a policy and a value head."""

    def __init__(self, seed, dtype, device="cuda"):
        g = gen(seed)
        def r(*s, k=1.0): return (torch.randn(*s, generator=g) * k).to(dtype).to(device)     # noqa: E306,E704
        self.w1, self.w2, self.wp, self.wv = r(64, 32, k=0.2), r(64, 64, k=0.12), r(8, 64, k=0.12), r(2, 64, k=0.12)
        self.g1, self.b1, self.g2, self.b2 = (r(64, k=0.1) + 1, r(64, k=0.1), r(64, k=0.1) + 1, r(64, k=0.1))
        self.policy, self.policy_b, self.value = r(362, 2888, k=0.05), r(362, k=0.1), r(1, 722, k=0.05)

    def run(self, ops, x, mask):
        n = x.shape[0]
        h = ops.group_norm(ops.dense(x, self.w1), 8, self.g1, self.b1, activation="relu")
        h = ops.group_norm(ops.dense(h, self.w2), 8, self.g2, self.b2, h, activation="relu")
        p = ops.dense(h, self.wp, activation="relu").view(n, 2888)
        v = ops.dense(h, self.wv, activation="relu").view(n, 722)
        logits = ops.adjust_logits(ops.dense(p, self.policy, self.policy_b, out_dtype=torch.float32), mask=mask)
        return ops.dense(v, self.value, activation="tanh", out_dtype=torch.float32)[:, 0], logits

    def run64(self, x, allowed):
        """The same in 64 bits, rounded where the operators round."""
        d = lambda t: t.double().cpu()                                                       # noqa: E731
        rnd = lambda t: t.to(self.w1.dtype).double()                                         # noqa: E731
        n, x = x.shape[0], d(x)
        h = rnd(x @ d(self.w1).t())
        h = rnd(torch.relu(group_norm64(h, 8, d(self.g1), d(self.b1), None, 1e-5)[0]))
        k = rnd(h @ d(self.w2).t())
        h = rnd(torch.relu(group_norm64(k, 8, d(self.g2), d(self.b2), h, 1e-5)[0]))
        p, v = rnd(torch.relu(h @ d(self.wp).t())).reshape(n, 2888), rnd(torch.relu(h @ d(self.wv).t())).reshape(n, 722)
        logits = (p @ d(self.policy).t() + d(self.policy_b)).masked_fill(~allowed, -math.inf)
        return torch.tanh(v @ d(self.value).t())[:, 0], logits


def planes(n, seed):
    return (torch.rand(n, 361, 32, generator=gen(seed)) < 0.2).half().cuda()


def legal(x):
    """Bits of the points whose plane 2 is empty, and the pass."""
    allowed = torch.cat([x[:, :, 2] == 0, torch.ones(x.shape[0], 1, dtype=torch.bool, device=x.device)], 1)
    bits = torch.zeros(x.shape[0], 12 * 32, dtype=torch.long, device=x.device)
    bits[:, :362] = allowed.long()
    words = (bits.view(-1, 12, 32) << torch.arange(32, device=x.device)).sum(-1)
    return torch.where(words >= 1 << 31, words - (1 << 32), words).to(torch.int32), allowed


@pytest.mark.parametrize("n", [1, 5, 64])
def test_a_network_of_them(ops, n):
    net, x = Net(1, torch.float16), planes(n, 7)
    mask, allowed = legal(x)
    value, logits = net.run(ops, x, mask)
    want_value, want_logits = net.run64(x, allowed.cpu())
    assert torch.equal(logits.cpu().isfinite(), allowed.cpu())
    # where fp32 and 64 bits round an intermediate differently it moves by one step, 2^-10 of its size: some of 2888 inputs, weights of 0.05
    fine = allowed.cpu()
    assert (logits.double().cpu() - want_logits)[fine].abs().max() < 2e-2 and (value.double().cpu() - want_value).abs().max() < 2e-2
    assert (logits.double().cpu() - want_logits)[fine].pow(2).mean().sqrt() < 2e-3


def test_a_network_of_them_behind_the_search(ops, api_full):
    """... as the predictor of a search: every leaf goes through the operators, twice the same search gives the same visits."""
    net = Net(2, torch.float16)
    seen = []

    def predict(features, n):
        x = torch.from_numpy(np.array(features, copy=True).view(np.float16).reshape(n, 361, 32)).cuda()
        mask, _ = legal(x)
        value, logits = net.run(ops, x, mask)
        seen.append(n)
        return value.half().cpu().numpy(), torch.softmax(logits, -1).half().cpu().numpy()

    def search():
        board = api_full.Board(7.5)
        for i, (px, py) in enumerate([(3, 3), (15, 15), (15, 3), (3, 15)]):
            board.place(i % 2, px, py)
        predictor = api_full.python_predictor(predict)
        _, prior, _ = api_full.full_forward(board, 0, predictor)
        root = api_full.Node(0, 0.0, prior)
        evals, _ = api_full.search_run(root, board, 48, seed=5, pool=predictor)
        return evals, [root.with_(i).count() for i in range(362)]

    first = search()
    assert 0 < sum(first[1]) <= 48 and sum(seen) >= first[0] > 0             # (a search may end before its limit)
    assert search() == first


def test_another_stream_than_the_current_one(ops):
    net, x = Net(3, torch.bfloat16), planes(33, 1).bfloat16()
    mask, _ = legal(x)
    want = net.run(ops, x, mask)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            for _ in range(4):
                got.append(net.run(ops, x, mask))
    torch.cuda.synchronize()
    for value, logits in got:
        assert torch.equal(value, want[0]) and torch.equal(logits, want[1])


def test_captured_into_graphs_that_replay(ops):
    """Two graphs of one network, replayed in turn beside eager calls: each replay is the eager result on its inputs."""
    net = Net(4, torch.float16)
    big = torch.randn(1, 30000, 64, generator=gen(2)).half().cuda()
    inputs = [planes(17, 2), planes(40, 3)]
    masks = [legal(x)[0] for x in inputs]

    def work(i):
        value, logits = net.run(ops, inputs[i], masks[i])
        return value, logits, ops.group_norm(big, 4 + 4 * i, activation="silu")

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for i in range(2):
            work(i)
    torch.cuda.current_stream().wait_stream(stream)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for i in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(work(i))
        graphs.append(graph)
    for step in range(4):
        for i in range(2):
            inputs[i].copy_(planes(inputs[i].shape[0], 10 * step + i))
            masks[i].copy_(legal(inputs[i])[0])
        graphs[0].replay()
        graphs[1].replay()
        eager = [work(i) for i in range(2)]
        torch.cuda.synchronize()
        for i in range(2):
            for a, b in zip(outs[i], eager[i]):
                assert torch.equal(a, b), (step, i)


def test_two_threads_at_once(ops):
    import threading
    net, xs = Net(5, torch.float16), [planes(9, 1), planes(70, 2)]
    masks = [legal(x)[0] for x in xs]
    want = [net.run(ops, x, m) for x, m in zip(xs, masks)]
    torch.cuda.synchronize()
    failed = []

    def go(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got = net.run(ops, xs[i], masks[i])
                torch.cuda.current_stream().synchronize()
                if not all(torch.equal(a, b) for a, b in zip(got, want[i])):
                    failed.append(i)

    threads = [threading.Thread(target=go, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed


def test_the_same_call_gives_the_same_bits(ops):
    g = gen(3)
    x, w = torch.randn(300, 1000, generator=g).half().cuda(), torch.randn(500, 1000, generator=g).half().cuda()
    maps, l = torch.randn(2, 30000, 64, generator=g).half().cuda(), torch.randn(4, 30000, generator=g).cuda()
    history = torch.randint(0, 300, (4, 3000), generator=g).to(torch.int32).cuda()
    runs = [lambda: ops.dense(x, w, activation="gelu"), lambda: ops.group_norm(maps, 8), lambda: ops.adjust_logits(l, history=history, frequency=0.3, repetition=1.1)]
    for run in runs:
        first = run()
        assert all(torch.equal(run(), first) for _ in range(5))
