"""GPU tests of products with packed INT layers and the adapters beside them (packed_linear.py over
csrc/packed_linear.hip) against the formula in 64 bits on the CPU.

Tolerance: the result's own rounding (half a unit in the last place: 2^-8 of it for bf16, 2^-11 fp16, 2^-24 fp32), and
2^-20 of the sum of the absolute values of all terms (fp32 sums of n <= 9000 terms in runs of 32: up to 280 additions, each
off by at most 2^-24 of a partial sum, which is below that sum and random in sign: 17 x 2^-24 < 2^-19.9; fp32 activations
in two pieces of 22 bits add 2^-23).  Adapters: 2^-16 of the sum of |x A^T| |B| for bf16 and fp16 (x A^T in two pieces of 8 bits
leaves out at most 2^-16), 2^-20 for fp32."""

import math

import pytest
import torch

import _hip
import model_driver as MD
import packing
from packed_linear import Adapters, packed_linear

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
OWN = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


class Layer:
    def __init__(self, m, n, qmin, qmax, group, zero, seed, bad_scales=False):
        g = torch.Generator().manual_seed(seed)
        groups = -(-n // group) if group else 1
        self.m, self.n, self.qmin, self.qmax, self.group, self.g = m, n, qmin, qmax, group, g
        self.scale = 0.01 + 0.02 * torch.rand(m, groups, generator=g)
        if bad_scales:  # zero, negative, tiny and huge ones: no step divides by a scale
            self.scale[0, 0], self.scale[1 % m, -1], self.scale[2 % m, 0], self.scale[3 % m, -1] = 0., -0.3, 1e-30, 1e25
        self.zero = torch.randint(-3, 4, (m, groups), generator=g) + 0.5 if zero else None
        self.codes = torch.randint(qmin, qmax + 1, (m, n), generator=g)
        self.column = torch.arange(n) // (group or n)
        self.bits = max(1, math.ceil(math.log2(qmax - qmin + 1)))

    def weights(self):
        z = 0. if self.zero is None else self.zero.double()[:, self.column]
        return (self.codes.double() - z) * self.scale.double()[:, self.column]

    def size(self):
        """Sum over a term's parts: |code - middle| + |zero point's distance from it|, times the scale."""
        middle = self.qmin + 2 ** (self.bits - 1)
        z = torch.full((self.m, 1), 0., dtype=torch.float64).expand(self.m, self.n) if self.zero is None \
            else self.zero.double()[:, self.column]
        return ((self.codes - middle).abs().double() + (z - middle).abs()) * self.scale.double().abs()[:, self.column]

    def words(self):
        u = (self.codes - self.qmin).tolist()
        row_words = -(-self.n * self.bits // 32)
        out = torch.zeros(self.m, row_words, dtype=torch.int64)
        for i in range(self.m):
            field = 0
            for k in range(self.n - 1, -1, -1):
                field = field << self.bits | u[i][k]
            for w in range(row_words):
                v = field >> 32 * w & 0xffffffff
                out[i, w] = v - (1 << 32) if v >> 31 else v
        return out.to(torch.int32).to(DEV)

    def call(self, x, **more):
        return packed_linear(x.to(DEV), self.words(), self.scale.to(DEV),
                             None if self.zero is None else self.zero.to(DEV), qmin=self.qmin, qmax=self.qmax,
                             group=self.group or None, **more)


def make_adapters(count, rank, layer, dtype, tokens, g):
    a = (torch.randn(count, rank, layer.n, generator=g) * layer.n ** -0.5).to(dtype)
    b = torch.randn(count, layer.m, rank, generator=g).to(dtype)
    scaling = 0.5 + torch.rand(count, generator=g)
    index = torch.randint(-1, count + 1, (tokens,), generator=g).to(torch.int32)  # `count` itself is none either
    return Adapters(a, b, scaling), index


def reference(x, layer, bias=None, adapters=None, index=None):
    """(y, allowed for its sums) in 64 bits."""
    xd = x.double()
    y = xd @ layer.weights().t()
    slack = 2.0 ** -20 * (xd.abs() @ layer.size().t())
    if bias is not None:
        y = y + bias.double()
        slack = slack + 2.0 ** -23 * bias.double().abs()
    if adapters is not None:
        a, b, scaling = (t.double() for t in adapters)
        for t in range(x.size(0)):
            e = int(index[t])
            if 0 <= e < a.size(0):
                v = a[e] @ xd[t]
                y[t] += scaling[e] * (b[e] @ v)
                each = 2.0 ** -20 if x.dtype is torch.float32 else 2.0 ** -16
                slack[t] += scaling[e] * (each * (b[e].abs() @ v.abs()) + 2.0 ** -20 * (b[e].abs() @ (a[e].abs() @ xd[t].abs())))
    return y, slack


def check(got, want, slack):
    off = (got.double().cpu() - want).abs()
    info = torch.finfo(got.dtype)  # below the type's normal numbers: half the step of the subnormal ones
    allowed = want.abs() * OWN[got.dtype] * 1.01 + info.smallest_normal * info.eps / 2 + slack
    assert bool((off <= allowed).all()), f"off by {float((off / allowed).max()):.3g} of what is allowed"


SHAPES = [  # tokens, m, n, (qmin, qmax), group, zero
    (1, 16, 128, (-8, 7), 0, False),
    (1, 1, 1, (0, 15), 0, True),
    (3, 37, 515, (-8, 7), 0, True),
    (16, 130, 1000, (0, 15), 128, True),
    (16, 40, 999, (-8, 7), 32, False),
    (5, 33, 700, (-7, 7), 96, False),
    (2, 50, 8999, (-4, 3), 0, False),
    (17, 129, 400, (-4, 3), 64, True),
    (33, 40, 515, (-2, 1), 0, True),
    (7, 48, 300, (0, 3), 32, True),
    (64, 100, 260, (-128, 127), 32, True),
    (11, 20, 513, (0, 255), 256, True),
    (65, 257, 384, (-8, 7), 128, True),
    (130, 150, 640, (-8, 7), 256, True),
    (200, 129, 333, (-8, 7), 0, False),
    (129, 64, 1030, (0, 15), 32, True),
    (300, 8, 2048, (-8, 7), 1024, True),
    (140, 260, 129, (-4, 3), 32, False),
    (128, 128, 128, (-128, 127), 0, False),
]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("case", range(len(SHAPES)))
def test_product(case, dtype):
    tokens, m, n, (qmin, qmax), group, zero = SHAPES[case]
    print(f"packed linear case {case} {dtype}", flush=True)
    layer = Layer(m, n, qmin, qmax, group, zero, seed=case, bad_scales=case % 3 == 2)
    x = torch.randn(tokens, n, generator=layer.g)
    x[:, ::17] *= 30.
    x = x.to(TYPES[dtype])
    bias = torch.randn(m, generator=layer.g).to(x.dtype)
    layer.scale.clamp_(max=1. if x.dtype is torch.float16 else 1e25)  # a result in fp16's range
    want, slack = reference(x, layer, bias if case % 2 else None)
    check(layer.call(x, bias=bias.to(DEV) if case % 2 else None), want, slack)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("tokens,count,rank", [(1, 1, 1), (1, 5, 16), (16, 16, 16), (13, 3, 33), (40, 7, 9), (90, 2, 64),
                                               (150, 4, 100), (300, 30, 8)])
def test_adapters(tokens, count, rank, dtype):
    print(f"adapters {tokens} {count} {rank} {dtype}", flush=True)
    layer = Layer(70, 1100, -8, 7, 0, False, seed=tokens + rank)
    x = torch.randn(tokens, layer.n, generator=layer.g).to(TYPES[dtype])
    adapters, index = make_adapters(count, rank, layer, x.dtype, tokens, layer.g)
    want, slack = reference(x, layer, None, adapters, index)
    got = layer.call(x, adapters=Adapters(*(t.to(DEV) for t in adapters)), index=index.to(DEV))
    check(got, want, slack)
    none = layer.call(x, adapters=Adapters(*(t.to(DEV) for t in adapters)), index=torch.full_like(index, -1).to(DEV))
    assert torch.equal(none, layer.call(x)), "tokens without an adapter"


def test_split_columns_and_many_rows():
    """Few rows and long columns (workgroups share a row's columns), with adapters, and many rows of few columns."""
    for tokens, m, n in ((1, 24, 8800), (16, 24, 8800), (50, 24, 8800), (2, 5000, 64)):
        layer = Layer(m, n, -8, 7, 128 if m < 100 else 0, m < 100, seed=m + tokens)
        x = torch.randn(tokens, n, generator=layer.g).bfloat16()
        adapters, index = make_adapters(3, 12, layer, x.dtype, tokens, layer.g)
        bias = torch.randn(m, generator=layer.g).bfloat16()
        want, slack = reference(x, layer, bias, adapters, index)
        got = layer.call(x, bias=bias.to(DEV), adapters=Adapters(*(t.to(DEV) for t in adapters)), index=index.to(DEV))
        check(got, want, slack)


def test_activations_extremes():
    """Rows of zeros, tiny and huge rows, elements of very different size; infinities and NaN stay in their token."""
    layer = Layer(40, 300, -8, 7, 0, False, seed=1)
    for dtype in TYPES.values():
        big = {torch.float32: 1e30, torch.bfloat16: 1e30, torch.float16: 60.}[dtype]
        small = {torch.float32: 1e-30, torch.bfloat16: 1e-30, torch.float16: 1e-6}[dtype]
        x = torch.randn(20, 300, generator=layer.g)
        x[0] = 0.
        x[1] *= big
        x[2] *= small
        x[3, ::2] *= 1e-4
        clean = x.to(dtype)
        want, slack = reference(clean, layer)
        got = layer.call(clean)
        check(got, want, slack)
        dirty = clean.clone()
        dirty[5, 7], dirty[6, 299], dirty[7, 0] = math.inf, -math.inf, math.nan
        bad = layer.call(dirty)
        keep = torch.ones(20, dtype=torch.bool)
        keep[5:8] = False
        assert torch.equal(bad.cpu()[keep], got.cpu()[keep])
        # an infinite activation times a weight that is not 0 is infinite, of the product's sign
        w = layer.weights()
        for row, column, sign in ((5, 7, 1.), (6, 299, -1.)):
            s = w[:, column].sign() * sign
            there = s != 0
            assert torch.equal(bad[row].double().cpu()[there], s[there] * math.inf)
        assert bool(bad[7].isnan().all())


def test_layouts():
    """Leading axes, strided activations, words with longer rows, scales as numbers, vectors and strided matrices, another
    stream."""
    layer = Layer(48, 200, -8, 7, 0, False, seed=2)
    x = torch.randn(2, 3, 5, 200, generator=layer.g).half()
    want = layer.call(x.reshape(-1, 200)).view(2, 3, 5, 48)
    assert torch.equal(layer.call(x), want)
    wide = torch.zeros(30, 333, dtype=torch.float16)
    wide[:, 7:207] = x.reshape(-1, 200)
    assert torch.equal(layer.call(wide.to(DEV)[:, 7:207]), want.view(-1, 48))
    assert torch.equal(layer.call(x.reshape(-1, 200).t().contiguous().to(DEV).t()), want.view(-1, 48))
    words = torch.full((48, 40), -1, dtype=torch.int32, device=DEV)
    words[:, 3:28] = layer.words()
    kw = dict(qmin=-8, qmax=7)
    xd = x.reshape(-1, 200).to(DEV)
    assert torch.equal(packed_linear(xd, words[:, 3:28], layer.scale.to(DEV), **kw), want.view(-1, 48))
    assert torch.equal(packed_linear(xd, words[:, 3:], layer.scale.to(DEV)[:, 0], **kw), want.view(-1, 48))
    one = packed_linear(xd, words[:, 3:], torch.tensor(0.5, device=DEV), torch.tensor(1., device=DEV), **kw)
    full = packed_linear(xd, words[:, 3:], torch.full((48, 1), 0.5, device=DEV), torch.ones(48, 1, device=DEV), **kw)
    assert torch.equal(one, full)
    grouped = Layer(48, 200, -8, 7, 64, True, seed=3)
    s = grouped.scale.t().contiguous().to(DEV).t()
    z = torch.stack([grouped.zero, grouped.zero + 9], dim=2).to(DEV)[:, :, 0]
    assert torch.equal(packed_linear(xd, grouped.words(), s, z, group=64, **kw), grouped.call(xd))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = layer.call(x)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


def test_graph():
    """Captured with adapters and split columns; replays follow the inputs, eager work between them."""
    layer = Layer(40, 9000, -8, 7, 128, True, seed=4)
    words, scale, zero = layer.words(), layer.scale.to(DEV), layer.zero.to(DEV)
    x = torch.randn(20, 9000, generator=layer.g).bfloat16().to(DEV)
    adapters, index = make_adapters(4, 10, layer, x.dtype, 20, layer.g)
    adapters, index = Adapters(*(t.to(DEV) for t in adapters)), index.to(DEV)
    run = lambda: packed_linear(x, words, scale, zero, qmin=-8, qmax=7, group=128, adapters=adapters, index=index)
    run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for turn in range(4):
        x.normal_()
        index.copy_((index + 2) % 5 - 1)
        want = run()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want), turn


def test_what_the_framework_packs():
    """From a layer that quantize_model packs: the product with its words equals the product with its weights."""
    g = torch.Generator().manual_seed(0)
    lin = torch.nn.Linear(96, 80, bias=True).to(DEV)
    model = torch.nn.Sequential(lin)
    x = torch.randn(40, 96, generator=g).to(DEV)
    with MD.HessianCollector(model, output_side=False) as col, torch.no_grad():
        model(x)
    res, = MD.quantize_model(model, col)
    y = packed_linear(x, res.words, res.scale, res.zero_point, qmin=-8, qmax=7, bias=lin.bias.detach())
    want = torch.nn.functional.linear(x.double().cpu(), lin.weight.detach().double().cpu(),
                                      lin.bias.detach().double().cpu())
    assert float((y.double().cpu() - want).abs().max()) < 1e-5
    spec = MD.int_row_quantizer(lin.weight.detach())
    words = packing.pack_int(lin.weight.detach(), res.scale, qmin=-8, qmax=7)
    assert torch.equal(words, res.words) and spec.pack_zero is None


def test_nothing_to_do():
    layer = Layer(20, 64, -8, 7, 0, False, seed=5)
    assert layer.call(torch.zeros(0, 64)).shape == (0, 20)
    x = torch.randn(3, 64, generator=layer.g)
    none = Adapters(torch.zeros(0, 4, 64, device=DEV), torch.zeros(0, 20, 4, device=DEV))
    got = layer.call(x, adapters=none, index=torch.zeros(3, dtype=torch.int32, device=DEV))
    assert torch.equal(got, layer.call(x))


def test_refusals():
    layer = Layer(20, 64, -8, 7, 0, False, seed=6)
    words, scale = layer.words(), layer.scale.to(DEV)
    x = torch.zeros(3, 64, device=DEV)
    a, b = torch.zeros(2, 4, 64, device=DEV), torch.zeros(2, 20, 4, device=DEV)
    index = torch.zeros(3, dtype=torch.int32, device=DEV)
    ok = dict(qmin=-8, qmax=7)
    packed_linear(x, words, scale, adapters=(a, b), index=index, **ok)
    bad = [
        lambda: packed_linear(x.double(), words, scale, **ok),
        lambda: packed_linear(torch.zeros(3, 65, device=DEV), words, scale, **ok),
        lambda: packed_linear(x, words.long(), scale, **ok),
        lambda: packed_linear(x, words.t().contiguous().t(), scale, **ok),
        lambda: packed_linear(x, words.cpu(), scale, **ok),
        lambda: packed_linear(x, words, scale.half(), **ok),
        lambda: packed_linear(x, words, scale.cpu(), **ok),
        lambda: packed_linear(x, words, scale[:7], **ok),
        lambda: packed_linear(x, words, scale, torch.zeros(20, 2, device=DEV), **ok),
        lambda: packed_linear(x, words, scale, group=48, **ok),
        lambda: packed_linear(x, words, scale, group=0, **ok),
        lambda: packed_linear(x, words, scale, qmin=-16, qmax=15),
        lambda: packed_linear(x, words, scale, qmin=0.5, qmax=15),
        lambda: packed_linear(x, words, scale, bias=torch.zeros(19, device=DEV), **ok),
        lambda: packed_linear(x, words, scale, bias=torch.zeros(20, device=DEV).half(), **ok),
        lambda: packed_linear(x, words, scale, adapters=(a, b), **ok),
        lambda: packed_linear(x, words, scale, index=index, **ok),
        lambda: packed_linear(x, words, scale, adapters=(a.half(), b.half()), index=index, **ok),
        lambda: packed_linear(x, words, scale, adapters=(a, b[:, :19]), index=index, **ok),
        lambda: packed_linear(x, words, scale, adapters=(a, b.transpose(1, 2).contiguous().transpose(1, 2)), index=index, **ok),
        lambda: packed_linear(x, words, scale, adapters=(a, b), index=index.long(), **ok),
        lambda: packed_linear(x, words, scale, adapters=(a, b), index=index[:2], **ok),
        lambda: packed_linear(x, words, scale, adapters=(a, b, torch.zeros(2, device=DEV).double()), index=index, **ok),
    ]
    for call in bad:
        with pytest.raises(ValueError):
            call()
    with pytest.raises(_hip.GPTQ2DError):
        packed_linear(x.cpu(), words, scale, **ok)


@pytest.mark.parametrize("dtype", list(TYPES))
def test_more_adapters_in_sixteen_tokens_than_workgroups(dtype):
    """1300 tokens (82 tiles of 16, each shared out to fewer workgroups than it has adapters), 40 adapters in any order."""
    layer = Layer(24, 160, -8, 7, 32, True, seed=9)
    x = torch.randn(1300, layer.n, generator=layer.g).to(TYPES[dtype])
    adapters, index = make_adapters(40, 35, layer, x.dtype, 1300, layer.g)
    want, slack = reference(x, layer, None, adapters, index)
    check(layer.call(x, adapters=Adapters(*(t.to(DEV) for t in adapters)), index=index.to(DEV)), want, slack)


@pytest.mark.parametrize("n", [8000, 16384, 16512, 20001])
def test_long_rows(n):
    """Rows that stay in a workgroup's registers while they are brought to fp16, and rows that do not."""
    for group, zero in ((0, True), (256, True), (32, True)):
        layer = Layer(5, n, -8, 7, group, zero, seed=n + group)
        x = torch.randn(3, n, generator=layer.g).bfloat16()
        want, slack = reference(x, layer)
        check(layer.call(x), want, slack * (n / 9000 if n > 9000 else 1))


def test_rows_too_far_apart_are_refused():
    """Byte offsets within a workgroup's rows have 31 bits: a stride beyond is an error, not a wrong result."""
    words = torch.zeros((1 << 28) + 300, dtype=torch.int32, device=DEV).as_strided((2, 16), ((1 << 28) + 1, 1))
    with pytest.raises(_hip.GPTQ2DError):
        packed_linear(torch.ones(3, 128, device=DEV), words, torch.ones(2, 1, device=DEV), qmin=-8, qmax=7)


@pytest.mark.parametrize("bits", [2, 3, 4, 8])
@pytest.mark.parametrize("tokens", [3, 30, 140])
def test_words_that_end_where_their_storage_does(tokens, bits):
    """Words as the last columns of a wider array, few tokens and many: nothing behind the last row's codes is read, and what
    lies between the rows' codes is of no matter."""
    half = 1 << (bits - 1)
    layer = Layer(40, 200, -half, half - 1, 0, False, seed=bits)
    x = torch.randn(tokens, 200, generator=layer.g).bfloat16().to(DEV)
    words = layer.words()
    wide = torch.full((40, words.size(1) + 15), -1, dtype=torch.int32, device=DEV)
    wide[:, 15:] = words
    kw = dict(qmin=-half, qmax=half - 1)
    got = packed_linear(x, wide[:, 15:], layer.scale.to(DEV), **kw)
    assert torch.equal(got, packed_linear(x, words, layer.scale.to(DEV), **kw))
    want, slack = reference(x.cpu(), layer)
    check(got, want, slack)


@pytest.mark.parametrize("tokens", [2, 24, 140])
def test_first_call_of_a_kernel_in_a_graph(tokens):
    """A kernel that the process has not launched yet may be captured: 2-bit codes in groups of 160, which no other test has."""
    layer = Layer(50, 800, -2, 1, 160, tokens > 30, seed=tokens)
    x = torch.randn(tokens, 800, generator=layer.g).half().to(DEV)
    words, scale = layer.words(), layer.scale.to(DEV)
    zero = None if layer.zero is None else layer.zero.to(DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = packed_linear(x, words, scale, zero, qmin=-2, qmax=1, group=160)
    for turn in range(3):
        x.normal_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        want, slack = reference(x.cpu(), layer)
        check(out, want, slack)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("what", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("tokens", [7, 60, 150, 400])
def test_adapters_that_are_no_numbers(tokens, what, dtype):
    """An infinity or NaN in one adapter (its A, its B or its scaling) changes the tokens that have it and no others, in short
    batches and in long ones, where 16 tokens share the matrix cores' tiles."""
    layer = Layer(70, 200, -8, 7, 0, False, seed=tokens)
    x = torch.randn(tokens, layer.n, generator=layer.g).to(TYPES[dtype])
    adapters, index = make_adapters(4, 20, layer, x.dtype, tokens, layer.g)
    index[tokens // 2] = 2
    run = lambda ad: layer.call(x, adapters=Adapters(*(t.to(DEV) for t in ad)), index=index.to(DEV)).cpu()
    clean, own = run(adapters), index == 2
    for part in range(3):
        dirty = [t.clone() for t in adapters]
        dirty[part].view(4, -1)[2] = what
        got = run(dirty)
        assert torch.equal(got[~own], clean[~own])
        assert not bool(got[own].isfinite().any())


@pytest.mark.parametrize("group", [0, 32, 128])
@pytest.mark.parametrize("tokens", [2, 20, 140])
def test_infinities_beside_rows_of_other_zero_points(tokens, group):
    """A row with whole zero points gives what it gives alone, whatever its neighbours' zero points are: infinities of the
    weight's sign where an activation is infinite."""
    layer = Layer(64, 300, 0, 15, group, True, seed=tokens + group)
    layer.zero = layer.zero - 0.5 + 8.
    x = torch.randn(tokens, 300, generator=layer.g).bfloat16()
    x[1, 40] = math.inf
    whole = layer.call(x).cpu()
    sign = layer.weights()[:, 40].sign()
    assert torch.equal(whole[1].double()[sign != 0], sign[sign != 0] * math.inf)
    layer.zero[1::2] += 0.25
    mixed = layer.call(x).cpu()
    assert torch.equal(mixed[:, ::2].nan_to_num(7.), whole[:, ::2].nan_to_num(7.))
    finite = torch.arange(tokens) != 1
    want, slack = reference(x[finite], layer)
    check(mixed[finite], want, slack)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("tokens", [3, 30, 150])
def test_tokens_of_subnormal_numbers(tokens, dtype):
    """Tokens whose largest element is anything down to the type's least positive number, against weights near 1e35."""
    layer = Layer(40, 300, -8, 7, 64, True, seed=tokens)
    layer.scale *= 1e36
    x = torch.randn(tokens, 300, generator=layer.g) * torch.logspace(-38, -44, tokens).view(-1, 1)
    least = 2.0 ** -149 if dtype == "f32" else 2.0 ** -133
    x[0], x[0, 5], x[1] = 0., least, 0.
    x = x.to(TYPES[dtype])
    want, slack = reference(x, layer)
    check(layer.call(x), want, slack)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("tokens", [2, 30, 150])
def test_a_large_element_whose_weight_is_zero(tokens, dtype):
    """What is held of the others beside it: 22 bits, or 2^-39 of the largest."""
    layer = Layer(40, 300, -8, 7, 0, False, seed=tokens)
    layer.codes[:, 7] = 0
    for up in (10, 20, 30, 36):
        x = torch.randn(tokens, 300, generator=layer.g)
        x[:, 7] = 0.
        x = x.double()
        x *= 2.0 ** (-20 if dtype == "f16" else 0)
        x[:, 7] = 2.0 ** (up - (20 if dtype == "f16" else 0)) * 0.99
        x = x.to(TYPES[dtype])
        if not bool(x.isfinite().all()):
            continue
        want, slack = reference(torch.where(torch.arange(300) == 7, 0., x), layer)
        held = 2.0 ** -39 * x.double().abs().amax(1, keepdim=True) * layer.size().sum(1)
        check(layer.call(x), want, slack + held)


@pytest.mark.parametrize("tokens", [2, 140])
def test_strides_of_axes_of_one(tokens):
    """One row, one word a row, one column: the stride of an axis with one entry is of no matter."""
    for m, n in ((1, 100), (70, 7), (1, 1)):
        layer = Layer(m, n, -8, 7, 0, False, seed=m + n)
        x = torch.randn(tokens, n, generator=layer.g).to(DEV)
        want, words = layer.call(x), layer.words()
        strides = (words.size(1) if m > 1 else 1, 1 if words.size(1) > 1 else m + 3)
        odd = torch.zeros(4096, dtype=torch.int32, device=DEV).as_strided(words.shape, strides)
        odd.copy_(words)
        assert torch.equal(packed_linear(x, odd, layer.scale.to(DEV), qmin=-8, qmax=7), want)
        if n == 1:
            wide = torch.zeros(tokens, 5, device=DEV)
            wide[:, :1] = x
            assert torch.equal(layer.call(wide.as_strided((tokens, 1), (5, 9))), want)
