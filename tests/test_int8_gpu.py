"""The 8-bit products and the kernels that make their operands, against the definitions in 64 bits.

The integer sums are exact, so a product has three or four fp32 roundings (2^-24 each, half a step) and the output's: half a step
of bfloat16 is 2^-8.  The rows' integers are compared for equality; behind a norm, whose fp32 value is a few roundings off,
an integer may be the neighbour where the quotient lies that near to a half."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
F64 = torch.float64
HALF = 2.0 ** -24
HALF_BF16 = 2.0 ** -8


@pytest.fixture(autouse=True)
def guard_bands():
    from gpu_util import GuardedOutputs
    with GuardedOutputs() as guard:
        yield guard
        guard.check()
        guard.forget()


def rows_of(R, K, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(R, K, generator=g) * torch.exp(torch.randn(R, 1, generator=g))
    x[:, :: max(1, K // 3)] *= 9.0
    return x.to(dtype)


def define(x):
    """Integers and scales by the definition, on the CPU in 64 bits (the scale is a 32-bit number)."""
    wide = x.to(F64)
    scale = (wide.abs().amax(dim=1) / 127).to(torch.float32)
    values = torch.where(scale[:, None] > 0, wide / scale.to(F64)[:, None], torch.zeros_like(wide)).round()
    return values.clamp(-127, 127), scale


def check_layout(q, R, K):
    assert q.shape == (R, K) and q.values.shape == (R, (K + 15) // 16 * 16) and q.values.dtype == torch.int8
    assert not q.values[:, K:].any(), "columns behind the last one must be zero"


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("R,K", [(1, 1), (3, 7), (1, 16), (5, 100), (2, 2047), (17, 2048), (4, 8192), (3, 10001), (300, 64),
                                 (1, 131071)])
def test_rows_become_the_defined_integers(R, K, dtype):
    from flyweight_b200.kernels import int8
    x = rows_of(R, K, dtype)
    got = int8.rows_int8(x.to(DEV))
    check_layout(got, R, K)
    values, scale = define(x)
    assert torch.equal(got.scales.cpu(), scale)
    assert torch.equal(got.values[:, :K].cpu().to(F64), values)
    assert torch.equal(got.float().cpu(), (values * scale.to(F64)[:, None]).float())


def test_ties_go_to_the_even_integer():
    from flyweight_b200.kernels import int8
    # the scale is exactly 1: halves are exact ties
    x = torch.tensor([[127.0, 0.5, 1.5, 2.5, -0.5, -1.5, -2.5, 63.5, 64.5, -125.5, 126.5, 0.0]])
    got = int8.rows_int8(x.to(DEV)).values[0, :12].tolist()
    assert got == [127, 0, 2, 2, 0, -2, -2, 64, 64, -126, 126, 0]
    # next to a tie by one step of fp32, on both sides
    up, down = math.nextafter(2.5, 3), math.nextafter(2.5, 2)
    near = torch.tensor([[127.0, 2.5 + 2.0 ** -22, 2.5 - 2.0 ** -22, -2.5 - 2.0 ** -22, -2.5 + 2.0 ** -22, 100.5 + 2.0 ** -17]])
    assert up > 2.5 > down
    assert int8.rows_int8(near.to(DEV)).values[0, :6].tolist() == [127, 3, 2, -3, -2, 101]


def test_many_values_next_to_a_half():
    """Scales that are no power of two, values placed on and around every half: the quotient's own rounding decides."""
    from flyweight_b200.kernels import int8
    g = torch.Generator().manual_seed(3)
    top = torch.rand(64, 1, generator=g) * 3 + 0.1
    scale = (top.to(F64) / 127).to(torch.float32)
    halves = torch.arange(-126, 126).to(F64) + 0.5
    x = (halves[None, :] * scale.to(F64)).to(torch.float32)
    x = torch.cat([top, x, torch.nextafter(x, torch.full_like(x, 9.0)), torch.nextafter(x, torch.full_like(x, -9.0))], dim=1)
    values, want_scale = define(x)
    got = int8.rows_int8(x.to(DEV))
    assert torch.equal(got.scales.cpu(), want_scale)
    assert torch.equal(got.values[:, :x.shape[1]].cpu().to(F64), values)


@pytest.mark.parametrize("exponent", [0, -60, 40])
def test_every_bfloat16_value_under_every_maximum(exponent):
    """All eight-bit mantissas of ten binades below all eight-bit maxima: the ties of bfloat16 rows are decided without a check."""
    from flyweight_b200.kernels import int8
    mantissa = torch.arange(128, 256).to(F64) / 128
    x = (mantissa[None, :] * 2.0 ** torch.arange(0, -10, -1).to(F64)[:, None]).flatten()
    rows = torch.cat([mantissa[:, None], x[None, :].expand(128, -1), -x[None, :].expand(128, -1)], dim=1)
    rows = torch.where(rows.abs() <= mantissa[:, None], rows, torch.zeros_like(rows)) * 2.0 ** exponent
    stored = rows.to(torch.bfloat16)
    assert torch.equal(stored.to(F64), rows)
    values, scale = define(stored)
    got = int8.rows_int8(stored.to(DEV))
    assert torch.equal(got.scales.cpu(), scale)
    assert torch.equal(got.values[:, :rows.shape[1]].cpu().to(F64), values)
    many = int8.rows_int8(stored.repeat(20, 1).to(DEV))           # the form that many rows take
    assert torch.equal(many.values[:, :rows.shape[1]].cpu().to(F64), values.repeat(20, 1))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("K", [24, 300, 520, 1000, 1500, 2048, 3500, 5000, 9000, 16392])
def test_many_rows_become_the_same_integers_as_few(K, dtype):
    from flyweight_b200.kernels import int8
    x = rows_of(2400, K, dtype).to(DEV)
    many, few = int8.rows_int8(x), int8.rows_int8(x[:100])
    assert torch.equal(many.values[:100], few.values) and torch.equal(many.scales[:100], few.scales)
    values, scale = define(x[-50:].cpu())
    assert torch.equal(many.values[-50:, :K].cpu().to(F64), values) and torch.equal(many.scales[-50:].cpu(), scale)
    assert not many.values[:, K:].any()
    if dtype == torch.float32:
        w = torch.rand(K, device=DEV) + 0.5
        delta = torch.randn(2400, K, device=DEV)
        held = x.clone()
        many, few = int8.rmsnorm_int8(held, w, 1e-5, delta=delta), int8.rmsnorm_int8(x + delta, w, 1e-5)
        assert torch.equal(held, x + delta)
        assert torch.equal(many.values, few.values) and torch.equal(many.scales, few.scales)


def test_rows_of_zeros_infinities_and_nan():
    from flyweight_b200.kernels import int8
    x = rows_of(6, 200, torch.float32)
    x[1] = 0.0
    x[2, 5] = math.inf
    x[3, 199] = math.nan
    x[4, 0] = -math.inf
    got = int8.rows_int8(x.to(DEV))
    scales = got.scales.cpu()
    assert scales[1] == 0 and not got.values[1].any()
    assert torch.isnan(scales[[2, 3, 4]]).all() and torch.isfinite(scales[[0, 1, 5]]).all()
    w = int8.matrix_int8(rows_of(40, 200, torch.bfloat16, 1).to(DEV))
    y = int8.linear_int8(got, w, torch.float32).cpu()
    assert torch.isnan(y[[2, 3, 4]]).all() and torch.isfinite(y[[0, 5]]).all() and not y[1].any()


@pytest.mark.parametrize("R,K", [(1, 64), (7, 100), (3, 2048), (33, 2047), (2, 8200)])
@pytest.mark.parametrize("with_delta", [False, True])
def test_normed_rows(R, K, with_delta):
    from flyweight_b200.kernels import int8
    g = torch.Generator().manual_seed(5)
    x, w = rows_of(R, K, torch.float32), 1 + 0.2 * torch.randn(K, generator=g)
    delta = torch.randn(R, K, generator=g) if with_delta else None
    held = x.to(DEV)
    got = int8.rmsnorm_int8(held, w.to(DEV), 1e-5, delta=None if delta is None else delta.to(DEV))
    check_layout(got, R, K)
    summed = x if delta is None else x + delta
    assert torch.equal(held.cpu(), summed)
    wide = summed.to(F64)
    y = wide / torch.sqrt((wide * wide).mean(dim=1, keepdim=True) + 1e-5) * w.to(F64)
    # squares: a product and K/2048 + 16 additions deep at most; mean, eps, root, reciprocal; two products
    off = (K / 2048 + 16 + 8) * HALF
    scale = y.abs().amax(dim=1) / 127
    assert ((got.scales.cpu().to(F64) - scale).abs() <= scale * (off + 2 * HALF)).all()
    quotient = y / got.scales.cpu().to(F64)[:, None]
    assert ((got.values[:, :K].cpu().to(F64) - quotient).abs() <= 0.5 + 127 * 2 * off).all()


def test_normed_rows_of_an_index():
    from flyweight_b200.kernels import int8
    x, w = rows_of(9, 96, torch.float32).to(DEV), torch.ones(96, device=DEV)
    rows = torch.tensor([4, 4, 0, 8], dtype=torch.int32, device=DEV)
    some, every = int8.rmsnorm_int8(x, w, 1e-5, rows=rows), int8.rmsnorm_int8(x, w, 1e-5)
    assert torch.equal(some.values, every.values[rows.long()]) and torch.equal(some.scales, every.scales[rows.long()])


@pytest.mark.parametrize("R,K", [(4, 96), (5, 2047), (7, 20000), (2400, 300)])
def test_an_index_that_is_no_row_gives_zeros(R, K):
    from flyweight_b200.kernels import int8
    x, w = rows_of(9, K, torch.float32).to(DEV), torch.ones(K, device=DEV)
    rows = torch.arange(R, dtype=torch.int32) % 9
    rows[1], rows[3] = -1, 9
    some, every = int8.rmsnorm_int8(x, w, 1e-5, rows=rows.to(DEV)), int8.rmsnorm_int8(x, w, 1e-5)
    there = [r for r in range(R) if r not in (1, 3)]
    assert not some.values[[1, 3]].any() and not some.scales[[1, 3]].any()
    assert torch.equal(some.float()[there], every.float()[rows[there].long().to(DEV)])


# tokens, columns, features: one token to a prompt, sizes that fill no tile on either side of every choice of kernel
PRODUCTS = [(1, 16, 8), (1, 2048, 2048), (2, 100, 33), (3, 4097, 130), (7, 1, 5), (8, 2048, 1024), (9, 640, 257), (16, 1024, 4608),
            (17, 512, 129), (24, 96, 300), (31, 1040, 1000), (33, 200, 64), (64, 4096, 512), (65, 129, 260), (100, 48, 1),
            (129, 300, 385), (200, 1024, 640), (257, 257, 257), (513, 2048, 768), (700, 100, 1030), (1100, 512, 520)]


@pytest.mark.parametrize("M,K,N", PRODUCTS)
@pytest.mark.parametrize("form", ["fp32", "bf16", "add", "in place"])
def test_product(M, K, N, form):
    from flyweight_b200.kernels import int8
    x, w = rows_of(M, K, torch.bfloat16, 1), rows_of(N, K, torch.bfloat16, 2)
    rows, matrix = int8.rows_int8(x.to(DEV)), int8.matrix_int8(w.to(DEV))
    (xq, xs), (wq, ws) = define(x), define(w)
    want = (xq @ wq.T) * xs.to(F64)[:, None] * ws.to(F64)[None, :]
    bound = want.abs() * 3 * HALF * 1.01 + 2.0 ** -148
    if form in ("fp32", "bf16"):
        got = int8.linear_int8(rows, matrix, torch.float32 if form == "fp32" else torch.bfloat16)
        if form == "bf16":
            bound = bound + want.abs() * HALF_BF16 * 1.001
    else:
        addend = torch.randn(M, N, generator=torch.Generator().manual_seed(9))
        held = addend.to(DEV)
        got = int8.linear_int8(rows, matrix, torch.float32, addend=held, out=held if form == "in place" else None)
        assert form != "in place" or got is held
        want = want + addend.to(F64)
        bound = bound + want.abs() * HALF * 1.01
    assert got.shape == (M, N)
    assert ((got.cpu().to(F64) - want).abs() <= bound).all()


@pytest.mark.parametrize("M", [1, 5, 40, 300])
def test_a_row_does_not_depend_on_the_others(M):
    """Exact sums and one order of the scales: the bits of a row are the same in every batch, so in every kernel."""
    from flyweight_b200.kernels import int8
    x, matrix = rows_of(600, 1000, torch.bfloat16).to(DEV), int8.matrix_int8(rows_of(700, 1000, torch.bfloat16, 1).to(DEV))
    every, some = int8.linear_int8(x, matrix, torch.float32), int8.linear_int8(x[:M], matrix, torch.float32)
    assert torch.equal(every[:M], some)


@pytest.mark.parametrize("M,K,N", [(1, 100, 40), (33, 700, 130), (70, 2048, 300), (129, 3000, 257), (300, 130, 600)])
@pytest.mark.parametrize("tile,splits", [(8, 1), (32, 1), (32, 2), (32, 8), (64, 1), (64, 4), (128, 1), (128, 2), (128, 8), (-128, 1), (-256, 1)])
def test_every_form_of_the_product_has_the_same_bits(M, K, N, tile, splits):
    """Forms and cuts that the sizes here would not choose; N is even, so that the same matrix has two halves."""
    from flyweight_b200.kernels import int8
    rows, matrix = int8.rows_int8(rows_of(M, K, torch.bfloat16).to(DEV)), int8.matrix_int8(rows_of(2 * N, K, torch.bfloat16, 1).to(DEV))
    addend = torch.randn(M, 2 * N, generator=torch.Generator().manual_seed(4)).to(DEV)
    for epilogue, dtype, features in ((0, torch.float32, 2 * N), (1, torch.bfloat16, 2 * N), (2, torch.float32, 2 * N), (3, torch.bfloat16, N)):
        outs = []
        for form in ((0, 1), (tile if M <= 32 or tile != 8 else 32, splits)):
            outs.append(torch.empty((M, features), dtype=dtype, device=DEV))
            int8._product(rows, matrix, outs[-1], addend if epilogue == 2 else None, features, epilogue, 0.0, *form)
        assert torch.equal(*outs)


def test_the_largest_integers_do_not_overflow():
    from flyweight_b200.kernels import int8
    K = int8.MAX_COLUMNS
    x = torch.ones(2, K, dtype=torch.bfloat16, device=DEV)
    x[1] = -1.0
    got = int8.linear_int8(x, int8.matrix_int8(torch.ones(3, K, dtype=torch.bfloat16, device=DEV)), torch.float32).cpu()
    scale = torch.tensor(1 / 127, dtype=F64).float().to(F64)
    want = 127.0 * 127.0 * K * scale * scale
    assert ((got.to(F64)[0] - want).abs() <= want * 4 * HALF).all() and torch.equal(got[1], -got[0])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("M,K,N", [(1, 8, 3), (1, 2048, 300), (2, 1032, 65), (3, 4096, 100), (5, 24, 1000), (7, 2040, 17), (8, 4088, 260),
                                   (8, 512, 2400), (1, 1024, 4000)])
def test_a_few_rows_become_integers_inside_the_product(M, K, N, dtype):
    """One launch for at most eight rows: the bits of two, with every epilogue, with rows of zeros, infinities and NaN."""
    from flyweight_b200.kernels import int8
    from flyweight_b200.kernels.lib import launch_count
    x = rows_of(M, K, dtype)
    if M > 4:
        x[1], x[2, 0], x[3, K - 1] = 0, math.nan, math.inf
    x, matrix = x.to(DEV), int8.matrix_int8(rows_of(2 * N, K, torch.bfloat16, 1).to(DEV))
    rows, addend = int8.rows_int8(x), torch.randn(M, 2 * N, device=DEV)
    for call in (lambda a: int8.linear_int8(a, matrix, torch.float32), lambda a: int8.linear_int8(a, matrix, torch.bfloat16),
                 lambda a: int8.linear_int8(a, matrix, torch.float32, addend=addend), lambda a: int8.gated_int8(a, matrix, "relu")):
        two, before = call(rows), launch_count()
        one = call(x)
        assert launch_count() - before == 1
        assert torch.equal(torch.isnan(one), torch.isnan(two)) and torch.equal(one.nan_to_num(0), two.nan_to_num(0))


def test_rows_off_a_border_take_two_launches():
    from flyweight_b200.kernels import int8
    matrix = int8.matrix_int8(rows_of(50, 64, torch.bfloat16, 1).to(DEV))
    held = rows_of(1, 1 + 3 * 64, torch.bfloat16).to(DEV).flatten()
    off = held[1:].view(3, 64)
    assert off.data_ptr() % 16 and off.is_contiguous()
    assert torch.equal(int8.linear_int8(off, matrix, torch.float32), int8.linear_int8(off.clone(), matrix, torch.float32))
    assert torch.equal(int8.rows_int8(off).values, int8.rows_int8(off.clone()).values)


@pytest.mark.parametrize("M", [1, 8, 9])
def test_a_result_over_its_own_input(M):
    """``x`` may be the result, and the addend too: every feature is made of the rows as they were."""
    from flyweight_b200.kernels import int8
    matrix = int8.matrix_int8(rows_of(2048, 2048, torch.bfloat16, 1).to(DEV))
    x = rows_of(M, 2048, torch.float32).to(DEV)
    rows = int8.rows_int8(x)
    for addend in (False, True):
        want = int8.linear_int8(rows, matrix, torch.float32, addend=x if addend else None)
        here = x.clone()
        assert int8.linear_int8(here, matrix, torch.float32, addend=here if addend else None, out=here) is here
        assert torch.equal(here, want)
    held = torch.cat([x, x])                                   # overlapping by a part
    over = held.flatten()[64:64 + M * 2048].view(M, 2048)
    want = int8.linear_int8(rows, matrix, torch.float32)
    assert torch.equal(int8.linear_int8(held[:M], matrix, torch.float32, out=over), want)


def test_inputs_in_32_bits_are_brought_to_integers_first():
    from flyweight_b200.kernels import int8
    for M in (1, 6, 130):
        x, matrix = rows_of(M, 333, torch.float32).to(DEV), int8.matrix_int8(rows_of(50, 333, torch.float32, 1).to(DEV))
        assert torch.equal(int8.linear_int8(x, matrix, torch.bfloat16), int8.linear_int8(int8.rows_int8(x), matrix, torch.bfloat16))


def gated(act, limit, g, u):
    if act == "silu":
        return g / (1 + torch.exp(-g)) * u
    if act == "gelu_tanh":
        # 0.5 (1 + tanh(a)) = 1 / (1 + e^(-2 a)), without the cancellation
        return g / (1 + torch.exp(-2 * math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3))) * u
    if act == "relu":
        return g.clamp(min=0) * u
    g, u = g.clamp(max=limit), u.clamp(-limit, limit)
    return g / (1 + torch.exp(-1.702 * g)) * (u + 1)


@pytest.mark.parametrize("M,K,F", [(1, 64, 16), (1, 2048, 1000), (5, 100, 33), (8, 2048, 512), (16, 512, 130), (20, 600, 257),
                                   (48, 300, 96), (64, 2048, 640), (130, 257, 65), (300, 1024, 400), (520, 512, 1000)])
@pytest.mark.parametrize("act", ["silu", "gelu_tanh", "relu", "swish_clamped"])
def test_gated_product(M, K, F, act):
    from flyweight_b200.kernels import int8
    x, w = rows_of(M, K, torch.bfloat16, 1), rows_of(2 * F, K, torch.bfloat16, 2) * K ** -0.5
    limit = 3.0 if act == "swish_clamped" else 0.0
    got = int8.gated_int8(x.to(DEV), int8.matrix_int8(w.to(DEV)), activation=act, limit=limit)
    (xq, xs), (wq, ws) = define(x), define(w)
    y = (xq @ wq.T) * xs.to(F64)[:, None] * ws.to(F64)[None, :]
    want = gated(act, limit, y[:, :F], y[:, F:])
    # the output's rounding; in front of it fp32: the exponent's argument is a few roundings of itself off (|z| up to 88), the
    # hardware exponential and quotient a few more.  From 1 + e^-z = 2^126 on the hardware quotient is 0 where the value is
    # g u 2^-126 at most: an absolute part of that size, which the first run of this test did not allow for
    bound = want.abs() * (HALF_BF16 * 1.001 + 2.0 ** -13) + (y[:, :F] * (y[:, F:].abs() + 1)).abs() * 2.0 ** -125
    if act == "swish_clamped":
        # u + 1 next to u = -1: u itself is three half steps off, the sum one more, of at most (limit + 1), times the swish of g
        g = y[:, :F].clamp(max=limit)
        bound += (g / (1 + torch.exp(-1.702 * g))).abs() * (limit + 1) * 4 * HALF
    assert got.dtype == torch.bfloat16 and got.shape == (M, F)
    assert ((got.cpu().to(F64) - want).abs() <= bound).all()


def test_no_rows_at_all():
    from flyweight_b200.kernels import int8
    matrix = int8.matrix_int8(rows_of(40, 64, torch.bfloat16).to(DEV))
    none = torch.empty((0, 64), dtype=torch.bfloat16, device=DEV)
    assert int8.rows_int8(none).shape == (0, 64)
    assert int8.linear_int8(none, matrix, torch.float32).shape == (0, 40)
    assert int8.gated_int8(none, matrix).shape == (0, 20)


def test_refusals():
    from flyweight_b200.kernels import KernelError, int8
    x, w = rows_of(4, 64, torch.bfloat16).to(DEV), rows_of(10, 64, torch.bfloat16).to(DEV)
    matrix, rows = int8.matrix_int8(w), int8.rows_int8(x)
    for call in (lambda: int8.rows_int8(x.to(torch.float16)), lambda: int8.rows_int8(x.t()), lambda: int8.rows_int8(x[0]),
                 lambda: int8.rows_int8(torch.empty((2, int8.MAX_COLUMNS + 1), dtype=torch.bfloat16, device=DEV)),
                 lambda: int8.rows_int8(torch.empty((2, 0), dtype=torch.bfloat16, device=DEV)),
                 lambda: int8.linear_int8(rows, w, torch.float32), lambda: int8.linear_int8(rows, rows, torch.float32),
                 lambda: int8.linear_int8(rows, matrix, torch.float16),
                 lambda: int8.linear_int8(x[:, :32].contiguous(), matrix, torch.float32),
                 lambda: int8.linear_int8(rows, matrix, torch.bfloat16, addend=torch.zeros(4, 10, device=DEV)),
                 lambda: int8.linear_int8(rows, matrix, torch.float32, addend=torch.zeros(4, 9, device=DEV)),
                 lambda: int8.linear_int8(rows, matrix, torch.float32, out=torch.zeros(3, 10, device=DEV)),
                 lambda: int8.gated_int8(rows, matrix, activation="tanh"),
                 lambda: int8.gated_int8(rows, int8.matrix_int8(w[:9].contiguous())),
                 lambda: int8.rmsnorm_int8(x, torch.ones(64, device=DEV), 1e-5),
                 lambda: int8.rmsnorm_int8(x.float(), torch.ones(63, device=DEV), 1e-5),
                 lambda: int8.rmsnorm_int8(x.float(), torch.ones(64, device=DEV), 1e-5, delta=x.float(),
                                           rows=torch.zeros(1, dtype=torch.int32, device=DEV))):
        with pytest.raises(KernelError):
            call()


@pytest.mark.parametrize("act", ["silu", "gelu_tanh", "relu", "swish_clamped"])
@pytest.mark.parametrize("M,form", [(7, None), (7, (8, 1)), (7, (32, 1)), (30, (8, 1)), (30, (32, 2)), (70, (64, 1)), (70, (64, 4)), (70, (128, 2)),
                                    (70, (-128, 1)), (300, (-256, 1))])
def test_nan_stays_nan_behind_every_gate(M, form, act):
    """A row with an infinity or NaN, and a feature whose gate or up weights hold one: NaN in all that is made of them, whatever the
    activation cuts off, and nowhere else.  ``form`` None: the integers are made inside the product."""
    from flyweight_b200.kernels import int8, ops
    K, F, limit = 512, 260, 3.0
    x, w = rows_of(M, K, torch.bfloat16, 1), rows_of(2 * F, K, torch.bfloat16, 2) * K ** -0.5
    x[2, 0], x[4, K - 1], w[9, 3], w[F + 130, 7], w[F - 1, 0] = math.nan, -math.inf, math.nan, math.inf, -math.inf
    nan = torch.zeros(M, F, dtype=torch.bool)
    nan[[2, 4]], nan[:, [9, 130, F - 1]] = True, True
    matrix, x = int8.matrix_int8(w.to(DEV)), x.to(DEV)
    if form is None:
        got = int8.gated_int8(x, matrix, activation=act, limit=limit)
    else:
        got = torch.empty((M, F), dtype=torch.bfloat16, device=DEV)
        int8._product(int8.rows_int8(x), matrix, got, None, F, 3 | ops.GATE_ACTIVATIONS[act] << 8, limit, *form)
    assert torch.equal(torch.isnan(got).cpu(), nan) and torch.isfinite(got.cpu()[~nan]).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("K", [64, 520, 9000])
def test_small_rows_become_the_defined_integers(K, dtype):
    """Down to rows whose largest value is 127 * 2^-125, so that half of the scale is a normal number; smaller rows are zeros."""
    from flyweight_b200.kernels import int8
    least = 127 * 2.0 ** -125
    tops = torch.tensor([1e-28, 1.1e-30, 9e-31, 3e-33, 1e-35, 3 * least, least * (1 + 2.0 ** -7), least], dtype=F64)
    g = torch.Generator().manual_seed(7)
    x = (torch.rand(len(tops), K, generator=g, dtype=F64) * 2 - 1) * tops[:, None]
    x[:, 5] = tops
    if dtype == torch.float32:                       # values on and next to every half
        scale = (tops.to(dtype).to(F64) / 127).to(dtype).to(F64)
        halves = (torch.arange(40).to(F64) + 0.5) * scale[:, None]
        x[:, 6:46] = halves * (1 + torch.tensor([0.0, 2.0 ** -23, -2.0 ** -23, 2.0 ** -22]).to(F64).repeat(10))
    x = x.to(dtype)
    assert (x.to(F64).abs().amax(dim=1) >= least).all()
    for rows in (x, x.repeat(400, 1)):               # the forms that few and many rows take
        values, scale = define(rows)
        got = int8.rows_int8(rows.to(DEV))
        assert torch.equal(got.scales.cpu(), scale) and torch.equal(got.values[:, :K].cpu().to(F64), values)
    below = torch.full((3, K), least * (1 - 2.0 ** -8), dtype=F64).to(dtype)
    below[1:] *= 2.0 ** -10
    below[2, 1:] = 0
    got = int8.rows_int8(below.to(DEV))
    assert not got.values.any() and not got.scales.any()
