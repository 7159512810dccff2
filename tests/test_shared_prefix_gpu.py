"""Attention of requests that share their first pages, against one softmax a token in 64 bits.

Tolerances.  A score is a dot product of hd fp32 multiply-adds, so it is off by (hd + 4) half steps (2^-24) of sum|q k| scale at most
(tanh and exp a few more: 8), which moves an output by twice that times the largest |v|; the weighted sum of n keys and the joins add
n + 64 half steps of max|v|.  Where products run in bfloat16 the weights are rounded to it (2^-8 of max|v|), and so is the output."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
F64 = torch.float64
PAGE = 64
FILL = 7.0


@pytest.fixture(autouse=True)
def guard_bands():
    from gpu_util import GuardedOutputs
    with GuardedOutputs() as guard:
        yield guard
        guard.check()
        guard.forget()


class Case:
    """Groups as lists of (shared pages, [(tokens, own keys), ...]); the pages lie in the pool in no order."""

    def __init__(self, groups, heads, kv, dim, dtype, seed=0, idle=0, sink=False, softcap=0.0, spare=2, q_scale=1.0):
        g = torch.Generator().manual_seed(seed)
        total = sum(p + sum(-(-own // PAGE) for _, own in reqs) for p, reqs in groups) + spare
        order = torch.randperm(total, generator=g).tolist()
        self.rows, self.positions, self.segment, self.starts = [], [], [], [0]
        for shared, reqs in groups:
            front = [order.pop() for _ in range(shared)]
            for tokens, own in reqs:
                self.rows.append(front + [order.pop() for _ in range(-(-own // PAGE))])
                self.positions += [shared * PAGE + own - tokens + t for t in range(tokens)]
                self.segment += [len(self.rows) - 1] * tokens
            self.starts.append(len(self.positions))
        self.live, self.idle = len(self.positions), idle
        self.width = max(1, max((len(r) for r in self.rows), default=1))
        self.table = torch.tensor([r + [-1] * (self.width - len(r)) for r in self.rows], dtype=torch.int32).reshape(-1, self.width)
        self.pages = [p for p, _ in groups]
        self.heads, self.kv, self.dim, self.dtype, self.softcap = heads, kv, dim, dtype, softcap
        self.k = torch.randn(total, kv, PAGE, dim, generator=g).to(dtype)
        self.v = torch.randn(total, kv, PAGE, dim, generator=g).to(dtype)
        self.q = (q_scale * torch.randn(self.live + idle, heads * dim, generator=g)).to(dtype)
        self.sink = torch.randn(heads, generator=g) if sink else None
        self.scale = dim ** -0.5

    def device(self):
        def i32(v):
            return torch.as_tensor(v, dtype=torch.int32).to(DEV)
        out = torch.full(self.q.shape, FILL, dtype=self.dtype, device=DEV)
        return dict(q=self.q.to(DEV), k_pool=self.k.to(DEV), v_pool=self.v.to(DEV), positions=i32(self.positions + [0] * self.idle),
                    tok_seg=i32(self.segment + [0] * self.idle), block_table=i32(self.table), group_start=i32(self.starts),
                    group_pages=i32(self.pages), n_heads=self.heads, scale=self.scale,
                    sink=None if self.sink is None else self.sink.to(DEV), softcap=self.softcap, out=out)

    def check(self, got):
        got = got.cpu().to(F64)
        assert (got[self.live:] == FILL).all(), "rows of no group were written"
        per = self.heads // self.kv
        for t in range(self.live):
            n, row = self.positions[t] + 1, self.rows[self.segment[t]]
            if n <= 0:
                assert not got[t].any()
                continue
            pages = row[:-(-n // PAGE)]
            k = self.k[pages].transpose(0, 1).flatten(1, 2)[:, :n].to(F64)
            v = self.v[pages].transpose(0, 1).flatten(1, 2)[:, :n].to(F64)
            q = self.q[t].to(F64).view(self.kv, per, self.dim)
            s = torch.bmm(q, k.transpose(1, 2)) * self.scale
            size = (torch.bmm(q.abs(), k.abs().transpose(1, 2)) * abs(self.scale)).amax().item()
            if self.softcap:
                s = self.softcap * torch.tanh(s / self.softcap)
            if self.sink is not None:
                s = torch.cat([s, self.sink.to(F64).view(self.kv, per, 1)], dim=2)
            want = torch.bmm(torch.softmax(s, dim=2)[:, :, :n], v).flatten()
            top = v.abs().max().item()
            bound = top * 2.0 ** -24 * (2 * (self.dim + 8) * size + 16 + n + 64)
            if self.dtype == torch.bfloat16:
                bound += 2 * 2.0 ** -8 * top
            err = (got[t] - want).abs().max().item()
            assert err <= bound, f"token {t} (position {n - 1}): off by {err:.3e}, allowed {bound:.3e}"


def attend(case, **more):
    from flyweight_b200.kernels import attention
    return attention.shared_prefix_attention(**{**case.device(), **more})


@pytest.fixture(params=["two launches", "one launch"])
def cut(request, monkeypatch):
    """The sizes of most tests here choose one launch; the same with the shared pages once a group, in slices."""
    from flyweight_b200.kernels import attention
    rule = attention.shared_prefix_splits

    def pinned(n_tokens, n_kv, group, head_dim, shared, own, wide, groups):
        if request.param == "one launch" and wide:
            return 0, 1 if own < 4 else 4
        return (min(shared, 7), 2 if wide and own > 3 else 1)
    monkeypatch.setattr(attention, "shared_prefix_splits", pinned)
    yield rule


SHAPES = [(4, 4, 64), (8, 2, 64), (6, 2, 128), (16, 1, 128), (8, 8, 16), (10, 5, 80), (12, 4, 96), (9, 3, 48), (5, 1, 32)]
WIDE = [(3, 1, 256), (20, 1, 64), (128, 1, 64), (70, 1, 40), (2, 2, 200)]
BATCHES = {
    "two": [(3, [(1, 5), (1, 64)])],
    "one request": [(2, [(1, 100)])],
    "groups": [(1, [(1, 1), (1, 65), (1, 130)]), (4, [(2, 3), (3, 70)]), (0, [(1, 200), (2, 2)])],
    "many": [(9, [(1, 1 + 7 * i) for i in range(40)])],
    "long": [(40, [(1, 300), (1, 1), (4, 64)])],
    "nothing shared": [(0, [(1, 1), (1, 63), (1, 129)])],
    "empty groups": [(2, []), (1, [(1, 9)]), (3, []), (2, [(1, 64)])],
}


@pytest.mark.parametrize("batch", sorted(BATCHES))
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("heads,kv,dim", SHAPES)
def test_against_one_softmax_a_token(cut, batch, dtype, heads, kv, dim):
    case = Case(BATCHES[batch], heads, kv, dim, dtype, idle=3 if batch == "groups" else 0)
    case.check(attend(case))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("heads,kv,dim", WIDE)
def test_wide_heads_and_wide_groups(cut, dtype, heads, kv, dim):
    case = Case(BATCHES["groups"], heads, kv, dim, dtype, idle=1)
    case.check(attend(case))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dim", [64, 80, 128])
@pytest.mark.parametrize("sink,softcap", [(True, 0.0), (False, 5.0), (True, 30.0)])
def test_sink_and_cap(cut, dtype, dim, sink, softcap):
    case = Case(BATCHES["groups"], 8, 2, dim, dtype, sink=sink, softcap=softcap, q_scale=3.0)
    case.check(attend(case))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dim", [64, 96])
def test_positions_inside_the_shared_pages_and_before_the_first(cut, dtype, dim):
    """A token may stand inside the shared pages (it sees them up to itself) or nowhere (a padded row)."""
    case = Case([(4, [(1, 10), (1, 10), (1, 10), (1, 10), (1, 10)])], 8, 2, dim, dtype)
    case.positions = [0, 100, 255, -1, 256 + 9]
    case.check(attend(case))


RUNS = {
    "drafts": [(2, [(3, 40), (1, 9), (4, 66), (2, 2), (5, 200)]), (1, [(7, 64), (3, 63)])],
    "a prompt beside": [(1, [(1, 5), (77, 140), (1, 30), (33, 33)]), (0, [(100, 100), (2, 65)])],
    "all of one": [(3, [(50, 300)])],
}


@pytest.fixture(params=["together", "one by one"])
def neighbours(request, monkeypatch):
    """The rule takes neighbours together in large batches only."""
    from flyweight_b200.kernels import attention
    monkeypatch.setattr(attention, "neighbours_together", lambda *sizes: request.param == "together")


def test_neighbours_are_taken_together_in_large_batches():
    from flyweight_b200.kernels.attention import neighbours_together
    assert neighbours_together(256, 64, 8) and neighbours_together(295, 96, 4)
    assert not neighbours_together(64, 16, 8) and not neighbours_together(256, 256, 8)
    case = Case([(2, [(4, 30 + i) for i in range(64)])], 8, 4, 64, torch.bfloat16)
    case.check(attend(case))


@pytest.mark.parametrize("batch", sorted(RUNS))
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("heads,kv,dim", [(4, 4, 64), (8, 4, 128), (3, 1, 64), (12, 3, 128), (10, 2, 80), (6, 1, 128), (7, 1, 48), (16, 2, 64),
                                          (9, 1, 64), (16, 1, 128), (34, 2, 64)])
def test_several_tokens_of_a_request(cut, neighbours, batch, dtype, heads, kv, dim):
    """Neighbouring tokens of a request are taken together, whatever their number and the heads of each."""
    case = Case(RUNS[batch], heads, kv, dim, dtype, idle=2)
    case.check(attend(case))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dim", [64, 128])
def test_tokens_of_a_request_in_any_order(cut, neighbours, dtype, dim):
    """Positions that fall, jump, repeat or are none; a request whose tokens do not lie together; one request on both sides of a
    border of groups."""
    case = Case([(2, [(9, 300)]), (1, [(4, 100), (3, 20)])], 6, 2, dim, dtype)
    case.positions[:9] = [427, 130, 131, -1, 300, 300, 129, 5, 426]
    case.check(attend(case))
    case = Case([(1, [(2, 50), (2, 60), (2, 70)])], 4, 2, dim, dtype)
    case.segment = [0, 1, 0, 2, 2, 1]
    case.positions = [64 + 48, 64 + 58, 64 + 49, 64 + 69, 64 + 68, 64 + 59]
    case.check(attend(case))
    case = Case([(1, [(6, 200)])], 4, 2, dim, dtype)
    case.starts, case.pages = [0, 2, 6], [1, 0]
    case.check(attend(case))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dim", [64, 128, 80])
def test_a_later_token_of_a_request_is_not_seen(cut, neighbours, dtype, dim):
    """Infinities in the value and NaN in the key of a request's last token: the tokens in front of it do not see them."""
    case = Case([(1, [(3, 40), (1, 7), (5, 66)])], 6, 2, dim, dtype)
    want = attend(case).clone()
    for row, n in zip((0, 2), (64 + 40, 64 + 66)):
        page = case.rows[row][(n - 1) // PAGE]
        case.k[page, :, (n - 1) % PAGE], case.v[page, :, (n - 1) % PAGE] = math.nan, math.inf
    got = attend(case)
    seen = [0, 1, 3, 4, 5, 6, 7]
    assert torch.equal(got[seen], want[seen])
    assert torch.isnan(got[[2, 8]].float()).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dim", [64, 128, 80])
def test_what_lies_behind_the_last_key_is_not_seen(cut, dtype, dim):
    """Infinities and NaN in keys and values that no token may see: behind the requests' last keys and in unmapped pages."""
    case = Case([(2, [(1, 5), (1, 70)]), (0, [(1, 33)])], 8, 4, dim, dtype)
    want = attend(case).clone()
    for row, n in zip(case.rows, (2 * PAGE + 5, 2 * PAGE + 70, 33)):
        page, inside = row[(n - 1) // PAGE], (n - 1) % PAGE + 1
        case.k[page, :, inside:], case.v[page, :, inside:] = math.nan, math.inf
    held = {p for row in case.rows for p in row}
    for page in range(case.k.shape[0]):
        if page not in held:
            case.k[page], case.v[page] = math.inf, math.nan
    assert torch.equal(attend(case), want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dim", [64, 128, 80])
def test_the_lowest_and_largest_numbers(cut, dtype, dim):
    """Scores far apart between shared and own keys, either way round: the part that weighs nothing adds nothing."""
    for which in (0, 1):
        case = Case([(3, [(1, 70), (1, 3)])], 4, 2, dim, dtype)
        q = torch.ones_like(case.q)
        case.q = q
        for r, row in enumerate(case.rows):
            for i, page in enumerate(row):
                case.k[page] = 30.0 if (i < 3) == (which == 0) else -30.0
        case.check(attend(case))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_the_cut_of_the_work_is_only_a_cut(dtype):
    case = Case([(30, [(1, 5 + 90 * i) for i in range(6)])], 8, 2, 64, dtype)
    for shared, own in ((1, 1), (30, 8), (1000, 1000), (7, 2)):
        case.check(attend(case, shared_pages=shared, own_pages=own))


@pytest.mark.parametrize("dim", [64, 128])
def test_equals_the_attention_that_reads_every_request(cut, dim):
    """Beside the framework's own decode attention on the same pages: two bfloat16 computations of one value."""
    from flyweight_b200.kernels import attention, ops
    case = Case([(20, [(1, 33 * i + 1) for i in range(9)])], 16, 4, dim, torch.bfloat16)
    d = case.device()
    splits, per, cluster = attention.decode_splits(case.live, 4, case.width, dim)
    other = ops.attention_decode_mma(d["q"], d["k_pool"], d["v_pool"], d["positions"], d["tok_seg"], d["block_table"], 16, 0,
                                     case.scale, splits, per, cluster)
    assert (attend(case).float() - other.float()).abs().max().item() <= 4 * 2.0 ** -8 * case.v.abs().max().item()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_pages_outside_the_pool_are_not_read(cut, dtype):
    """A page id that is none: its keys are not seen, and nothing is read for it."""
    for dim in (64, 80):
        case = Case([(3, [(1, 10), (1, 100)])], 4, 2, dim, dtype)
        d = case.device()
        d["block_table"][:, 1] = 10 ** 6
        d["block_table"][1, 3] = -1
        from flyweight_b200.kernels import attention
        got = attention.shared_prefix_attention(**d)
        # what is left: pages 0 and 2 of both, request 0's own keys, request 1's second own page
        short = Case([(3, [(1, 10), (1, 100)])], 4, 2, dim, dtype)
        short.rows = [[r[0], r[2], r[3]] if i == 0 else [r[0], r[2], r[4]] for i, r in enumerate(short.rows)]
        short.positions = [2 * PAGE + 9, 2 * PAGE + 35]
        short.check(got)


def test_the_rule_of_the_cut():
    """Few shared pages a block: one launch; else slices by what walking a page and what a slice's results cost, not more than fill
    the SMs twice (once, where that leaves room for the kernel behind), at most 64 and one a page."""
    from flyweight_b200.kernels import attention
    rule = attention.shared_prefix_splits
    assert rule(2, 8, 2, 64, 7, 1, True) == (0, 8)
    assert rule(2, 8, 2, 128, 128, 1, True)[0] == 32               # one row tile of eight KV heads: 37 slices at most, 4 pages each
    assert rule(4, 8, 4, 64, 128, 4, True)[0] == 16                # 128 blocks, beside which the own kernel's find room
    assert rule(64, 8, 4, 64, 8, 1, True)[0] == 0 and rule(64, 8, 4, 64, 16, 1, True)[0] > 1
    assert rule(2048, 8, 4, 64, 8, 1, True)[0] > 0                 # several rounds of blocks
    assert rule(2, 8, 2, 64, 7, 1, False) == (7, 1)                # the 32-bit kernels always read the shared pages once
    for tokens in (1, 5, 300):
        for pages in (1, 9, 1000):
            shared, own = rule(tokens, 4, 6, 64, pages, 50, True)
            assert 0 <= shared <= min(64, pages) and own in (1, 2, 4, 8)


@pytest.mark.parametrize("which", ["q", "k_pool", "v_pool", "out"])
def test_tensors_off_a_border(which):
    """Storage that starts two bytes behind a border of 16 takes the kernels that read value by value."""
    from flyweight_b200.kernels import attention
    case = Case(BATCHES["two"], 8, 2, 64, torch.bfloat16)
    d = case.device()
    held = torch.full((d[which].numel() + 1,), FILL, dtype=torch.bfloat16, device=DEV)
    held[1:] = d[which].flatten()
    d[which] = held[1:].view(d[which].shape)
    assert d[which].data_ptr() % 16 and d[which].is_contiguous()
    case.check(attention.shared_prefix_attention(**d))
    assert which != "out" or held[0] == FILL


@pytest.mark.parametrize("more", [dict(scale=0.0), dict(scale=-0.125), dict(scale=math.nan), dict(scale=math.inf),
                                  dict(softcap=math.inf), dict(shared_pages=-1), dict(own_pages=-1)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_numbers_that_are_refused(dtype, more):
    from flyweight_b200.kernels import KernelError
    with pytest.raises(KernelError):
        attend(Case(BATCHES["two"], 4, 2, 64, dtype), **more)


def test_no_groups_and_no_tokens():
    case = Case(BATCHES["two"], 4, 4, 64, torch.bfloat16)
    d = case.device()
    from flyweight_b200.kernels import attention
    none = {**d, "group_start": d["group_start"][:1], "group_pages": d["group_pages"][:0]}
    assert (attention.shared_prefix_attention(**none) == FILL).all()
    empty = {**d, "q": d["q"][:0], "out": None}
    assert attention.shared_prefix_attention(**empty).shape == (0, 256)


def test_refusals():
    from flyweight_b200.kernels import KernelError, attention
    case = Case(BATCHES["two"], 4, 2, 64, torch.bfloat16)
    good = case.device()
    bad = [dict(q=good["q"].float()), dict(q=good["q"][:, :128].contiguous()), dict(v_pool=good["v_pool"][:1]),
           dict(k_pool=good["k_pool"][:, :, :32].contiguous(), v_pool=good["v_pool"][:, :, :32].contiguous()), dict(n_heads=3),
           dict(n_heads=0), dict(positions=good["positions"].long()), dict(positions=good["positions"][:1]),
           dict(block_table=good["block_table"].t()), dict(block_table=good["block_table"][:0]),
           dict(group_start=good["group_start"][:1]), dict(softcap=-1.0), dict(softcap=math.nan),
           dict(sink=torch.zeros(3, device=DEV)), dict(out=good["out"].float()), dict(out=good["out"][:1])]
    wide = Case(BATCHES["two"], 2, 2, 264, torch.float32).device()
    for more in bad:
        with pytest.raises(KernelError):
            attention.shared_prefix_attention(**{**good, **more})
    with pytest.raises(KernelError):
        attention.shared_prefix_attention(**wide)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dim", [64, 80, 128])
@pytest.mark.parametrize("position", [-1, -2, -64, -2 ** 31])
def test_a_token_before_the_first_key_sees_nothing(cut, neighbours, dtype, dim, position):
    """Among tokens that see all of the shared pages, so that no other row of the block needs a mask."""
    case = Case([(18, [(1, 10 + i) for i in range(12)]), (2, [(3, 70)])], 8, 2, dim, dtype)
    for token in (0, 5, 11, 13):
        case.positions[token] = position
    case.check(attend(case))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dim", [64, 80, 128])
@pytest.mark.parametrize("position", [-1, -2, -2 ** 31])
def test_a_token_before_the_first_key_takes_nothing_from_its_neighbours(cut, neighbours, dtype, dim, position):
    """Infinities and NaN in the last key and value of the token's own request, which another of its tokens sees."""
    case = Case([(18, [(3, 40), (1, 7), (5, 66)])], 6, 2, dim, dtype)
    case.positions[0] = case.positions[5] = position
    want = attend(case).clone()
    for row, n in zip((0, 2), (18 * 64 + 40, 18 * 64 + 66)):
        page = case.rows[row][(n - 1) // PAGE]
        case.k[page, :, (n - 1) % PAGE], case.v[page, :, (n - 1) % PAGE] = math.nan, math.inf
    got = attend(case)
    seen = [0, 1, 3, 4, 5, 6, 7]
    assert not got[[0, 5]].any() and torch.equal(got[seen], want[seen])
    assert torch.isnan(got[[2, 8]].float()).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("leading", [1, 3, 35])
def test_a_group_led_by_tokens_of_no_request(cut, neighbours, dtype, dim, leading):
    """Finished slots stay in a batch as tokens of no request: they get zeros, and the others of the group see what they saw."""
    from flyweight_b200.kernels import attention
    case = Case([(9, [(1, 10 + i) for i in range(leading + 2)]), (2, [(3, 70), (1, 5)]), (3, [(1, 9)])], 8, 4, dim, dtype)
    d = case.device()
    gone = list(range(leading)) + [leading + 2, leading + 6]       # ... the second group's first token, all of the third group's
    d["tok_seg"][gone] = torch.tensor([-1, len(case.rows)], dtype=torch.int32, device=DEV).repeat(len(gone))[:len(gone)]
    got = attention.shared_prefix_attention(**d)
    for token in gone:
        case.positions[token] = -1
    case.check(got)


@pytest.mark.parametrize("kv,dim", [(0, 64), (2, 0), (0, 0)])
def test_pools_without_heads_are_refused(kv, dim):
    from flyweight_b200.kernels import KernelError
    case = Case(BATCHES["two"], 4, 2, 64, torch.bfloat16)
    pool = torch.zeros(5, kv, 64, dim, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(KernelError):
        attend(case, k_pool=pool, v_pool=pool, q=torch.zeros(2, 4 * dim, dtype=torch.bfloat16, device=DEV), out=None)
