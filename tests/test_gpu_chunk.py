"""Operators on ragged batches of chunks, and copies of cache units, against plain forms in 64 bits (GPU).

Tolerances, all from the types: an output rounded to bf16 is off by up to 2^-8 of itself.  On top of that
  attention   probabilities and partial sums of 11 bits, 2^-11 and 2^-12, and scores and exponentials in fp32 (together
              less than 2^-12): 2^-10 of the weighted mean of |v|;
  delta rule  the operands of its products carry 16 bits or more: each of about six products in a row leaves 2^-16 of the
              sum of its terms' magnitudes, which for 64 or 128 terms of either sign is about 11 times the result:
              2^-10 of the largest output of the sequence and head.  State values: half a code, and 2^-10 of the largest
              of the head's state (a row is a sum of u k over the tokens, off by 2^-16 of the terms; the terms of a row that
              happens to cancel are as large as those of the others, so its own peak says nothing about them);
  gates       decay exp(-x), x = exp(a_log) softplus(a + dt) from two functions and a product in fp32, each off by an ulp
              or two: x is off by at most five of its 2^-23, which moves exp(-x) by |x| 5 2^-23 < |x| 2^-20 of itself, and
              the functions' own roundings 2^-20.  (Until x reaches 104, where fp32 underflows.)
"""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

HEADS, KV, GROUP, WIDE = 24, 4, 6, 256
KEY_HEADS, DIM = 16, 128
EPS = 1e-6


@pytest.fixture(scope="module")
def ops(cuda, built_library):
    from qwencore_b200 import abi, ops as module

    before = abi.get_shape()
    assert abi.lib.qwc_device_status() == 0
    yield module
    abi.configure(*before)
    assert abi.lib.qwc_device_status() == 0


def generator(torch, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def i32(torch, values):
    return torch.tensor(list(values), dtype=torch.int32, device="cuda")


def begins_of(lengths, first=0):
    return [first + int(x) for x in np.concatenate([[0], np.cumsum(lengths)])]


# ---- attention ------------------------------------------------------------------------------------

class Attention:
    """A ragged batch over a shuffled cache; rows before `first` and behind the last chunk belong to nobody."""

    def __init__(self, torch, seed, lengths, past, page=16, gated=True, scaled=True, first=0, padding=0, query_std=1.0,
                 gate_stride=0):
        g = generator(torch, seed)
        self.torch, self.page, self.lengths, self.past = torch, page, lengths, past
        self.contexts = [n + p for n, p in zip(lengths, past)]
        blocks = [max(1, -(-c // page)) for c in self.contexts]
        self.pool, self.widest = sum(blocks) + 2, max(blocks)
        order = np.random.default_rng(seed).permutation(self.pool)
        # behind a sequence's pages the table holds what no pool has
        table = np.full((len(lengths), self.widest), 0x7ffffff0, dtype=np.int64)
        at = 0
        for row, count in enumerate(blocks):
            table[row, :count] = order[at:at + count]
            at += count
        self.table = torch.from_numpy(table.astype(np.int32)).cuda()
        self.first = begins_of(lengths, first)
        self.tokens = self.first[-1] + padding
        randn = lambda *shape: torch.randn(shape, device="cuda", generator=g)  # noqa: E731
        self.query = (randn(self.tokens, HEADS, WIDE) * query_std).bfloat16()
        self.gate_stride = gate_stride
        self.gate = randn(self.tokens, gate_stride or HEADS * 2 * WIDE).bfloat16() if gated else None
        self.scale = (0.5 + torch.rand(KV, device="cuda", generator=g)) / 64.0 if scaled else None
        factor = torch.ones(KV, device="cuda") if self.scale is None else self.scale
        self.caches = [(randn(self.pool, KV, page, WIDE) / factor[None, :, None, None]).clamp(-448, 448)
                       .to(torch.float8_e4m3fn).view(torch.uint8) for _ in range(2)]
        self.output = torch.full((self.tokens, HEADS, WIDE), 7.0, device="cuda").bfloat16()

    def run(self, ops, workspace=None, **other):
        torch = self.torch
        if workspace is None:
            workspace = torch.zeros(max(16, ops.attention_chunk_workspace_bytes()), dtype=torch.uint8, device="cuda")
        self.workspace = workspace
        ops.paged_attention_chunk(self.query, self.gate, *self.caches, self.table, i32(torch, self.contexts),
                                  i32(torch, self.first), self.widest, self.output, self.tokens, len(self.lengths),
                                  workspace, self.page, self.pool, key_scales=self.scale, value_scales=self.scale,
                                  gate_stride=self.gate_stride)
        return self.output

    def want(self):
        torch = self.torch
        out = torch.full((self.tokens, HEADS, WIDE), 7.0, dtype=torch.float64, device="cuda")
        spread = torch.zeros_like(out)
        for s, n in enumerate(self.lengths):
            if n == 0:
                continue
            context = self.contexts[s]
            ids = self.table[s, :max(1, -(-context // self.page))].long() & 0xffffffff  # u32
            k, v = (c[ids.clamp(max=self.pool - 1)].view(torch.float8_e4m3fn).double() *
                    (ids < self.pool)[:, None, None, None] for c in self.caches)
            if self.scale is not None:
                k, v = (x * self.scale.double()[None, :, None, None] for x in (k, v))
            k, v = (x.transpose(0, 1).reshape(KV, -1, WIDE)[:, :context].repeat_interleave(GROUP, 0) for x in (k, v))
            rows = slice(self.first[s], self.first[s] + n)
            q = self.query[rows].double().transpose(0, 1)
            scores = q @ k.transpose(1, 2) / 16.0
            at = torch.arange(n, device="cuda") + context - n
            scores = scores.masked_fill(torch.arange(context, device="cuda")[None] > at[:, None], -torch.inf)
            weights = torch.softmax(scores, -1).nan_to_num(0.0)
            out[rows] = (weights @ v).transpose(0, 1)
            spread[rows] = (weights @ v.abs()).transpose(0, 1)
        if self.gate is not None:
            gate = self.gate[:, :HEADS * 2 * WIDE].reshape(self.tokens, HEADS, 2 * WIDE)[..., WIDE:].double()
            live = slice(self.first[0], self.first[-1])
            out[live] *= torch.sigmoid(gate[live])
            spread[live] *= torch.sigmoid(gate[live])
        return out, spread

    def check(self, ops, **other):
        got = self.run(ops, **other).double()
        want, spread = self.want()
        over = (got - want).abs() - (2.0 ** -8 * want.abs() + 2.0 ** -10 * spread)
        assert not got.isnan().any()
        worst = int(over.argmax())
        assert over.max() <= 0, (np.unravel_index(worst, tuple(got.shape)), float(got.flatten()[worst]),
                                 float(want.flatten()[worst]), float(spread.flatten()[worst]))


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("lengths,past", [
    ([1], [0]), ([1], [1]), ([2], [127]), ([1], [4999]), ([21], [0]), ([22], [107]), ([43], [300]), ([128], [0]),
    ([129], [1]), ([257], [511]), ([5, 1, 64, 3], [0, 700, 65, 129]), ([0, 17, 0, 1, 0], [5, 0, 9, 63, 0]),
    ([1] * 40, list(range(0, 4000, 100))), ([300, 1, 2], [0, 6000, 128])])
def test_attention_chunk(cuda, ops, page, lengths, past):
    Attention(cuda, 3 * page + len(lengths), lengths, past, page).check(ops)


@pytest.mark.parametrize("gated,scaled,stride", [(False, True, 0), (True, False, 0), (False, False, 0),
                                                 (True, True, HEADS * 2 * WIDE + 2048)])
def test_attention_chunk_gate_and_scales(cuda, ops, gated, scaled, stride):
    Attention(cuda, 5, [33, 2, 70], [95, 0, 1000], 16, gated, scaled, gate_stride=stride).check(ops)


def test_attention_chunk_leaves_foreign_rows(cuda, ops):
    case = Attention(cuda, 6, [33, 2, 70], [95, 0, 1000], 64, first=5, padding=9)
    case.check(ops)  # (rows of nobody are 7 in the plain form too)


def test_attention_chunk_rows_that_see_nothing(cuda, ops):
    # a context shorter than its chunk: the first rows would stand before the sequence
    case = Attention(cuda, 7, [50, 4, 30], [0, 0, 40], 16)
    case.contexts = [13, 0, 70]
    case.check(ops)
    assert (case.output[:37] == 0).all() and (case.output[50:54] == 0).all() and (case.output[37:50] != 0).any()


def test_attention_chunk_positions_behind_the_context(cuda, ops):
    # codes that are no number in the rest of the last page, and in pages that no row sees
    case = Attention(cuda, 8, [10, 3], [25, 200], 64)
    for cache in case.caches:
        cache[case.table[0, 0].long(), :, 35:] = 0x7f
        cache[case.table[1, 3].long(), :, 11:] = 0xff
    case.check(ops)


def test_attention_chunk_pages_beyond_the_pool_read_as_zeros(cuda, ops):
    case = Attention(cuda, 9, [40], [200], 16)
    case.table[0, 3] = case.pool
    case.table[0, 7] = -1
    case.check(ops)


def test_attention_chunk_table_shorter_than_the_context(cuda, ops):
    # what the table cannot name is not there, as in the decode attention
    case = Attention(cuda, 10, [20], [300], 16)
    capacity = case.widest * 16
    case.contexts = [capacity]
    case.past = [capacity - 20]
    want, spread = case.want()
    case.contexts = [capacity + 1000]
    got = case.run(ops).double()
    assert ((got - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -10 * spread).all()


@pytest.mark.parametrize("std", [1e-3, 30.0, 3000.0])
def test_attention_chunk_flat_and_steep_scores(cuda, ops, std):
    case = Attention(cuda, 11, [70, 3], [500, 900], 16, query_std=std)
    got = case.run(ops).double()
    want, spread = case.want()
    # a score of magnitude m is off by up to 2^-18 m in fp32 sums of 256 products, and a weight by as much of itself
    largest = float(case.query.double().abs().max()) * 2.0 * 4.0
    bound = 2.0 ** -8 * want.abs() + (2.0 ** -10 + 2.0 ** -18 * largest * 16) * 2 * spread.clamp_min(1.0)
    assert ((got - want).abs() <= bound).all()


@pytest.mark.parametrize("rows", [slice(None), slice(50, 51), slice(0, 300, 90)])
def test_attention_chunk_queries_with_an_outlier(cuda, ops, rows):
    # one element of a million times the others, where all keys are zero: the others decide
    case = Attention(cuda, 14, [300, 40], [700, 90], 16)
    case.caches[0][..., 17] = 0
    case.query[rows, :, 17] = 1.0e6
    case.check(ops)


def test_attention_chunk_queries_that_are_no_numbers(cuda, ops):
    case = Attention(cuda, 15, [100, 50], [300, 0], 16)
    want, spread = case.want()
    case.query[30, 7, 5] = float("nan")
    case.query[120, 3, 9] = float("inf")
    got = case.run(ops).double()
    broken = cuda.zeros((150, HEADS), dtype=cuda.bool, device="cuda")
    broken[30, 7] = broken[120, 3] = True
    assert got[30, 7].isnan().all()
    close = (got - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -10 * spread
    assert close[~broken].all()


def test_attention_chunk_one_large_weight_and_many_small(cuda, ops):
    # a first token that draws half of every row's weight, the rest spread over thousands
    case = Attention(cuda, 12, [40], [8000], 16, gated=False)
    page = case.table[0, 0].long()
    direction = case.query[:, ::GROUP].float().mean(0)
    case.query[:] = (case.query.float() * 0.05 + direction.repeat_interleave(GROUP, 0)[None] * 4).bfloat16()
    case.caches[0][page, :, 0] = ((direction * 12.0) / case.scale[:, None]).clamp(-448, 448).to(
        cuda.float8_e4m3fn).view(cuda.uint8)
    case.check(ops)


def test_attention_chunk_is_the_same_every_time(cuda, ops):
    case = Attention(cuda, 13, [300, 1, 65], [2000, 9000, 0], 16)
    first = case.run(ops).clone()
    for _ in range(3):
        case.output.fill_(1.0)
        assert cuda.equal(case.run(ops, workspace=case.workspace), first)


# ---- delta rule -----------------------------------------------------------------------------------

class Delta:
    def __init__(self, torch, seed, lengths, heads, continues=None, first=0, padding=0, normed=False, gate_offset=0,
                 alike=0.0, rate=(0.002, 2.0)):
        g = generator(torch, seed)
        self.torch, self.lengths, self.heads, self.normed = torch, lengths, heads, normed
        self.first = begins_of(lengths, first)
        self.tokens = tokens = self.first[-1] + padding
        self.capacity = len(lengths) + 2
        rng = np.random.default_rng(seed)
        self.slots = [int(s) for s in rng.permutation(self.capacity)[:len(lengths)]]
        self.continues = continues
        randn = lambda *shape: torch.randn(shape, device="cuda", generator=g)  # noqa: E731
        base = randn(KEY_HEADS, DIM)  # keys that resemble one another
        q, k = (torch.nn.functional.normalize(randn(tokens, KEY_HEADS, DIM) * (1 - alike) + base * alike, dim=-1)
                for _ in range(2))
        v = torch.nn.functional.silu(randn(tokens, heads, DIM))
        self.qkv = torch.cat([(q * DIM ** -0.5).reshape(tokens, -1), k.reshape(tokens, -1), v.reshape(tokens, -1)], 1).bfloat16()
        speed = torch.exp(torch.linspace(np.log(rate[0]), np.log(rate[1]), heads, device="cuda"))
        self.alpha = torch.exp(-speed * torch.nn.functional.softplus(randn(tokens, heads)))
        self.beta = torch.sigmoid(randn(tokens, heads))
        held = randn(self.capacity, heads, DIM, DIM) * 0.1
        peak = held.abs().amax(-1)
        self.codes = (held * (127.0 / peak)[..., None]).round().to(torch.int8)
        self.scales = peak / 127.0
        self.out = torch.full((tokens, heads, DIM), 7.0, device="cuda").bfloat16()
        self.gate = self.weight = None
        self.gate_offset = gate_offset
        self.gate_stride = gate_offset + heads * DIM if gate_offset else 0
        if normed:
            self.gate = randn(tokens, gate_offset + heads * DIM).bfloat16()
            self.weight = (1 + 0.1 * randn(DIM)).bfloat16()

    def run(self, ops, workspace=None):
        from qwencore_b200 import abi
        torch = self.torch
        abi.configure(self.heads, 64)
        if workspace is None:
            workspace = torch.zeros(max(16, ops.delta_chunk_workspace_bytes(self.tokens, len(self.lengths))), dtype=torch.uint8,
                                    device="cuda")
        continues = None if self.continues is None else i32(torch, self.continues)
        ops.delta_chunk(self.codes, self.scales, i32(torch, self.slots), continues, i32(torch, self.first), self.qkv,
                        self.alpha, self.beta, self.out, self.capacity, self.tokens, len(self.lengths), workspace,
                        gate=self.gate, gate_offset=self.gate_offset, gate_stride=self.gate_stride,
                        norm_weight=self.weight, epsilon=EPS)

    def want(self):
        torch = self.torch
        ratio = self.heads // KEY_HEADS
        out = torch.full((self.tokens, self.heads, DIM), 7.0, dtype=torch.float64, device="cuda")
        largest = torch.zeros_like(out)
        rows = self.qkv.double()
        q = rows[:, :KEY_HEADS * DIM].reshape(-1, KEY_HEADS, DIM).repeat_interleave(ratio, 1)
        k = rows[:, KEY_HEADS * DIM:2 * KEY_HEADS * DIM].reshape(-1, KEY_HEADS, DIM).repeat_interleave(ratio, 1)
        v = rows[:, 2 * KEY_HEADS * DIM:].reshape(-1, self.heads, DIM)
        states = self.codes.double() * self.scales.double()[..., None]
        for s, n in enumerate(self.lengths):
            if n == 0:
                continue
            state = states[self.slots[s]].clone()
            if self.continues is not None and not self.continues[s]:
                state.zero_()
            for t in range(self.first[s], self.first[s] + n):
                state *= self.alpha[t].double()[:, None, None]
                wrong = v[t] - torch.einsum("hij,hj->hi", state, k[t])
                state += torch.einsum("hi,hj->hij", wrong * self.beta[t].double()[:, None], k[t])
                out[t] = torch.einsum("hij,hj->hi", state, q[t])
            span = slice(self.first[s], self.first[s] + n)
            largest[span] = out[span].abs().amax((0, 2))[None, :, None]
            states[self.slots[s]] = state
        return out, largest, states

    def check(self, ops, **other):
        torch = self.torch
        before = self.codes.clone(), self.scales.clone()
        want, largest, states = self.want()
        self.run(ops, **other)
        got = self.out.double()
        assert not got.isnan().any()
        live = slice(self.first[0], self.first[-1])
        if self.normed:
            # y = o / sqrt(mean o^2 + eps): an error e of o's elements moves y by e / rms or less, and twice that with the mean's
            rms = torch.sqrt(want.square().mean(-1, keepdim=True) + EPS)
            gate = self.gate[:, self.gate_offset:].double().reshape(self.tokens, self.heads, DIM)
            factor = self.weight.double() * torch.nn.functional.silu(gate)
            error = (2.0 ** -8 * want.abs().amax(-1, keepdim=True) + 2.0 ** -10 * largest) / rms
            want[live] = (want / rms * factor)[live]
            bound = 2.0 ** -8 * want.abs() + 2 * error * factor.abs()
        else:
            bound = 2.0 ** -8 * want.abs() + 2.0 ** -10 * largest
        bound[:live.start] = 0
        bound[live.stop:] = 0
        over = (got - want).abs() - bound
        worst = int(over.argmax())
        assert over.max() <= 0, (np.unravel_index(worst, tuple(got.shape)), float(got.flatten()[worst]),
                                 float(want.flatten()[worst]), float(bound.flatten()[worst]))
        touched = [self.slots[s] for s, n in enumerate(self.lengths) if n]
        values = self.codes.double() * self.scales.double()[..., None]
        peak = states.abs().amax(-1, keepdim=True)
        for slot in range(self.capacity):
            if slot in touched:
                off = (values[slot] - states[slot]).abs() - (peak[slot] * (0.5 / 127) + 2.0 ** -10 * peak[slot].amax(1, keepdim=True))
                assert off.max() <= 0, (slot, float(off.max()))
                assert int(self.codes[slot].abs().max()) == 127 or float(peak[slot].max()) == 0.0
            else:
                assert torch.equal(self.codes[slot], before[0][slot]) and torch.equal(self.scales[slot], before[1][slot])


@pytest.mark.parametrize("heads", [32, 48])
@pytest.mark.parametrize("lengths", [[1], [2], [15], [16], [17], [63], [64], [65], [128], [200], [1, 64, 0, 130, 7],
                                     [3] * 20])
def test_delta_chunk(cuda, ops, heads, lengths):
    Delta(cuda, heads + len(lengths) + lengths[0], lengths, heads).check(ops)


@pytest.mark.parametrize("normed", [False, True])
def test_delta_chunk_begins_and_foreign_rows(cuda, ops, normed):
    Delta(cuda, 21, [70, 1, 0, 65, 30], 32, continues=[1, 0, 0, 0, 1], first=3, padding=6, normed=normed).check(ops)


def test_delta_chunk_gate_inside_wider_rows(cuda, ops):
    Delta(cuda, 22, [70, 9], 48, normed=True, gate_offset=10240).check(ops)


@pytest.mark.parametrize("alike", [0.5, 0.9, 1.0])
def test_delta_chunk_keys_alike(cuda, ops, alike):
    # the triangular system of a block is at its worst when all keys are the same
    Delta(cuda, 23, [130, 40], 32, alike=alike).check(ops)


@pytest.mark.parametrize("rate", [(1e-6, 1e-6), (8.0, 8.0), (60.0, 200.0)])
def test_delta_chunk_decay_of_every_speed(cuda, ops, rate):
    # from a state that nothing leaves to one that the next token has forgotten (alpha underflows)
    Delta(cuda, 24, [150, 20], 32, rate=rate).check(ops)


def test_delta_chunk_alpha_zero_and_one(cuda, ops):
    case = Delta(cuda, 25, [150, 70], 32)
    case.alpha[10::17] = 0.0
    case.alpha[3::5] = 1.0
    case.beta[4::7] = 0.0
    case.beta[5::7] = 1.0
    case.check(ops)


@pytest.mark.parametrize("factor", [1e-6, 1e6])
def test_delta_chunk_small_and_large_values(cuda, ops, factor):
    case = Delta(cuda, 26, [100, 30], 32)
    case.qkv[:, 2 * KEY_HEADS * DIM:] *= factor
    case.scales *= factor
    case.check(ops)


def test_delta_chunk_state_of_zeros(cuda, ops):
    case = Delta(cuda, 27, [20, 5], 32, continues=[0, 0])
    case.qkv[:, 2 * KEY_HEADS * DIM:] = 0
    case.check(ops)
    for slot in case.slots:
        assert not case.codes[slot].any() and not case.scales[slot].any()


def test_delta_chunk_slot_beyond_the_pool(cuda, ops):
    from qwencore_b200 import abi
    case = Delta(cuda, 28, [70, 30], 32)
    want, largest, _ = case.want()
    before = case.codes.clone()
    good = case.slots[1]
    case.slots[0] = case.capacity + 5
    case.run(ops)
    assert abi.lib.qwc_device_status() == 0x105
    abi.check(abi.lib.qwc_device_status_reset(), "reset")
    assert (case.out[:70] == 7.0).all()
    assert ((case.out.double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -10 * largest)[70:].all()
    for slot in range(case.capacity):
        assert slot == good or cuda.equal(case.codes[slot], before[slot])


def test_delta_chunk_is_the_same_every_time(cuda, ops):
    case = Delta(cuda, 29, [200, 65], 48)
    codes, scales = case.codes.clone(), case.scales.clone()
    case.run(ops)
    first = case.out.clone(), case.codes.clone(), case.scales.clone()
    for _ in range(3):
        case.codes.copy_(codes)
        case.scales.copy_(scales)
        case.run(ops)
        assert all(cuda.equal(a, b) for a, b in zip(first, (case.out, case.codes, case.scales)))


# ---- preparation ----------------------------------------------------------------------------------

class Prepare:
    def __init__(self, torch, seed, lengths, heads, continues=None, first=0, padding=0, extra=0, std=1.0):
        g = generator(torch, seed)
        self.torch, self.lengths, self.heads, self.continues = torch, lengths, heads, continues
        self.first = begins_of(lengths, first)
        self.tokens = tokens = self.first[-1] + padding
        self.capacity = len(lengths) + 2
        self.slots = [int(s) for s in np.random.default_rng(seed).permutation(self.capacity)[:len(lengths)]]
        self.channels = (2 * KEY_HEADS + heads) * DIM
        self.width = self.channels + 2 * heads + extra
        randn = lambda *shape: torch.randn(shape, device="cuda", generator=g)  # noqa: E731
        self.mixed = (randn(tokens, self.width) * std).bfloat16()
        self.taps = (randn(self.channels, 4) * 0.5).bfloat16()
        self.a_log, self.dt_bias = (randn(heads) * 0.5).bfloat16(), (randn(heads) * 0.5).bfloat16()
        self.history = randn(self.capacity, self.channels, 3).bfloat16().float()
        self.qkv = torch.full((tokens, self.channels), 7.0, device="cuda").bfloat16()
        self.alpha, self.beta = (torch.full((tokens, heads), 7.0, device="cuda") for _ in range(2))

    def run(self, ops):
        from qwencore_b200 import abi
        torch = self.torch
        abi.configure(self.heads, 64)
        ops.delta_prepare_chunk(self.mixed, self.channels, self.channels + self.heads, self.taps, self.a_log, self.dt_bias,
                                self.history, i32(torch, self.slots),
                                None if self.continues is None else i32(torch, self.continues), i32(torch, self.first),
                                self.qkv, self.alpha, self.beta, self.capacity, self.tokens, len(self.lengths), self.width)

    def check(self, ops):
        torch = self.torch
        history = self.history.double().clone()
        qkv = torch.full(self.qkv.shape, 7.0, dtype=torch.float64, device="cuda")
        for s, n in enumerate(self.lengths):
            rows = self.mixed[self.first[s]:self.first[s] + n, :self.channels].double().T
            before = history[self.slots[s]]
            if self.continues is not None and not self.continues[s]:
                before = torch.zeros_like(before)
            if n == 0:
                continue
            line = torch.cat([before, rows], 1)
            value = torch.nn.functional.silu(sum(line[:, j:j + n] * self.taps[:, j:j + 1].double() for j in range(4))).T
            for part, factor in ((0, DIM ** -0.5), (1, 1.0)):
                at = slice(part * KEY_HEADS * DIM, (part + 1) * KEY_HEADS * DIM)
                x = value[:, at].reshape(n, KEY_HEADS, DIM)
                value[:, at] = (factor * x / torch.sqrt(x.square().sum(-1, keepdim=True) + 1e-6)).reshape(n, -1)
            qkv[self.first[s]:self.first[s] + n] = value
            history[self.slots[s]] = line[:, -3:]
        live = slice(self.first[0], self.first[-1])
        self.run(ops)
        # half a bf16 step, and fp32 sums of four products (of either sign) through __expf: 2^-16 of their magnitudes' mean
        assert ((self.qkv.double() - qkv).abs() <= 2.0 ** -8 * qkv.abs() + 2.0 ** -16 * qkv.abs().mean()).all()
        a = self.mixed[:, self.channels:self.channels + self.heads].double() + self.dt_bias.double()
        b = self.mixed[:, self.channels + self.heads:self.channels + 2 * self.heads].double()
        alpha = torch.exp(-self.a_log.double().exp() * torch.nn.functional.softplus(a, threshold=60.0))
        for got, value in ((self.alpha, alpha), (self.beta, torch.sigmoid(b))):
            exponent = value.clamp_min(1e-45).log().abs()
            assert ((got.double() - value).abs() <= 2.0 ** -20 * (1 + exponent) * value + 1e-37)[live].all()
            assert (got[:live.start] == 7.0).all() and (got[live.stop:] == 7.0).all()
        assert torch.equal(self.history, history.float())


@pytest.mark.parametrize("heads", [32, 48])
@pytest.mark.parametrize("lengths", [[1], [2], [3], [4], [7], [8], [9], [100], [1, 2, 0, 3, 50, 1], [5] * 30])
def test_delta_prepare_chunk(cuda, ops, heads, lengths):
    Prepare(cuda, heads + len(lengths) + lengths[0], lengths, heads).check(ops)


def test_delta_prepare_chunk_begins_and_foreign_rows(cuda, ops):
    Prepare(cuda, 31, [1, 2, 0, 40, 9], 32, continues=[0, 1, 0, 0, 1], first=2, padding=5, extra=4096).check(ops)


def test_delta_prepare_chunk_steep_gates(cuda, ops):
    Prepare(cuda, 32, [30], 32, std=12.0).check(ops)


# ---- copies ---------------------------------------------------------------------------------------

@pytest.mark.parametrize("units,shapes,pairs", [
    (7, [(16,)], [(0, 1)]), (9, [(4096,), (16,), (48,)], [(3, 0), (8, 2), (4, 4)]),
    (64, [(16384 + 16,)] * 5, [(i, 63 - i) for i in range(30)]), (3, [(65536,)] * 130, [(2, 0)])])
def test_cache_copy(cuda, ops, units, shapes, pairs):
    g = generator(cuda, units)
    arrays = [cuda.randint(0, 256, (units,) + shape, dtype=cuda.uint8, device="cuda", generator=g) for shape in shapes]
    want = [a.clone() for a in arrays]
    for a in want:
        for source, target in pairs:
            a[target] = a[source]
    listed = i32(cuda, [x for pair in pairs + [(-1, -1)] for x in pair])
    ops.cache_copy(ops.copy_table(arrays, units), listed, len(pairs) + 1)
    assert all(cuda.equal(a, b) for a, b in zip(arrays, want))


def test_cache_copy_beyond_the_array(cuda, ops):
    from qwencore_b200 import abi
    array = cuda.arange(40, dtype=cuda.float32, device="cuda").reshape(5, 8)
    want = array.clone()
    want[1] = want[3]
    ops.cache_copy(ops.copy_table([array], 5), i32(cuda, [0, 5, 3, 1, 7, 0]), 3)
    assert cuda.equal(array, want)
    assert abi.lib.qwc_device_status() == 0x107
    abi.check(abi.lib.qwc_device_status_reset(), "reset")
    ops.cache_copy(ops.copy_table([array], 5), i32(cuda, [0, 1]), 0)
    assert cuda.equal(array, want)
