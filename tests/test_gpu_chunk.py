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


# ---- as they are used -----------------------------------------------------------------------------

class Layers:
    """A DeltaNet and an attention layer that take a ragged batch of prompts, share a prefix and go on token by token."""

    def __init__(self, torch, ops, seed, lengths, past, heads, page=16):
        from qwencore_b200 import abi
        abi.configure(heads, 64)
        g = generator(torch, seed)
        self.torch, self.ops, self.heads, self.page, self.lengths = torch, ops, heads, page, lengths
        self.sequences = count = len(lengths)
        self.first, self.tokens = begins_of(lengths), sum(lengths)
        self.channels = (2 * KEY_HEADS + heads) * DIM
        self.z = self.channels
        self.a = self.z + heads * DIM
        self.b = self.a + heads
        self.width = self.b + heads + (-(self.b + heads)) % 8
        randn = lambda *shape: torch.randn(shape, device="cuda", generator=g)  # noqa: E731
        # rows of the prompts, and of the next token of every sequence and of a copy of the first
        self.mixed, self.next_mixed = randn(self.tokens, self.width).bfloat16(), randn(count + 1, self.width).bfloat16()
        self.next_mixed[count] = self.next_mixed[0]
        self.taps = (randn(self.channels, 4) * 0.5).bfloat16()
        self.a_log, self.dt_bias = (randn(heads) * 0.5).bfloat16(), (randn(heads) * 0.5).bfloat16()
        self.weight = (1 + 0.1 * randn(DIM)).bfloat16()
        self.slots = list(range(count, 0, -1)) + [0]  # the copy's is the last
        self.capacity = count + 1
        held = randn(self.capacity, heads, DIM, DIM) * 0.1
        peak = held.abs().amax(-1)
        self.codes, self.scales = (held * (127.0 / peak)[..., None]).round().to(torch.int8), peak / 127.0
        self.history = randn(self.capacity, self.channels, 3).bfloat16().float()
        self.continues = [int(p > 0) for p in past]
        # attention: the sequences' pages, with room for a token more, and as many for the copy
        self.contexts = [n + p for n, p in zip(lengths, past)]
        blocks = [c // page + 1 for c in self.contexts]
        self.widest, self.pool = max(blocks), sum(blocks) + blocks[0]
        order = np.random.default_rng(seed).permutation(self.pool)
        table = np.zeros((count + 1, self.widest), dtype=np.int32)
        at = 0
        for row, blocks_of in enumerate(blocks + [blocks[0]]):
            table[row, :blocks_of] = order[at:at + blocks_of]
            at += blocks_of
        self.table = torch.from_numpy(table).cuda()
        self.state_pairs = i32(torch, [self.slots[0], 0])
        self.page_pairs = i32(torch, np.stack([table[0, :blocks[0]], table[count, :blocks[0]]], 1).flatten())
        self.copied = blocks[0]
        self.kv_scale = (0.5 + torch.rand(KV, device="cuda", generator=g)) / 32.0
        self.caches = [(randn(self.pool, KV, page, WIDE) / self.kv_scale[None, :, None, None]).clamp(-448, 448)
                       .to(torch.float8_e4m3fn).view(torch.uint8) for _ in range(2)]
        self.row = 2 * HEADS * WIDE + 2 * KV * WIDE  # [q | gate per head][k][v]
        self.projected, self.next_projected = (randn(n, self.row).bfloat16() for n in (self.tokens, count + 1))
        self.next_projected[count] = self.next_projected[0]
        self.q_weight, self.k_weight = (randn(WIDE) * 0.1).bfloat16(), (randn(WIDE) * 0.1).bfloat16()
        positions = [p + i for n, p in zip(lengths, past) for i in range(n)]
        self.places = self.place(positions, [s for s, n in enumerate(lengths) for _ in range(n)])
        self.next_places = self.place(self.contexts + [self.contexts[0]], list(range(count + 1)))
        # what the calls write
        bf16 = lambda *shape: torch.zeros(shape, dtype=torch.bfloat16, device="cuda")  # noqa: E731
        f32 = lambda *shape: torch.zeros(shape, device="cuda")  # noqa: E731
        self.qkv, self.alpha, self.beta = bf16(self.tokens, self.channels), f32(self.tokens, heads), f32(self.tokens, heads)
        self.out, self.attended, self.query = bf16(self.tokens, heads, DIM), bf16(self.tokens, HEADS, WIDE), bf16(self.tokens, HEADS, WIDE)
        n = count + 1
        self.q, self.k, self.v = f32(n, KEY_HEADS, DIM), f32(n, KEY_HEADS, DIM), f32(n, heads, DIM)
        self.next_alpha, self.next_beta, self.kq = f32(n, heads), f32(n, heads), f32(n, KEY_HEADS)
        self.next_values, self.next_out = f32(n, heads, DIM), bf16(n, heads, DIM)
        self.next_query, self.next_attended = bf16(n, HEADS, WIDE), bf16(n, HEADS, WIDE)
        self.lists = [i32(torch, x) for x in (self.slots, self.continues, self.first, self.contexts,
                                              [c + 1 for c in self.contexts] + [self.contexts[0] + 1])]
        size = lambda n: torch.zeros(max(16, n), dtype=torch.uint8, device="cuda")  # noqa: E731
        self.workspaces = [size(ops.delta_chunk_workspace_bytes(self.tokens, count)), size(ops.attention_chunk_workspace_bytes()),
                           size(ops.packed_workspace_bytes(n, 8))]
        self.tables = [ops.copy_table([self.codes, self.scales, self.history], self.capacity), ops.copy_table(self.caches, self.pool)]
        self.state = [self.codes, self.scales, self.history, *self.caches]
        self.before = [x.clone() for x in self.state]
        self.between = [torch.empty_like(x) for x in self.state]  # behind the prompts and the copies
        self.results = [self.qkv, self.alpha, self.beta, self.out, self.query, self.attended, self.next_values, self.next_out,
                        self.next_query, self.next_attended, *self.state]

    def place(self, positions, rows):
        """cos, sin, page and offset of every row's token."""
        torch = self.torch
        at = torch.tensor(positions, dtype=torch.float64, device="cuda")
        angle = at[:, None] * 10.0 ** (-(torch.arange(64, dtype=torch.float64, device="cuda") % 32) / 8)[None]
        pages = self.table[torch.tensor(rows, device="cuda"), torch.tensor([p // self.page for p in positions], device="cuda")]
        return angle.cos().bfloat16(), angle.sin().bfloat16(), pages.contiguous(), i32(torch, [p % self.page for p in positions])

    def restore(self):
        for held, before in zip(self.state, self.before):
            held.copy_(before)

    def prompts(self):
        ops, (slots, continues, first, contexts, _) = self.ops, self.lists
        ops.delta_prepare_chunk(self.mixed, self.a, self.b, self.taps, self.a_log, self.dt_bias, self.history, slots, continues,
                                first, self.qkv, self.alpha, self.beta, self.capacity, self.tokens, self.sequences, self.width)
        ops.delta_chunk(self.codes, self.scales, slots, continues, first, self.qkv, self.alpha, self.beta, self.out, self.capacity,
                        self.tokens, self.sequences, self.workspaces[0], gate=self.mixed, gate_offset=self.z,
                        gate_stride=self.width, norm_weight=self.weight, epsilon=EPS)
        self.attention_rows(self.projected, self.places, self.query, self.tokens)
        ops.paged_attention_chunk(self.query, self.projected, *self.caches, self.table, contexts, first, self.widest,
                                  self.attended, self.tokens, self.sequences, self.workspaces[1], self.page, self.pool,
                                  key_scales=self.kv_scale, value_scales=self.kv_scale, gate_stride=self.row)
        ops.cache_copy(self.tables[0], self.state_pairs, 1)
        ops.cache_copy(self.tables[1], self.page_pairs, self.copied)

    def attention_rows(self, projected, places, query, rows):
        k, v = projected[0, 2 * HEADS * WIDE:], projected[0, (2 * HEADS + KV) * WIDE:]
        self.ops.prepare_attention_decode(projected, k, v, self.q_weight, self.k_weight, *places, query, *self.caches, rows,
                                          self.page, self.row, self.row, self.row, self.kv_scale, self.kv_scale)

    def next_token(self):
        ops, (slots, _, _, _, contexts), n = self.ops, self.lists, self.sequences + 1
        ops.delta_prepare_decode(self.next_mixed, self.a, self.b, self.taps, self.a_log, self.dt_bias, self.history, slots, self.q,
                                 self.k, self.v, self.next_alpha, self.next_beta, self.kq, self.capacity, n, self.width)
        ops.delta_decode_slots_packed(self.codes, self.scales, slots, self.q, self.k, self.v, self.next_alpha, self.next_beta,
                                      self.kq, self.next_values, self.capacity, n)
        ops.delta_gated_rmsnorm(self.next_values, self.next_mixed, self.z, self.weight, self.next_out, n, self.width)
        self.attention_rows(self.next_projected, self.next_places, self.next_query, n)
        ops.gated_packed(self.next_query, self.next_projected, *self.caches, self.table, contexts, self.widest,
                         self.next_attended, n, 0, 8, self.workspaces[2], self.page, self.kv_scale, self.kv_scale, self.row)

    def run(self):
        self.prompts()
        for held, state in zip(self.between, self.state):
            held.copy_(state)
        self.next_token()


def layers_as_cases(torch, layers):
    """The chunk operators' cases on what the layers' calls have read and written."""
    delta = Delta(torch, 0, layers.lengths, layers.heads, continues=layers.continues, normed=True, gate_offset=layers.z)
    delta.slots, delta.capacity = layers.slots[:-1], layers.capacity
    delta.qkv, delta.alpha, delta.beta = layers.qkv, layers.alpha, layers.beta
    delta.codes, delta.scales = layers.before[0].clone(), layers.before[1].clone()
    delta.gate, delta.gate_stride, delta.weight = layers.mixed[:, :layers.a].contiguous(), 0, layers.weight
    delta.gate_stride = layers.a
    attention = Attention(torch, 0, layers.lengths, [c - n for c, n in zip(layers.contexts, layers.lengths)], layers.page)
    attention.table, attention.widest, attention.pool = layers.table[:-1].contiguous(), layers.widest, layers.pool
    attention.query, attention.gate, attention.gate_stride = layers.query, layers.projected, layers.row
    attention.caches, attention.scale = layers.between[3:], layers.kv_scale
    return delta, attention


@pytest.mark.parametrize("heads,page,lengths,past", [(32, 16, [70, 1, 33], [0, 40, 95]), (48, 64, [130, 64], [0, 0]),
                                                    (32, 64, [5], [1000])])
def test_prompts_a_shared_prefix_and_the_next_token(cuda, ops, heads, page, lengths, past):
    torch = cuda
    layers = Layers(torch, ops, 41, lengths, past, heads, page)
    layers.run()
    count = layers.sequences
    # the chunk operators, on what they were given (the same calls again: the same bits), against their plain forms
    delta, attention = layers_as_cases(torch, layers)
    delta.check(ops)
    attention.check(ops)
    assert torch.equal(delta.out, layers.out) and torch.equal(attention.output, layers.attended)
    for s in range(count):
        assert torch.equal(delta.codes[layers.slots[s]], layers.between[0][layers.slots[s]])
    # the decode step begins where the chunk ended: the convolution's history ...
    for s in range(count):
        rows = layers.mixed[layers.first[s]:layers.first[s + 1], :layers.channels].float().T
        before = layers.before[2][layers.slots[s]] * layers.continues[s]
        assert torch.equal(layers.between[2][layers.slots[s]], torch.cat([before, rows], 1)[:, -3:])
    # ... the state (fp32 sums of 128 products of either sign: 2^-17 of their magnitudes) ...
    held = layers.between[0].double() * layers.between[1].double()[..., None]
    state = held[layers.slots]
    ratio = heads // KEY_HEADS
    q, k = (x.double().repeat_interleave(ratio, 1) for x in (layers.q, layers.k))
    state = state * layers.next_alpha.double()[..., None, None]
    u = (layers.v.double() - torch.einsum("shij,shj->shi", state, k)) * layers.next_beta.double()[..., None]
    want = torch.einsum("shij,shj->shi", state, q) + u * (k * q).sum(-1, keepdim=True)
    terms = torch.einsum("shij,shj->shi", state.abs(), q.abs() + k.abs()) + layers.v.abs().double()
    assert ((layers.next_values.double() - want).abs() <= 2.0 ** -17 * terms + 1e-6 * want.abs().amax()).all()
    # ... and the cache
    tail = Attention(torch, 0, [1] * (count + 1), layers.contexts + [layers.contexts[0]], page)
    tail.table, tail.widest, tail.pool = layers.table, layers.widest, layers.pool
    tail.query, tail.gate, tail.gate_stride = layers.next_query, layers.next_projected, layers.row
    tail.caches, tail.scale = layers.caches, layers.kv_scale
    tail.check(ops)
    want, spread = tail.want()
    # (the decode attention's own rounding: see its tests)
    assert ((layers.next_attended.double() - want).abs() <= 2.0 ** -7 * want.abs() + 2.0 ** -6 * spread).all()
    # the copy of the first sequence says what that one says (the decode attention cuts rows where its shares end, so that
    # row is above, within its rounding)
    for x in (layers.next_values, layers.next_out, layers.next_query):
        assert torch.equal(x[0], x[count])
    for x in layers.state[:3]:
        assert torch.equal(x[layers.slots[0]], x[0])


def test_captured_and_replayed(cuda, ops):
    torch = cuda
    layers = Layers(torch, ops, 42, [100, 1, 60], [0, 500, 30], 32)
    layers.run()
    want = [x.clone() for x in layers.results]
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    layers.restore()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        layers.run()
    for _ in range(3):
        layers.restore()
        for x in layers.results[:-5]:
            x.fill_(3.0)
        graph.replay()
        assert all(torch.equal(x, y) for x, y in zip(layers.results, want))


def test_two_at_once_on_streams_of_their_own(cuda, ops):
    torch = cuda
    both = [Layers(torch, ops, 43, [300, 1, 60], [0, 900, 30], 48), Layers(torch, ops, 44, [65, 129], [3000, 0], 48)]
    wants = []
    for layers in both:
        layers.run()
        wants.append([x.clone() for x in layers.results])
    streams = [torch.cuda.Stream() for _ in both]
    torch.cuda.synchronize()
    for _ in range(5):
        for layers in both:
            layers.restore()
        for stream in streams:
            stream.wait_stream(torch.cuda.current_stream())
        for layers, stream in zip(both, streams):
            with torch.cuda.stream(stream):
                layers.run()
        torch.cuda.synchronize()
        for layers, want in zip(both, wants):
            assert all(torch.equal(x, y) for x, y in zip(layers.results, want))


# ---- ranges ---------------------------------------------------------------------------------------

def off_by_16(torch, tensor):
    """The same numbers at an address that is a multiple of 16 and not of 32."""
    room = torch.empty(tensor.numel() + 32, dtype=tensor.dtype, device="cuda")
    skip = 16 // tensor.element_size()
    if room.data_ptr() % 32:
        skip = 0
    moved = room[skip:skip + tensor.numel()].view(tensor.shape)
    moved.copy_(tensor)
    assert moved.data_ptr() % 32 == 16
    return moved


@pytest.mark.parametrize("part", ["query", "gate", "output", "workspace"])
def test_attention_chunk_rows_at_16_byte_boundaries(cuda, ops, part):
    case = Attention(cuda, 51, [100, 1, 30], [2000, 40, 0], 16, gate_stride=HEADS * 2 * WIDE + (8 if part == "gate" else 0))
    workspace = cuda.zeros(ops.attention_chunk_workspace_bytes(), dtype=cuda.uint8, device="cuda")
    if part == "workspace":
        workspace = off_by_16(cuda, workspace)
    else:
        setattr(case, part, off_by_16(cuda, getattr(case, part)))
    case.check(ops, workspace=workspace)


def test_delta_chunk_rows_at_16_byte_boundaries(cuda, ops):
    case = Delta(cuda, 52, [100, 1, 30], 32, normed=True, gate_offset=8)
    for name in ("qkv", "gate", "out", "codes", "weight"):
        setattr(case, name, off_by_16(cuda, getattr(case, name)))
    case.check(ops, workspace=off_by_16(cuda, cuda.zeros(ops.delta_chunk_workspace_bytes(131, 3), dtype=cuda.uint8, device="cuda")))


def test_128_sequences(cuda, ops):
    lengths = [(7 * i) % 13 for i in range(128)]
    Attention(cuda, 53, lengths, [(31 * i) % 200 for i in range(128)], 16).check(ops)
    Delta(cuda, 54, lengths, 32, continues=[i % 3 % 2 for i in range(128)], normed=True).check(ops)
    Prepare(cuda, 55, lengths, 32, continues=[i % 3 % 2 for i in range(128)]).check(ops)


def test_attention_chunk_pages_beyond_four_gigabytes(cuda, ops):
    torch = cuda
    case = Attention(cuda, 56, [50, 3], [300, 700], 16)
    small, pool = case.caches, 266000  # pages of 16 KiB
    first = pool - case.pool
    assert first * KV * 16 * WIDE > 1 << 32
    big = [torch.full((pool, KV, 16, WIDE), 0x7f, dtype=torch.uint8, device="cuda") for _ in range(2)]
    want, spread = case.want()
    for to, rows in zip(big, small):
        to[first:] = rows
    case.table[case.table < case.pool] += first
    case.caches, case.pool = big, pool
    got = case.run(ops).double()
    assert ((got - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -10 * spread).all()


def test_cache_copy_beyond_four_gigabytes(cuda, ops):
    torch = cuda
    array = torch.zeros((70000, 65536), dtype=torch.uint8, device="cuda")
    array[3] = torch.arange(65536, device="cuda") % 251
    ops.cache_copy(ops.copy_table([array], 70000), i32(torch, [3, 69999]), 1)
    assert torch.equal(array[69999], array[3]) and not array[69998].any()


def test_longest_chunk(cuda, ops):
    """65536 tokens: rows of the beginning, and of the end, where nothing of the beginning is left."""
    torch, n, warm, rows = cuda, 65536, 400, 100
    case = Delta(cuda, 57, [n], 32, rate=(0.8, 2.0))  # (alpha^400 is below e^-150)
    case.run(ops)
    start = Delta(cuda, 57, [rows], 32)
    start.qkv, start.alpha, start.beta = (x[:rows].contiguous() for x in (case.qkv, case.alpha, case.beta))
    fresh = Delta(cuda, 57, [n], 32, rate=(0.8, 2.0))
    start.slots, start.codes, start.scales = fresh.slots, fresh.codes, fresh.scales
    want, largest, _ = start.want()
    assert ((case.out[:rows].double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -10 * largest).all()
    end = Delta(cuda, 57, [warm + rows], 32, continues=[0])
    end.qkv, end.alpha, end.beta = (x[-warm - rows:].contiguous() for x in (case.qkv, case.alpha, case.beta))
    want, largest, _ = end.want()
    got = case.out[-rows:].double()
    assert ((got - want[-rows:]).abs() <= 2.0 ** -8 * want[-rows:].abs() + 2.0 ** -10 * largest[-rows:]).all()
    attention = Attention(cuda, 58, [n], [0], 64, gated=False)
    got = attention.run(ops)
    picked = torch.tensor([0, 1, 41, 42, 127, 128, 4095, 32767, 50000, 65535], device="cuda")
    k, v = (c[attention.table[0].long()].view(torch.float8_e4m3fn).double().transpose(0, 1).reshape(KV, -1, WIDE) *
            attention.scale.double()[:, None, None] for c in attention.caches)
    for row in picked.tolist():
        q = attention.query[row].double().reshape(KV, GROUP, WIDE)
        weights = torch.softmax(q @ k[:, :row + 1].transpose(1, 2) / 16.0, -1)
        want, spread = ((weights @ x[:, :row + 1]).reshape(HEADS, WIDE) for x in (v, v.abs()))
        assert ((got[row].double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -10 * spread).all(), row


def test_delta_chunk_a_gate_that_is_no_number(cuda, ops):
    # it reaches its head's rows from there on, and nothing else
    case = Delta(cuda, 59, [100, 30], 32)
    want, largest, _ = case.want()
    case.alpha[40, 5] = float("nan")
    case.run(ops)
    got = case.out.double()
    reached = cuda.zeros((130, 32), dtype=cuda.bool, device="cuda")
    reached[64:100, 5] = True   # (of the block that holds it, rows in front may be reached too)
    inside = cuda.zeros_like(reached)
    inside[:64, 5] = True
    close = ((got - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -10 * largest).all(-1)
    assert close[~(reached | inside)].all() and got[64:100, 5].isnan().all() and got[40:64, 5].isnan().all()


def test_chunks_that_overlap_or_run_backwards_stay_in_bounds(cuda, ops):
    """Not what the calls are for: no row of theirs has a meaning, but nothing else is touched and the next call is right."""
    torch = cuda
    for begins in ([0, 100, 0, 100, 0, 100, 0, 100], [100, 0, 90, 10, 80, 20, 70, 30], [2 ** 31 - 1, 0, 100, 100, 50, 2 ** 31 - 1, 3, 4]):
        delta = Delta(torch, 61, [100] + [0] * 6, 32, normed=True, padding=3)
        delta.first = begins
        delta.run(ops)
        assert (delta.out[100:] == 7.0).all() or max(begins) > 103
        idle = [s for s in range(delta.capacity) if s not in delta.slots]
        fresh = Delta(torch, 61, [100] + [0] * 6, 32, normed=True, padding=3)
        assert all(torch.equal(delta.codes[s], fresh.codes[s]) for s in idle)
        attention = Attention(torch, 62, [100] + [0] * 6, [30] * 7, padding=3)
        attention.first = begins
        attention.run(ops)
        prepared = Prepare(torch, 63, [100] + [0] * 6, 32, padding=3)
        prepared.first = begins
        prepared.run(ops)
        torch.cuda.synchronize()
    Delta(torch, 64, [100, 70], 32, normed=True).check(ops)
    Attention(torch, 65, [100, 70], [30, 0]).check(ops)
    Prepare(torch, 66, [100, 70], 32).check(ops)


def test_attention_chunk_value_codes_that_are_no_number(cuda, ops):
    # seen by every row: 480 times the scale, of either sign
    case = Attention(cuda, 67, [20], [100], gated=False)
    page = case.table[0, 1].long()
    case.caches[1][page, 2, 5, 40:44] = cuda.tensor([0x7f, 0xff, 0x7e, 0xfe], dtype=cuda.uint8, device="cuda")
    got = case.run(ops).double()[:, 12:18, 40:44]
    ids = case.table[0, :8].long()
    k, v = (c[ids].view(cuda.float8_e4m3fn).double().transpose(0, 1).reshape(KV, -1, WIDE)[2, :120] * case.scale[2].double()
            for c in case.caches)
    v = v[:, 40:44].nan_to_num(0.0)
    v[21, :2] = cuda.tensor([480.0, -480.0], dtype=cuda.float64, device="cuda") * case.scale[2].double()
    scores = case.query[:, 12:18].double().transpose(0, 1) @ k.T / 16.0
    scores = scores.masked_fill(cuda.arange(120, device="cuda")[None] > (cuda.arange(20, device="cuda") + 100)[:, None], -cuda.inf)
    weights = cuda.softmax(scores, -1)
    want, spread = (weights @ v).transpose(0, 1), (weights @ v.abs()).transpose(0, 1)
    assert ((got - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -10 * spread).all()


@pytest.mark.parametrize("heads", [32, 48])
def test_delta_chunk_more_jobs_than_sms_and_slots_beyond_the_pool(cuda, ops, heads):
    """Every CTA takes several (chunk, value head) pairs, some of which are left out."""
    from qwencore_b200 import abi
    lengths = [5, 200, 0, 64, 130, 1, 70, 65, 128, 3, 17, 90, 33, 64]
    case = Delta(cuda, 71 + heads, lengths, heads, normed=True, continues=[i % 3 != 0 for i in range(len(lengths))])
    whole = Delta(cuda, 71 + heads, lengths, heads, normed=True, continues=[i % 3 != 0 for i in range(len(lengths))])
    whole.check(ops)
    lost = [1, 5, 8]  # the longest among them
    before = case.codes.clone(), case.scales.clone()
    kept = [s for s in range(len(lengths)) if s not in lost]
    good = list(case.slots)
    for s in lost:
        case.slots[s] = case.capacity + s
    case.run(ops)
    assert abi.lib.qwc_device_status() == 0x105
    abi.check(abi.lib.qwc_device_status_reset(), "reset")
    for s, n in enumerate(lengths):
        rows = slice(case.first[s], case.first[s] + n)
        if s in kept:
            assert cuda.equal(case.out[rows], whole.out[rows])
            assert cuda.equal(case.codes[good[s]], whole.codes[good[s]]) and cuda.equal(case.scales[good[s]], whole.scales[good[s]])
        else:
            assert (case.out[rows] == 7.0).all()
            assert cuda.equal(case.codes[good[s]], before[0][good[s]]) and cuda.equal(case.scales[good[s]], before[1][good[s]])


@pytest.mark.parametrize("lead", [9.0, 14.0, 18.0])
@pytest.mark.parametrize("tokens,past,at", [(40, 8000, 0), (40, 8000, 8000), (3, 200, 0), (1000, 0, 0)])
def test_attention_chunk_small_weights_decide(cuda, ops, tokens, past, at, lead):
    """A token that draws nearly all of the weight and has no value: the result is what thousands of small weights say.

    Probabilities are off by 2^-36 of the largest, partial results by 2^-32 of the value scale (which is 1 here)."""
    torch = cuda
    case = Attention(torch, 81, [tokens], [past], 16, gated=False, scaled=False, query_std=0.5)
    keys, values = case.caches
    keys[..., 0] = 0
    case.query[..., 0] = 16.0
    values[:] = (values.view(torch.float8_e4m3fn).float().abs() + 0.5).to(torch.float8_e4m3fn).view(torch.uint8)
    page = case.table[0, at // 16].long()
    keys[page, :, at % 16] = 0
    keys[page, :, at % 16, 0] = torch.tensor([lead], device="cuda").to(torch.float8_e4m3fn).view(torch.uint8)
    values[page, :, at % 16] = 0
    got = case.run(ops).double()
    want, spread = case.want()
    largest = float(values[case.table[0].long()].view(torch.float8_e4m3fn).float().max())
    bound = 2.0 ** -8 * want.abs() + 2.0 ** -10 * spread + 2.0 ** -36 * (tokens + past) * largest + 2.0 ** -32
    assert ((got - want).abs() <= bound).all(), float(((got - want).abs() / bound).max())


@pytest.mark.parametrize("code", [0x103, 0x108, 0x109])
def test_a_wait_that_gave_up_stops_the_operators_on_chunks(cuda, ops, code):
    """Attention and delta rule leave everything as it was, and are right again behind a reset."""
    from qwencore_b200 import abi
    attention = Attention(cuda, 82, [100, 1, 30], [2000, 40, 0], 16)
    delta = Delta(cuda, 83, [100, 1, 30], 32, normed=True)
    codes, scales = delta.codes.clone(), delta.scales.clone()
    abi.check(abi.lib.qwc_device_status_set(code), "set")
    try:
        attention.run(ops)
        delta.run(ops)
        assert abi.lib.qwc_device_status() == code
    finally:
        abi.check(abi.lib.qwc_device_status_reset(), "reset")
    assert (attention.output == 7.0).all() and (delta.out == 7.0).all()
    assert cuda.equal(delta.codes, codes) and cuda.equal(delta.scales, scales)
    attention.check(ops, workspace=attention.workspace)
    delta.check(ops)


@pytest.mark.parametrize("code", [0x105, 0x107])
def test_ids_out_of_range_do_not_stop_the_operators_on_chunks(cuda, ops, code):
    from qwencore_b200 import abi
    attention = Attention(cuda, 84, [100, 1, 30], [2000, 40, 0], 16)
    delta = Delta(cuda, 85, [100, 1, 30], 32)
    abi.check(abi.lib.qwc_device_status_set(code), "set")
    try:
        attention.check(ops)
        delta.check(ops)
        assert abi.lib.qwc_device_status() == code
    finally:
        abi.check(abi.lib.qwc_device_status_reset(), "reset")


def test_delta_prepare_chunk_behind_a_write_of_its_weights(cuda, ops):
    """The kernel in front lets this one start early and writes the taps at its end."""
    from qwencore_b200 import abi
    torch = cuda
    case = Prepare(torch, 86, [9, 100], 32)
    taps = case.taps
    big = torch.zeros((2, 1 << 28), dtype=torch.uint8, device="cuda")
    held = torch.zeros((2,) + tuple(taps.shape), dtype=torch.bfloat16, device="cuda")
    held[0] = taps
    case.taps = held[1]
    table, pairs = ops.copy_table([big, held], 2), i32(torch, [0, 1])
    slots, begins, history = i32(torch, case.slots), i32(torch, case.first), case.history.clone()
    qkv = torch.zeros_like(case.qkv)
    abi.configure(case.heads, 64)
    torch.cuda.synchronize()
    ops.cache_copy(table, pairs, 1)
    ops.delta_prepare_chunk(case.mixed, case.channels, case.channels + case.heads, case.taps, case.a_log, case.dt_bias,
                            case.history, slots, None, begins, qkv, case.alpha, case.beta, case.capacity, case.tokens, 2,
                            case.width)
    case.history.copy_(history)
    case.check(ops)
    assert torch.equal(qkv, case.qkv)


@pytest.mark.parametrize("std", [1e-3, 30.0, 3000.0])
def test_attention_chunk_scores_as_steep_as_they_are(cuda, ops, std):
    """A score s_j is a sum of 256 products in fp32, 16 steps of the tensor cores: each cuts off less than 2^-23 of what it has
    summed up, twice that with the alignment of its products, so s_j is off by d_j <= 2^-18 sum |q||k_j| / 16.  To first
    order that moves the result by sum_j w_j (d_j - mean) (v_j - o), 2 max d sum_j w_j |v_j - o| at most: nothing where
    one weight is 1.  (e^(2 d) - 1 in place of 2 d for those that are large.)  And where a weight is 1 and its value 0, what
    is left of the others: a probability is an f16 whose row's largest is 2^11 or more, off by half of its smallest step of 2^-24, so
    a weight is off by 2^-36; a partial result is an f16 of 2^7 times the value over its scale, off by 2^-32 scales."""
    torch = cuda
    case = Attention(torch, 87, [70, 3], [500, 900], 16, query_std=std)
    got = case.run(ops).double()
    want, spread = case.want()
    winners = 0
    for s, n in enumerate(case.lengths):
        context = case.contexts[s]
        ids = case.table[s, :-(-context // case.page)].long()
        k, v = (c[ids].view(torch.float8_e4m3fn).double().transpose(0, 1).reshape(KV, -1, WIDE)[:, :context].repeat_interleave(GROUP, 0) *
                case.scale.double().repeat_interleave(GROUP)[:, None, None] for c in case.caches)
        for i in range(n):
            row, seen = case.first[s] + i, context - n + i + 1
            q = case.query[row].double()[:, None]
            weights = torch.softmax(q @ k[:, :seen].transpose(1, 2) / 16.0, -1)
            off = 2.0 ** -18 * (q.abs() @ k[:, :seen].abs().transpose(1, 2)).amax((1, 2)) / 16.0
            result = (weights @ v[:, :seen])[:, 0]
            around = (weights.transpose(1, 2) * (v[:, :seen] - result[:, None]).abs()).sum(1)
            gate = torch.sigmoid(case.gate[row].double().reshape(HEADS, 2 * WIDE)[:, WIDE:])
            bound = 2.0 ** -8 * want[row].abs() + 2.0 ** -10 * spread[row] + torch.expm1(2 * off)[:, None] * around * gate
            bound += 2.0 ** -36 * seen * v[:, :seen].abs().amax(1) + 2.0 ** -32 * case.scale.repeat_interleave(GROUP)[:, None]
            assert ((got[row] - want[row]).abs() <= bound).all(), (row, float(((got[row] - want[row]).abs() / bound).max()))
            winners += int((weights.amax(-1) > 0.9999).sum())
    assert winners > 1000 or std < 1000.0


@pytest.mark.parametrize("lengths,past", [([100, 3], [0, 40]), ([20], [3000])])
def test_attention_chunk_scales_of_keys_and_values(cuda, ops, lengths, past):
    """Different ones, in items of one piece and in items that are cut."""
    torch = cuda
    case = Attention(torch, 88, lengths, past, 16)
    ratio = torch.tensor([0.5, 3.0, 8.0, 0.125], device="cuda")
    workspace = torch.zeros(ops.attention_chunk_workspace_bytes(), dtype=torch.uint8, device="cuda")
    ops.paged_attention_chunk(case.query, case.gate, *case.caches, case.table, i32(torch, case.contexts), i32(torch, case.first),
                              case.widest, case.output, case.tokens, len(lengths), workspace, case.page, case.pool,
                              key_scales=case.scale, value_scales=case.scale * ratio)
    want, spread = (x * ratio.double().repeat_interleave(GROUP)[None, :, None] for x in case.want())
    assert ((case.output.double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -10 * spread).all()


@pytest.mark.parametrize("heads", [32, 48])
def test_delta_chunk_norm_of_exact_results(cuda, ops, heads):
    """Keys that are unit vectors, one for each token, and no decay: o_t = v_t / 8 without any rounding, so what is off is the
    norm's: fp32 sums of 128 squares, a root, two products and a sigmoid (2^-19 together) and half a bf16 step."""
    torch = cuda
    lengths = [100, 1, 64, 128, 30]
    case = Delta(torch, 89, lengths, heads, continues=[0] * 5, normed=True)
    place = torch.cat([torch.arange(n, device="cuda") for n in lengths])
    keys = torch.nn.functional.one_hot(place, DIM).bfloat16()[:, None].expand(-1, KEY_HEADS, -1).reshape(case.tokens, -1)
    case.qkv[:, :KEY_HEADS * DIM] = keys / 8
    case.qkv[:, KEY_HEADS * DIM:2 * KEY_HEADS * DIM] = keys
    case.alpha.fill_(1.0)
    case.beta.fill_(1.0)
    case.run(ops)
    o = case.qkv[:, 2 * KEY_HEADS * DIM:].double().reshape(case.tokens, heads, DIM) / 8
    gate = case.gate.double().reshape(case.tokens, heads, DIM)
    want = o / torch.sqrt(o.square().mean(-1, keepdim=True) + EPS) * case.weight.double() * torch.nn.functional.silu(gate)
    assert ((case.out.double() - want).abs() <= (2.0 ** -8 + 2.0 ** -19) * want.abs()).all()


@pytest.mark.parametrize("tokens,strength", [(2048, 1.0), (8192, 1.0), (8192, 0.02)])
def test_delta_chunk_states_that_last(cuda, ops, tokens, strength):
    """Hardly any decay over 32 and 128 blocks; with weak writes the state keeps what thousands of tokens have put there."""
    case = Delta(cuda, 90, [tokens, 65], 32, rate=(1e-6, 1e-3))
    case.beta *= strength
    case.check(ops)
