"""Token sampling on the GPU against the definition in 64 bits: the tokens are equal."""
import itertools
import math

import pytest
import torch

import solvedelta_b200 as sd
from tests import serving_reference as ref

pytestmark = pytest.mark.gpu


def _logits(rows, vocab, seed, dtype=torch.bfloat16, spread=2.5):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = spread * torch.randn(rows, vocab, generator=gen, device="cuda")
    x.scatter_add_(1, torch.randint(0, vocab, (rows, 6), generator=gen, device="cuda"), 6 * torch.rand(rows, 6, generator=gen, device="cuda"))
    return x.to(dtype), torch.rand(rows, generator=gen, device="cuda")


def _same(logits, u, **settings):
    got = sd.sample_tokens(logits, u, **settings)
    assert got.dtype == torch.long and got.shape == (logits.shape[0],)
    assert got.tolist() == ref.tokens(logits, u, **{k: v for k, v in settings.items() if k != "empty_token"})


@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float32))
@pytest.mark.parametrize("rows,vocab", ((1, 1), (3, 2), (5, 7), (4, 97), (2, 1000), (3, 4099), (1, 32000), (20, 32000), (2, 50021), (40, 8200),
                                        (200, 777), (1, 262144), (2, 131071)))
def test_every_rule_at_every_size(rows, vocab, dtype):
    logits, u = _logits(rows, vocab, rows + vocab, dtype)
    rules = itertools.product((0.7, 1.3), (0, 1, 5, 60, vocab), (1.0, 0.9, 0.3), (0.0, 0.05))
    for n, (temperature, top_k, top_p, min_p) in enumerate(rules):
        if rows * vocab > 60000 and n % 7:
            continue
        _same(logits, u, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)


@pytest.mark.parametrize("dtype,rows,vocab", ((torch.float32, 300, 26001), (torch.bfloat16, 310, 60003), (torch.float32, 160, 90000)))
def test_rows_too_long_for_shared_memory(dtype, rows, vocab):
    """Many rows of a large vocabulary: few candidates, some thousands, and nearly all of them stay."""
    logits, u = _logits(rows, vocab, 11, dtype)
    logits[::7, ::3] = -math.inf
    logits[5] = -math.inf
    logits[6, 100:] = math.nan
    logits[9, 5], logits[9, vocab - 1] = math.inf, math.inf
    logits[12] = 0.25
    for settings in (dict(), dict(top_k=40, top_p=0.9), dict(top_k=3000), dict(top_k=vocab - 100, top_p=0.97), dict(top_p=0.9), dict(top_p=0.999, temperature=1.5),
                     dict(min_p=0.05), dict(min_p=1e-4, top_p=0.99), dict(temperature=0.0), dict(top_p=0.3, temperature=30.0)):
        _same(logits, u, **settings)


@pytest.mark.parametrize("dtype,rows,vocab", ((torch.float32, 30, 30000), (torch.bfloat16, 140, 30000), (torch.float32, 400, 20000),
                                              (torch.float32, 300, 40000), (torch.bfloat16, 200, 60000), (torch.float32, 2, 262144)))
def test_borders_among_thousands_of_candidates(dtype, rows, vocab):
    """More candidates than the first CTA lists, borders of both rules: the definition's tokens, and the same ones every time."""
    logits, u = _logits(rows, vocab, 21, dtype)
    for settings in (dict(top_k=600), dict(top_k=2000, temperature=1.4), dict(top_k=5000, top_p=0.97), dict(top_p=0.95, temperature=0.7),
                     dict(top_p=0.99, temperature=2.0), dict(top_k=4000, min_p=1e-3)):
        _same(logits, u, **settings)
        first = sd.sample_tokens(logits, u, **settings)
        for _ in range(12):
            assert torch.equal(sd.sample_tokens(logits, u, **settings), first)


@pytest.mark.parametrize("dtype,rows,vocab", ((torch.float32, 3, 262143), (torch.bfloat16, 160, 120007)))
def test_more_stay_than_shared_memory_takes(dtype, rows, vocab):
    """Flat rows that are read again: most of them stay; a border's step of some hundred entries, of thousands, of equal ones,
    under masks."""
    logits, u = _logits(rows, vocab, 31, dtype, 0.6)
    few_values = (logits.float() * 4).round().to(dtype) / 4   # thousands of ties on the border
    masked = logits.clone()
    masked[:, 1000::5] = -math.inf
    masked[:, ::1001] = math.nan
    uneven = logits.clone()
    uneven[:, : vocab // 2] += 3.0   # one half is in front of the border, the other spreads over it
    for x in (logits, few_values, masked, uneven):
        for settings in (dict(top_p=0.9), dict(top_p=0.6, temperature=0.3), dict(top_p=0.95, min_p=1e-3), dict(top_k=90001),
                         dict(top_k=100000, top_p=0.97)):
            first = sd.sample_tokens(x, u, **settings)
            assert first[::53].tolist() == ref.tokens(x[::53], u[::53], **settings)
            for _ in range(3):
                assert torch.equal(sd.sample_tokens(x, u, **settings), first)


def test_a_number_and_a_tensor_of_it_draw_the_same():
    logits, u = _logits(50, 9000, 4)
    for name, value in (("temperature", 0.7), ("top_p", 0.95), ("min_p", 0.01), ("top_k", 700)):
        full = torch.full((50,), value, device="cuda", dtype=torch.int32 if name == "top_k" else torch.float32)
        assert torch.equal(sd.sample_tokens(logits, u, **{name: value}), sd.sample_tokens(logits, u, **{name: full}))


def test_settings_of_each_row():
    logits, u = _logits(64, 3000, 3)
    gen = torch.Generator().manual_seed(1)

    def pick(values, dtype):
        return torch.tensor(values, dtype=dtype)[torch.randint(0, len(values), (64,), generator=gen)].cuda()

    settings = dict(temperature=pick([0.0, 0.5, 1.0, 2.0], torch.float32), top_k=pick([0, 1, 3, 40, 5000], torch.int32),
                    top_p=pick([1.0, 0.9, 0.5, 0.01], torch.float32), min_p=pick([0.0, 0.1, 1.0], torch.float32))
    _same(logits, u, **settings)
    _same(logits, u, **dict(settings, top_k=settings["top_k"].long(), top_p=0.8))
    _same(logits, u, **dict(settings, temperature=settings["temperature"].double()))
    odd = dict(temperature=torch.full((64,), -1.0), top_k=torch.full((64,), -4, dtype=torch.int64), top_p=torch.full((64,), 1.5),
               min_p=torch.full((64,), -0.5))
    odd = {k: v.cuda() for k, v in odd.items()}
    assert sd.sample_tokens(logits, u, **odd).tolist() == ref.tokens(logits, u, temperature=0.0)
    odd["temperature"] = torch.ones(64, device="cuda")
    assert sd.sample_tokens(logits, u, **odd).tolist() == ref.tokens(logits, u)


def test_equal_logits_go_by_index():
    """Ties on the border of top-k and top-p: the lowest indices stay; with a uniform row every token is drawn in turn."""
    for dtype, vocab in itertools.product((torch.bfloat16, torch.float32), (4, 64, 4096, 40000)):
        logits = torch.full((8, vocab), 1.5, dtype=dtype, device="cuda")
        logits[:, vocab // 2] = 1.75
        u = torch.tensor([0.0, 0.1, 0.25, 0.5, 0.625, 0.75, 0.9, 1 - 2 ** -24], device="cuda")
        for top_k, top_p in ((0, 1.0), (3, 1.0), (vocab // 2 + 1, 1.0), (0, 0.5), (3, 0.7), (vocab - 1, 0.99)):
            _same(logits, u, top_k=top_k, top_p=top_p)
    flat = torch.zeros(16, 16, device="cuda")
    u = (torch.arange(16, device="cuda") / 16).float()
    assert sd.sample_tokens(flat, u).tolist() == list(range(16))
    # half of the weight, exactly: what has half of it before it goes
    assert sd.sample_tokens(flat[:3], torch.tensor([0.0, 0.5, 0.999], device="cuda"), top_p=0.5).tolist() == [0, 4, 7]
    assert sd.sample_tokens(flat[:2], torch.tensor([0.5, 0.999], device="cuda"), top_k=2).tolist() == [1, 1]


def test_both_zeros_are_equal():
    for dtype, vocab in itertools.product((torch.bfloat16, torch.float32), (40, 3000, 30000)):
        logits = torch.zeros(8, vocab, dtype=dtype, device="cuda")
        logits[:, ::2] = -0.0
        logits[:, -1] = 1.0
        u = torch.tensor([0.0, 0.1, 0.25, 0.5, 0.625, 0.75, 0.9, 0.99], device="cuda")
        for settings in (dict(), dict(top_k=3), dict(top_k=11), dict(top_k=vocab // 2), dict(top_p=0.3), dict(top_p=0.5, top_k=vocab - 3), dict(temperature=0.0)):
            _same(logits, u, **settings)


def test_borders_of_the_uniform_number():
    logits, _ = _logits(6, 5000, 8)
    u = torch.tensor([0.0, 2.0 ** -24, 1 - 2.0 ** -24, 0.5, 1e-30, 0.999], device="cuda")
    _same(logits, u)
    _same(logits, u, top_k=10)
    # out of range: clamped; a NaN counts as zero
    got = sd.sample_tokens(logits[:3], torch.tensor([-1.0, 2.0, float("nan")], device="cuda"))
    assert got.tolist() == [ref.token(ref.as64(logits)[0], 0.0), ref.token(ref.as64(logits)[1], 1 - 2.0 ** -53), ref.token(ref.as64(logits)[2], 0.0)]


@pytest.mark.parametrize("vocab", (50, 5000, 70001))
@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float32))
def test_masked_and_infinite_logits(vocab, dtype):
    logits, u = _logits(12, vocab, 5, dtype)
    logits[0] = -math.inf                               # nothing to draw
    logits[1] = -math.inf
    logits[1, vocab - 1] = -3.0                         # one token alone
    logits[2, ::2] = torch.finfo(dtype).min             # masked by the lowest value
    logits[3] = torch.finfo(dtype).min                  # all of them: equally likely
    logits[4, 1::2] = -math.inf
    logits[5, 7], logits[5, 20] = math.inf, math.inf    # they share the draw
    logits[6, :] = math.inf
    logits[7, 3::5] = math.nan
    logits[8] = math.nan
    logits[9, :40] = math.nan
    logits[9, 40:] = -math.inf
    logits[10] = torch.finfo(dtype).max
    logits[11, 0] = torch.finfo(dtype).max
    for settings in (dict(), dict(top_k=9), dict(top_p=0.8), dict(min_p=0.1), dict(temperature=0.0), dict(top_k=20, top_p=0.5, temperature=3.0),
                     dict(temperature=1e-20), dict(temperature=1e30), dict(temperature=1e30, top_k=7, top_p=0.9)):
        _same(logits, u, **settings)
    got = sd.sample_tokens(logits, u, empty_token=17)
    assert [got[i].item() for i in (0, 8, 9)] == [17, 17, 17]


def test_top_k_keeps_what_there_is():
    logits, u = _logits(4, 3000, 2)
    logits[:, 6:] = -math.inf
    _same(logits, u, top_k=50)
    _same(logits, u, top_k=50, top_p=0.7)
    _same(logits, u, top_k=6)


def test_far_and_close_logits():
    """Values around zero, in one step of the histogram, many binades apart, and next to each other in their type."""
    gen = torch.Generator(device="cuda").manual_seed(4)
    tiny = 1e-30 * torch.randn(3, 9000, generator=gen, device="cuda")
    close = 7.0 + 1e-6 * torch.randn(3, 9000, generator=gen, device="cuda")
    wide = 1e4 * torch.randn(3, 9000, generator=gen, device="cuda")
    mixed = torch.randn(3, 9000, generator=gen, device="cuda") * torch.logspace(-20, 1, 9000, device="cuda")
    u = torch.tensor([0.1, 0.55, 0.97], device="cuda")
    for x in (tiny, close, wide, mixed):
        for settings in (dict(), dict(top_k=100), dict(top_p=0.6), dict(top_k=4000, top_p=0.9), dict(temperature=40.0, top_p=0.7),
                         dict(temperature=1e4, top_k=3000), dict(min_p=0.9)):
            _same(x, u, **settings)


def test_layouts():
    logits, u = _logits(10, 4001, 6)
    wide = torch.randn(10, 4100, device="cuda").to(torch.bfloat16)
    for start in range(0, 9):
        view = wide[:, start:start + 4001]
        _same(view, u, top_k=30, top_p=0.9)
    _same(wide[::3], u[:4], top_p=0.9)
    _same(wide.t()[:50], torch.rand(50, device="cuda"), top_k=5)
    _same(logits[:1].expand(10, 4001), u)
    assert sd.sample_tokens(logits[:0], u[:0]).shape == (0,)


def test_a_row_does_not_depend_on_its_batch():
    """One row alone is split over eight CTAs, in a large batch it is not: the same token."""
    logits, u = _logits(300, 20000, 7, torch.float32)
    for settings in (dict(), dict(top_p=0.9), dict(top_k=40, top_p=0.95)):
        whole = sd.sample_tokens(logits, u, **settings)
        for lo, hi in ((0, 1), (10, 40), (100, 180)):
            assert torch.equal(sd.sample_tokens(logits[lo:hi], u[lo:hi], **settings), whole[lo:hi])


def test_draws_follow_the_distribution():
    """All quantiles of one row: the share of each token is its probability to one part in the number of draws."""
    logits = torch.tensor([[0.0, 1.0, 2.0, 3.0, -1.0]], device="cuda")
    n = 4096
    u = ((torch.arange(n, device="cuda") + 0.5) / n).float()
    got = torch.bincount(sd.sample_tokens(logits.expand(n, 5), u, temperature=0.8), minlength=5).double() / n
    want = torch.softmax(logits[0].double() / 0.8, 0)
    assert (got - want).abs().max().item() <= 1.0 / n


def test_streams_and_graphs():
    logits, u = _logits(3, 32000, 1)
    graph = torch.cuda.CUDAGraph()
    keep = torch.tensor([40, 0, 5], dtype=torch.int32, device="cuda")
    with torch.cuda.graph(graph):
        out = sd.sample_tokens(logits, u, top_k=keep, top_p=0.95, temperature=0.9)
    for seed in (2, 3):
        fresh = _logits(3, 32000, seed)
        logits.copy_(fresh[0])
        u.copy_(fresh[1])
        graph.replay()
        assert out.tolist() == ref.tokens(logits, u, top_k=keep, top_p=0.95, temperature=0.9)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = sd.sample_tokens(logits, u, top_p=0.9)
    side.synchronize()
    assert got.tolist() == ref.tokens(logits, u, top_p=0.9)


def test_refusals():
    logits, u = _logits(4, 100, 1)
    with pytest.raises(TypeError, match="BF16 or FP32"):
        sd.sample_tokens(logits.half(), u)
    with pytest.raises(ValueError, match="B,V"):
        sd.sample_tokens(logits[0], u)
    with pytest.raises(TypeError, match="uniform must be FP32"):
        sd.sample_tokens(logits, u.double())
    with pytest.raises(ValueError, match="uniform must be"):
        sd.sample_tokens(logits, u[:3])
    with pytest.raises(ValueError, match="262144"):
        sd.sample_tokens(torch.zeros(1, 262145, device="cuda"), u[:1])
    for bad in (dict(temperature=-0.1), dict(temperature=math.nan), dict(temperature=math.inf), dict(top_p=1.01), dict(top_p=-0.1),
                dict(min_p=2.0), dict(min_p=math.nan), dict(top_k=-1)):
        with pytest.raises(ValueError, match=next(iter(bad))):
            sd.sample_tokens(logits, u, **bad)
    with pytest.raises(ValueError, match="top_p must be"):
        sd.sample_tokens(logits, u, top_p=torch.ones(3, device="cuda"))
    with pytest.raises(ValueError, match="device of the logits"):
        sd.sample_tokens(logits, u, top_p=torch.ones(4))
    with pytest.raises(TypeError, match="whole numbers"):
        sd.sample_tokens(logits, u, top_k=torch.ones(4, device="cuda"))


@pytest.mark.parametrize("dtype,rows,vocab", ((torch.float32, 160, 70000), (torch.bfloat16, 256, 128000), (torch.bfloat16, 300, 170001), (torch.float32, 3, 262144)))
def test_flat_rows_of_more_entries_than_a_short_counter_takes(dtype, rows, vocab):
    """Equal and nearly equal logits, tens of thousands of them in one step and one CTA, top-p with and without min-p."""
    u = ((torch.arange(rows, device="cuda") % 16 + 0.4) / 16).float()
    equal = torch.full((rows, vocab), -2.5, dtype=dtype, device="cuda")
    two = equal.clone()
    two[:, 7::3] = -1.0
    for x in (equal, two):
        for settings in (dict(top_p=0.5, min_p=0.1), dict(top_p=0.9, min_p=0.05), dict(top_p=0.5), dict(top_p=0.97, temperature=1e20, min_p=0.5),
                         dict(top_p=0.4, top_k=vocab - 10, min_p=0.1), dict(top_p=0.5, min_p=0.3)):
            got = sd.sample_tokens(x, u, **settings)
            assert got[:16].tolist() == ref.tokens(x[:16], u[:16], **settings)
            assert torch.equal(got[16:], got[:16].repeat(-(-rows // 16))[16:rows])


@pytest.mark.parametrize("dtype,rows,vocab,spread", ((torch.float32, 24, 128000, 0.5), (torch.bfloat16, 24, 128000, 0.5), (torch.float32, 200, 40000, 0.4),
                                                     (torch.bfloat16, 2, 32000, 0.3)))
def test_top_p_next_to_one_beside_min_p(dtype, rows, vocab, spread):
    """Flat rows whose top-p border lies at their end, close in front of what min-p takes or behind it."""
    gen = torch.Generator(device="cuda").manual_seed(vocab + rows)
    row = (spread * torch.randn(1, vocab, generator=gen, device="cuda")).to(dtype)
    u = ((torch.arange(24, device="cuda") + 0.5) / 24).float().repeat(-(-rows // 24))[:rows].contiguous()
    logits = row.expand(rows, vocab).contiguous()
    weights = (row[0].double() - row.max().double()).exp().sort().values.cpu()
    for smallest in (0, 5, 40):   # min-p at the smallest weight (nothing goes), and at others in front of it
        min_p = float(weights[smallest]) * 0.999
        for top_p in (0.999, 0.9999, 0.99999, 0.999995, 1 - 2 ** -24):
            got = sd.sample_tokens(logits, u, top_p=top_p, min_p=min_p)
            assert got[:24].tolist() == ref.tokens(logits[:24], u[:24], top_p=top_p, min_p=min_p)
            assert torch.equal(got[24:], got[:24].repeat(-(-rows // 24))[24:rows])
