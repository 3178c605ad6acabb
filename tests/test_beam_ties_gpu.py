"""What decides between the beams of a group, at the last of its 64 bits: totals that are equal, and the logarithms in them."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -53  # half a step of 64 bits, relative


@pytest.fixture(scope="module")
def ctx():
    import needle_amd as na

    c = na.Context(0)
    yield c
    c.close()


@pytest.fixture(scope="module")
def torch():
    import torch

    return torch


def _select(ctx, torch, x, scores, k, beams, mask=None, finished=None, end=0):
    import needle_amd as na

    groups = x.shape[0] // beams
    p, t = (torch.full((groups, k), 12345, dtype=torch.int32, device="cuda") for _ in range(2))
    s, c = torch.full((groups, k), 7.0, device="cuda"), torch.full((groups,), 12345, dtype=torch.int32, device="cuda")
    words = None if mask is None else torch.from_numpy(np.stack([na.pack_bitmask(r) for r in mask]).view(np.int32)).cuda()
    ctx.beam_select_device(x, None if scores is None else torch.as_tensor(scores, dtype=torch.float32).cuda(), k, p, t, s, c, beams=beams, d_mask=words,
                           d_finished=None if finished is None else torch.as_tensor(finished).cuda(), end_token=end)
    return p.cpu().numpy(), t.cpu().numpy(), s.cpu().numpy(), c.cpu().numpy()


@pytest.mark.parametrize("others", ("mask", "-inf", "lowest", "low"))
@pytest.mark.parametrize("dtype,vocab", [("float32", 50), ("float16", 9000), ("bfloat16", 20_001), ("float32", 1_000_003)])
def test_a_forced_beam_equals_an_ended_one(ctx, torch, dtype, vocab, others):
    """A beam with one continuation that counts -- what a mask admits, or the only logit that is not -inf, the type's lowest
    value or 65 below -- has log-probability 0 for it, so that its total is its score, as an ended beam's is: the lower beam
    comes first, whichever of the two has ended.  (The longest row is cut into more than 64 pieces.)"""
    t = getattr(torch, dtype)
    rng = np.random.default_rng(vocab)
    for token in {0, 17, vocab // 2, vocab - 1}:
        x = torch.randn(2, vocab, generator=torch.Generator(device="cuda").manual_seed(token), device="cuda").to(t)
        mask = None
        if others == "mask":
            mask = np.tile(np.arange(vocab) == token, (2, 1))
        else:
            x[:] = {"-inf": -np.inf, "lowest": torch.finfo(t).min, "low": -60.0}[others]
            x[:, token] = 5.0
        for ended in (0, 1):
            for s in (None, 0.0, -3.7, 1e-3, np.float32(rng.standard_normal() * 20)):
                for k in (1, 2):
                    finished = np.arange(2) == ended
                    p, tok, got, c = _select(ctx, torch, x, None if s is None else [s, s], k, 2, mask, finished, 3)
                    assert p.tolist() == [[0, 1][:k]] and tok.tolist() == [[3 if b == ended else token for b in (0, 1)][:k]]
                    assert (got == np.float32(0.0 if s is None else s)).all() and c.tolist() == [k]
        p, tok, got, c = _select(ctx, torch, x, [-2.0, -2.0], 2, 2, mask)  # neither ended
        assert p.tolist() == [[0, 1]] and tok.tolist() == [[token, token]] and (got == -2.0).all() and c.tolist() == [2]


@pytest.mark.parametrize("few", (2, 4))
def test_rows_of_few_equal_logits_tie_wherever_those_lie(ctx, torch, few):
    """log 2 and log 4 are one number each, whether the logits meet in one thread, one piece or only in the join."""
    vocab, rows = 300_000, 6
    places = [np.arange(few), np.arange(few) * 256, np.arange(few) * 4096, np.arange(few) * 60_000, vocab - 1 - np.arange(few) * 3, 5000 + np.arange(few) * 70_001]
    x = torch.full((rows, vocab), -np.inf, device="cuda")
    for r, at in enumerate(places):
        x[r, torch.from_numpy(np.sort(at)).cuda()] = 1.5 * r  # (a row's log-probabilities do not depend on its height)
    p, tok, s, c = _select(ctx, torch, x, None, rows * few, rows)
    assert p.tolist() == [np.repeat(np.arange(rows), few).tolist()] and tok.tolist() == [np.concatenate([np.sort(a) for a in places]).tolist()]
    assert (s == np.float32(-np.log(float(few)))).all() and c.tolist() == [rows * few]


@pytest.mark.parametrize("dtype,vocab,spread", [("float32", 700, 2.5), ("float32", 20_001, 2.5), ("bfloat16", 20_001, 2.5), ("float16", 131_072, 1.0),
                                                ("float32", 1_000_003, 6.0), ("bfloat16", 50_021, 0.0), ("float32", 30_000, 30.0)])
def test_the_logarithm_of_a_row(ctx, torch, dtype, vocab, spread):
    """A running score next to a row's logarithm leaves its last bits in the total.  With u = 2^-53 an exponential e^x is off
    by (4 + |x|) u of itself at most (its polynomial, its table, the product with 1 / ln 2), a term of the sum meets up to
    one rounding for each of its thread's logits, a rescaling (an exponential and a product; their arguments add up to |x|) per
    chunk, and less than 60 for the sums of waves and pieces and their scalings; then the logarithm and its sum with the
    row's maximum, half a step or one of theirs.  The report is rounded to f32."""
    g = torch.Generator(device="cuda").manual_seed(vocab)
    x = (torch.randn(4, vocab, generator=g, device="cuda") * spread).to(getattr(torch, dtype))
    x[2] = x[2].sort().values             # every chunk has a new largest
    x[3] = x[3].sort(descending=True).values
    wide = x.double().cpu().numpy().astype(np.longdouble)
    top = wide.max(axis=1)
    terms = np.exp(wide - top[:, None])
    log = np.log(terms.sum(axis=1))
    start = log.astype(np.float32)
    want = start.astype(np.longdouble) - log
    chunk = 256 * 32 // x.element_size()
    chunks = -(-vocab // chunk)
    depth = (terms * (top[:, None] - wide)).sum(axis=1) / terms.sum(axis=1)
    room = U * (4 + 2 * depth + chunks * (chunk // 256) + 6 * chunks + 60) + 2 * U * (log + np.abs(top + log)) + U * np.abs(want) + 2.0 ** -24 * np.abs(want)
    _, tok, got, c = _select(ctx, torch, x, start, 1, 1)
    assert (c == 1).all() and np.array_equal(tok[:, 0], x.float().cpu().numpy().argmax(axis=1))
    off = np.abs(got[:, 0].astype(np.longdouble) - want)
    assert (off <= room).all(), (off, room)
