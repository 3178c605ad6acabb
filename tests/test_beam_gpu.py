"""The selection over the beams of a group and the move of their states through the C ABI, against a plain computation in
64 bits: picks and counts equal, scores the totals rounded to f32."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

NONE = -1
INF = float("inf")


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


def _reference(x, scores, k, beams, normalize, mask=None, finished=None, end=0):
    """x: [rows, vocab] in f64 -> (parents, tokens, totals, counts); a beam's continuations rank by logit where 64 bits do not
    tell their totals apart (all of them +inf, say)."""
    rows, vocab = x.shape
    groups = rows // beams
    parents, tokens = np.full((groups, k), NONE), np.full((groups, k), NONE)
    totals, counts = np.full((groups, k), -INF), np.zeros(groups, int)
    with np.errstate(all="ignore"):
        for g in range(groups):
            offers = []
            for b in range(beams):
                r = g * beams + b
                start = 0.0 if scores is None else float(scores[r])
                if finished is not None and finished[r]:
                    offers.append((np.array([start]), np.array([b]), np.array([end]), np.array([0.0])))
                    continue
                at = np.arange(vocab) if mask is None else np.flatnonzero(mask[r] if mask.ndim == 2 else mask)
                v = x[r, at]
                if normalize and v.size:
                    v = v - (v.max() + np.log(np.exp(v - v.max()).sum()))
                offers.append((start + v, np.full(at.size, b), at, x[r, at]))
            t, b, a, y = (np.concatenate([o[i] for o in offers]) for i in range(4))
            ok = ~np.isnan(t) & (t > -INF)
            t, b, a, y = t[ok], b[ok], a[ok], y[ok]
            order = np.lexsort((a, -y, b, -t))[:k]
            n = order.size
            counts[g], totals[g, :n], parents[g, :n], tokens[g, :n] = n, t[order], b[order], a[order]
    return parents, tokens, totals, counts


def _outputs(torch, groups, k):
    return (torch.full((groups, k), 12345, dtype=torch.int32, device="cuda"), torch.full((groups, k), 12345, dtype=torch.int32, device="cuda"),
            torch.full((groups, k), 7.0, device="cuda"), torch.full((groups,), 12345, dtype=torch.int32, device="cuda"))


def _words(torch, mask):
    import needle_amd as na

    m = np.atleast_2d(mask)
    return torch.from_numpy(np.stack([na.pack_bitmask(r) for r in m]).view(np.int32)).cuda()


def _check(ctx, torch, x, scores, k, beams, normalize, mask=None, finished=None, end=0, states=()):
    rows = x.shape[0]
    groups = rows // beams
    p, t, s, c = _outputs(torch, groups, k)
    ctx.beam_select_device(x, None if scores is None else torch.as_tensor(scores, dtype=torch.float32).cuda(), k, p, t, s, c, beams=beams,
                           normalize=normalize, d_mask=None if mask is None else _words(torch, mask),
                           d_finished=None if finished is None else torch.as_tensor(finished).cuda(), end_token=end, states=states)
    wp, wt, ws, wc = _reference(x.double().cpu().numpy(), None if scores is None else np.asarray(scores, np.float32), k, beams, normalize, mask,
                                finished, end)
    assert np.array_equal(c.cpu().numpy(), wc)
    assert np.array_equal(p.cpu().numpy(), wp) and np.array_equal(t.cpu().numpy(), wt)
    s = s.double().cpu().numpy()
    there = np.isfinite(ws)
    assert np.array_equal(s[~there], ws[~there])
    # half a step of f32 for the report; the sum of exponentials in 64 bits is 1e-10 of itself off at most
    assert (np.abs(s[there] - ws[there]) <= 2.0 ** -24 * np.abs(ws[there]) + 1e-9).all()
    return p, t, c


def _logits(torch, seed, rows, vocab, dtype="float32", pad=0, spread=2.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = (torch.randn(rows, vocab + pad, generator=g, device="cuda") * spread).to(getattr(torch, dtype))
    return x[:, :vocab]


def _scores(seed, rows):
    return -10.0 - 4.0 * np.random.default_rng(seed).random(rows).astype(np.float32)


@pytest.mark.parametrize("dtype", ("float32", "float16", "bfloat16"))
@pytest.mark.parametrize("groups,beams,vocab,k", [(1, 1, 1, 1), (1, 4, 7, 3), (3, 2, 33, 5), (2, 5, 2047, 10), (2, 3, 2049, 64), (1, 4, 8192, 4),
                                                  (5, 4, 8193, 8), (2, 8, 20_001, 65), (1, 2, 50_021, 256), (1, 16, 32_000, 16), (4, 1, 300, 200),
                                                  (1, 3, 1_000_003, 6), (130, 3, 500, 3)])
def test_select(ctx, torch, dtype, groups, beams, vocab, k):
    rows = groups * beams
    x = _logits(torch, vocab + k, rows, vocab, dtype)
    for normalize in (True, False):
        _check(ctx, torch, x, _scores(vocab, rows), k, beams, normalize)


@pytest.mark.parametrize("groups,beams,vocab,k,dtype", [(1, 1000, 300, 5, "float32"), (2, 100, 20_000, 7, "float32"), (3, 33, 9000, 64, "float16"),
                                                        (1, 10, 40_000, 64, "bfloat16"), (1, 7, 70_000, 33, "float16"), (1, 3, 20_000, 256, "bfloat16")])
def test_lists_that_meet_in_one_group(ctx, torch, groups, beams, vocab, k, dtype):
    """Many beams, or many pieces of long lists, with rows among them that end, offer nothing or have no sum."""
    rows = groups * beams
    x = _logits(torch, beams, rows, vocab, dtype)
    finished = np.zeros(rows, np.uint8)
    finished[::5] = 1
    x[1] = -INF
    x[2::9, vocab - 1] = float("nan")
    scores = _scores(k, rows)
    for normalize in (True, False):
        _check(ctx, torch, x, scores, k, beams, normalize, finished=finished, end=vocab - 1)
        _check(ctx, torch, x, None, k, beams, normalize)


@pytest.mark.parametrize("dtype,vocab,pad", [("float32", 1001, 3), ("bfloat16", 9000, 1), ("float16", 8200, 5)])
def test_rows_that_lie_apart(ctx, torch, dtype, vocab, pad):
    x = _logits(torch, 4, 12, vocab, dtype, pad)
    _check(ctx, torch, x, _scores(1, 12), 7, 3, True)
    _check(ctx, torch, x[1:], _scores(2, 11), 7, 11, False)


@pytest.mark.parametrize("share", (0.5, 0.01, 0.0))
@pytest.mark.parametrize("vocab", (31, 1000, 8200, 17_000))
def test_masks(ctx, torch, share, vocab):
    rng = np.random.default_rng(vocab)
    x = _logits(torch, 5, 12, vocab, "float16")
    mask = rng.random((12, vocab)) < share
    mask[2] = False
    mask[3] = np.arange(vocab) == vocab - 1  # one admitted continuation, the last
    mask[8] = True
    x[8, 5 % vocab] = INF  # behind no mask: without a log-softmax under normalize, the best there is otherwise
    x[0, ~torch.from_numpy(mask[0]).cuda()] = float("nan")  # what is not admitted is not looked at
    x[1, ~torch.from_numpy(mask[1]).cuda()] = INF
    for normalize in (True, False):
        _check(ctx, torch, x, _scores(3, 12), 9, 4, normalize, mask)
        _check(ctx, torch, x, _scores(3, 12), 70, 6, normalize, mask)
        _check(ctx, torch, x[4:8], _scores(3, 4), 9, 2, normalize, mask[5])  # one mask for all rows


def test_what_is_not_offered(ctx, torch):
    x = _logits(torch, 6, 16, 9000)
    x[1, 17], x[2, 8999], x[3, 3] = float("nan"), INF, -INF
    x[4] = -INF
    x[5] = float("nan")
    x[6, :8990] = -INF
    x[7] = torch.finfo(torch.float32).min  # the type's lowest value as a mask: finite, so offered
    s = _scores(4, 16)
    s[8], s[9], s[10] = -INF, float("nan"), INF
    for normalize in (True, False):
        for k in (5, 100):
            _check(ctx, torch, x, s, k, 4, normalize)
            _check(ctx, torch, x[4:7], s[4:7], k, 3, normalize)
            _check(ctx, torch, x[4:6], s[4:6], k, 1, normalize)  # groups without a pick
            _check(ctx, torch, x[8:10], s[8:10], k, 2, normalize)


def test_first_step_and_ended_beams(ctx, torch):
    x = _logits(torch, 7, 24, 10_000, "bfloat16")
    s = np.zeros(24, np.float32)
    s[np.arange(24) % 4 != 0] = -INF
    _check(ctx, torch, x, s, 4, 4, True)
    s = _scores(5, 24)
    finished = np.random.default_rng(1).random(24) < 0.4
    finished[:4] = True
    s[2], s[3] = -INF, float("nan")
    x[torch.from_numpy(finished).cuda()] = float("nan")
    mask = np.random.default_rng(2).random(10_000) < 0.3
    for m in (None, mask):
        _check(ctx, torch, x, s, 6, 4, True, m, finished, 9999)
        _check(ctx, torch, x, s, 130, 8, False, m, finished.astype(np.uint8) * 3, 17)
    _check(ctx, torch, x, None, 6, 4, True, None, finished, 5)  # no running scores: zeros


@pytest.mark.parametrize("k", (1, 10, 64, 65, 256))
def test_ties_and_orders(ctx, torch, k):
    """Equal logits in thousands (lowest token, lowest beam), logits in ascending and descending order, few distinct values,
    all large ones where one thread holds them, equal beams."""
    vocab = 20_000
    rows = [torch.zeros(vocab), torch.arange(vocab) * 1e-3, -torch.arange(vocab) * 1e-3, (torch.arange(vocab) % 3).float(),
            torch.where(torch.arange(vocab) % 1024 < 4, 50.0, 0.0) + torch.arange(vocab) * 1e-4, torch.full((vocab,), -0.0), torch.zeros(vocab), torch.zeros(vocab)]
    x = torch.stack(rows).float().cuda()
    s = np.zeros(8, np.float32)
    for normalize in (True, False):
        _check(ctx, torch, x, s, k, 1, normalize)
        _check(ctx, torch, x[5:8], s[5:8], k, 3, normalize)
        _check(ctx, torch, x[[3, 3, 3, 3]].contiguous(), s[:4], k, 2, normalize)
    _check(ctx, torch, x, s, k, 8, False)
    _check(ctx, torch, x[[0] * 40].contiguous(), np.zeros(40, np.float32), k, 40, False)


@pytest.mark.parametrize("dtype,k", [("float32", 256), ("bfloat16", 256), ("float32", 100), ("float16", 20)])
def test_rows_that_rise(ctx, torch, dtype, k):
    """Logits that grow along the row, slowly to steeply: lists of every length meet chunks of which all, many or few logits
    reach the bound, equal ones among them."""
    rows, vocab = 1024, 20_000
    g = torch.Generator(device="cuda").manual_seed(k)
    x = torch.randn(rows, vocab, generator=g, device="cuda")
    at = torch.arange(vocab, device="cuda") / 2048.0
    slope = torch.logspace(-2.5, 1.0, rows, device="cuda")[:, None]
    x = x + slope * at
    x[1::4] = x[1::4].floor()                              # thousands of equal ones
    x[2::4, 8192:9000] += 30.0                             # a block of large ones late in the row
    x[3::4] = torch.where(torch.rand(rows // 4, vocab, generator=g, device="cuda") < 0.1, x[3::4] + 5.0, x[3::4])
    x = x.to(getattr(torch, dtype))
    p, t, s, c = _outputs(torch, rows, k)
    for normalize in (True, False):
        ctx.beam_select_device(x, None, k, p, t, s, c, beams=1, normalize=normalize)
        want = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :k].to(torch.int32)
        assert (c == k).all() and not p.any() and torch.equal(t, want)
        total = torch.gather(x, 1, want.long()).double()
        if normalize:
            total = total - torch.logsumexp(x.double(), 1, keepdim=True)
        assert ((s.double() - total).abs() <= 2.0 ** -24 * total.abs() + 1e-8).all()


def test_values_over_the_range(ctx, torch):
    """Logits of any size: nothing but the largest counts in the sum, or all count alike."""
    x = _logits(torch, 9, 6, 4000)
    x[0] *= 1e30
    x[1] *= 1e-30
    x[2] += 3e4
    x[3] -= 3e4
    x[4] *= 200.0
    for normalize in (True, False):
        _check(ctx, torch, x[2:], np.float32([0, -1, 0, 2]), 5, 4, normalize)
        for r in range(6):
            p, t, s, c = _outputs(torch, 1, 5)
            ctx.beam_select_device(x[r:r + 1], None, 5, p, t, s, c, beams=1, normalize=normalize)
            assert np.array_equal(t.cpu().numpy()[0], np.argsort(-x[r].cpu().numpy(), kind="stable")[:5])


def test_many_groups_in_blocks(ctx, torch):
    """More pieces than one launch takes: the blocks of groups line up, masks, scores and ends with them."""
    rows, vocab, k = 9000 * 4, 200, 256
    x = _logits(torch, 10, rows, vocab, "bfloat16")
    rng = np.random.default_rng(6)
    s, finished, mask = _scores(6, rows), rng.random(rows) < 0.2, rng.random((rows, vocab)) < 0.5
    p, t, sc, c = _outputs(torch, 9000, k)
    words = _words(torch, mask)
    ctx.beam_select_device(x, torch.from_numpy(s).cuda(), k, p, t, sc, c, beams=4, normalize=True, d_mask=words,
                           d_finished=torch.from_numpy(finished).cuda(), end_token=3)
    for g0 in (0, 4400, 8950):
        r = slice(g0 * 4, (g0 + 50) * 4)
        wp, wt, ws, wc = _reference(x[r].double().cpu().numpy(), s[r], k, 4, True, mask[r], finished[r], 3)
        g = slice(g0, g0 + 50)
        assert np.array_equal(p[g].cpu().numpy(), wp) and np.array_equal(t[g].cpu().numpy(), wt) and np.array_equal(c[g].cpu().numpy(), wc)


def test_no_continuations(ctx, torch):
    for groups, beams, vocab, k in ((3, 2, 0, 4), (3, 2, 10, 0), (0, 2, 10, 4)):
        p, t, s, c = _outputs(torch, groups, k)
        ctx.beam_select_device(torch.empty(groups * beams, vocab, device="cuda"), None, k, p, t, s, c, beams=beams)
        assert not c.any() and (p == NONE).all() and (t == NONE).all() and (s == -INF).all()


def test_host_form(ctx, torch):
    rng = np.random.default_rng(8)
    x = (rng.standard_normal((6, 3001)) * 2).astype(np.float32)
    s, mask = _scores(7, 6), rng.random((6, 3001)) < 0.2
    finished = np.array([0, 0, 1, 0, 0, 0])
    for xx, m, f in ((x, None, None), (x, mask, finished), (x.astype(np.float16), mask[1], None)):
        p, t, sc, c = ctx.beam_select(xx, s, 8, beams=3, mask=m, finished=f, end_token=1)
        wp, wt, ws, wc = _reference(xx.astype(np.float64), s, 8, 3, True, m, f, 1)
        assert np.array_equal(p.view(np.int32), wp) and np.array_equal(t.view(np.int32), wt) and np.array_equal(c, wc)
        assert (np.abs(sc - ws) <= 2.0 ** -24 * np.abs(ws) + 1e-9).all()
    p, t, sc, c = ctx.beam_select(x, None, 2, beams=2, normalize=False)
    assert p.shape == (3, 2) and (c == 2).all()


# ---- states ---------------------------------------------------------------------------------------------


def _moved(torch, src, dst, parents, beams, axis=0):
    want = dst.clone()
    groups, k = parents.shape
    for g in range(groups):
        for j in range(k):
            b = int(parents[g, j])
            if 0 <= b < beams:
                want.select(axis, g * k + j).copy_(src.select(axis, g * beams + b))
    return want


def test_states_move_with_the_picks(ctx, torch):
    groups, beams, k = 5, 4, 6
    g = torch.Generator(device="cuda").manual_seed(3)

    def pair(shape, axis, dtype):
        out = []
        for n in (groups * beams, groups * k):
            s = list(shape)
            s[axis] = n
            out.append((torch.randn(s, generator=g, device="cuda") * 50).to(dtype))
        return out

    keys = pair((0, 3, 20, 64), 0, torch.bfloat16)
    layers = pair((7, 0, 2, 33), 1, torch.float16)
    wide = pair((0, 5000), 0, torch.float32)
    narrow = pair((0, 5), 0, torch.int8)
    single = pair((0,), 0, torch.int64)
    states = [(keys[0][:, :, :13], keys[1][:, :, :13]), (layers[0], layers[1], 1), (wide[0], wide[1]), (narrow[0][:, 1:4], narrow[1][:, 1:4]),
              (single[0], single[1]), (layers[0][:, :, 0].clone(), layers[1][:, :, 0].clone(), 1)]
    states += [(torch.randn(groups * beams, n, generator=g, device="cuda"), torch.zeros(groups * k, n, device="cuda")) for n in range(1, 12)]
    before = [s[1].clone() for s in states]
    whole = [keys[1].clone(), narrow[1].clone()]
    x = _logits(torch, 11, groups * beams, 900)
    mask = np.ones((groups * beams, 900), bool)
    mask[4:8] = False       # a group without a pick
    mask[8:12, 3:] = False  # and one with few
    mask[8:11] = False
    p, _, c = _check(ctx, torch, x, _scores(8, groups * beams), k, beams, True, mask, states=states)
    assert int(c[1]) == 0 and int(c[2]) == 3
    for s, was in zip(states, before):
        assert torch.equal(s[1], _moved(torch, s[0], was, p.cpu(), beams, s[2] if len(s) > 2 else 0))
    assert torch.equal(keys[1][:, :, 13:], whole[0][:, :, 13:]) and torch.equal(narrow[1][:, [0, 4]], whole[1][:, [0, 4]])


def test_reorder_alone(ctx, torch):
    src, dst = torch.randn(6, 1000, device="cuda"), torch.randn(8, 1000, device="cuda")
    parents = torch.tensor([[2, 2, -1, 0], [1, 7, 0, 3]], dtype=torch.int32, device="cuda")  # -1, 7 and 3 name no beam of three
    want = _moved(torch, src, dst, parents.cpu(), 3)
    ctx.beam_reorder_device(parents, [(src, dst)], beams=3)
    assert torch.equal(dst, want)
    ctx.beam_reorder_device(parents, [], beams=3)
    ctx.beam_reorder_device(parents[:0], [(src[:0], dst[:0])], beams=3)


def test_states_that_interleave_in_one_array(ctx, torch):
    """Keys and values of several layers, a beam's all in one row, and as pairs of runs."""
    groups, beams, k = 3, 4, 5
    g = torch.Generator(device="cuda").manual_seed(14)
    src = torch.randn(groups * beams, 2, 3, 7, 64, generator=g, device="cuda")  # rows, keys / values, layers, heads, dims
    dst = torch.randn(groups * k, 2, 3, 7, 64, generator=g, device="cuda")
    parents = torch.randint(0, beams, (groups, k), generator=g, device="cuda", dtype=torch.int32)
    parents[1, 2] = -1
    want = _moved(torch, src, dst, parents.cpu(), beams)
    for parts in ([lambda t, j=j: t[:, j] for j in range(2)], [lambda t, j=j, y=y: t[:, j, y] for j in range(2) for y in range(3)],
                  [lambda t, j=j: t[:, :, :, j] for j in range(7)], [lambda t, j=j: t.reshape(t.shape[0], 42, 2, 32)[:, :, j] for j in range(2)]):
        out = dst.clone()
        ctx.beam_reorder_device(parents, [(part(src), part(out)) for part in parts], beams=beams)
        assert torch.equal(out, want)
    out = dst.clone()
    with pytest.raises(Exception, match="overlaps"):
        ctx.beam_reorder_device(parents, [(src[:, 0], out[:, 0]), (src[:, :, 0], out[:, :, 0])], beams=beams)
    assert torch.equal(out, dst)


def test_states_behind_four_gigabytes(ctx, torch):
    rows = torch.randint(-128, 128, (4, 2 ** 31 - 77), device="cuda", dtype=torch.int8)  # offsets of rows 2 and 3 pass 2^32
    dst = torch.zeros(4, 2 ** 31 - 77, device="cuda", dtype=torch.int8)
    parents = torch.tensor([[3, 2, 3, 0]], dtype=torch.int32, device="cuda")
    ctx.beam_reorder_device(parents, [(rows, dst)], beams=4)
    for j, b in enumerate((3, 2, 3, 0)):
        assert torch.equal(dst[j], rows[b])


# ---- together -----------------------------------------------------------------------------------------------


def test_hops_of_a_retrieval_chain(ctx, torch):
    """Three hops: the chains' query vectors are scored against an int8 base, the best chains of every request are kept, and
    their vectors and histories move; against the same steps in 64 bits from the same codes."""
    groups, beams, n, dim = 3, 4, 5000, 96
    g = torch.Generator(device="cuda").manual_seed(12)
    base = torch.randn(n, dim, generator=g, device="cuda")
    codes, scales = torch.empty(n, dim, dtype=torch.int8, device="cuda"), torch.empty(n, device="cuda")
    ctx.quantize_rows_device(base, codes, scales)
    deq = codes.double() * scales.double()[:, None]
    q = torch.randn(groups, dim, generator=g, device="cuda").repeat_interleave(beams, 0).contiguous()
    path = torch.full((groups * beams, 3), -1, dtype=torch.int32, device="cuda")
    total = torch.full((groups, beams), -INF, device="cuda")
    total[:, 0] = 0.0
    want_total, want_path = total.double().cpu(), path.cpu().clone()
    out = torch.empty(groups * beams, n, device="cuda")
    for hop in range(3):
        ctx.linear_i8_device(q, codes, scales, out)
        q_codes, q_scales = torch.empty(groups * beams, dim, dtype=torch.int8, device="cuda"), torch.empty(groups * beams, device="cuda")
        ctx.quantize_rows_device(q, q_codes, q_scales)
        ref = (q_codes.double() * q_scales.double()[:, None]) @ deq.t().contiguous()
        rt = want_total.reshape(-1, 1).numpy() + torch.log_softmax(ref, 1).cpu().numpy()
        order = np.argsort(-rt.reshape(groups, -1), axis=1, kind="stable")[:, :beams]
        want_total = torch.from_numpy(np.take_along_axis(rt.reshape(groups, -1), order, 1))
        p, t, s, c = _outputs(torch, groups, beams)
        q2, path2 = torch.empty_like(q), torch.empty_like(path)
        ctx.beam_select_device(out, total.reshape(-1), beams, p, t, s, c, beams=beams, states=[(q, q2), (path, path2)])
        assert (c == beams).all()
        assert np.array_equal(p.cpu().numpy(), order // n) and np.array_equal(t.cpu().numpy(), order % n)
        # logits of size about 100 with three f32 roundings, their largest again in the sum, and totals added up in f32
        assert (s.double().cpu() - want_total).abs().max() < 3 * (8 * 2.0 ** -24 * 200)
        want_path = want_path[torch.from_numpy((np.arange(groups)[:, None] * beams + order // n).reshape(-1))]
        want_path[:, hop] = torch.from_numpy((order % n).reshape(-1))
        path2[:, hop] = t.reshape(-1)
        q, path, total = (q2 + base[t.reshape(-1).long()]) * 0.5, path2, s
        assert torch.equal(path.cpu(), want_path)
