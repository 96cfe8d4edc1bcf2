"""append_paged() and attend_paged() against plain 64-bit forms."""

import math

import pytest
import torch

from conftest import requires_gpu
from paged_oracle import Paged, check_attention
from test_rope_gpu import check as check_rope

import flashattn_cuda

pytestmark = [pytest.mark.gpu, requires_gpu]
F16, BF16 = torch.float16, torch.bfloat16


def attend(c, scale=None, **kw):
    return flashattn_cuda.attend_paged(c.q, c.starts, c.kp, c.vp, c.table, c.seq_lens,
                                       scale or c.d ** -0.5, **kw)


def clean():
    assert flashattn_cuda.take_device_error() == 0


# ---------------------------------------------------------------- attention
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("h,h_kv", [(12, 12), (14, 2), (8, 1), (40, 2)])
@pytest.mark.parametrize("news,lens", [
    ([1], [1]),
    ([1, 1, 1, 1], [1, 17, 128, 1291]),
    ([3, 1, 5, 8], [3, 700, 129, 64]),
    ([130, 0, 37, 1], [130, 50, 437, 2000]),
    ([300], [1324]),
])
def test_attention_matches_the_definition(dtype, d, h, h_kv, news, lens):
    c = Paged(news, lens, h, h_kv, d, 16, dtype, seed=h + d)
    for causal in (True, False):
        out, lse = attend(c, causal=causal, return_lse=True)
        check_attention(c, out, d ** -0.5, causal, lse)
        assert torch.equal(out, attend(c, causal=causal))
    clean()


@pytest.mark.parametrize("token_major", [False, True])
@pytest.mark.parametrize("page", [8, 16, 24, 56, 64, 96, 128, 200, 256])
@pytest.mark.parametrize("news,lens", [([1, 1, 1], [255, 256, 1000]),
                                       ([70, 129, 1], [70, 600, 385])])
def test_page_sizes_and_layouts(token_major, page, news, lens):
    for d, h, h_kv in ((64, 6, 3), (128, 8, 2)):
        c = Paged(news, lens, h, h_kv, d, page, F16, token_major, seed=page)
        check_attention(c, attend(c), d ** -0.5)
    clean()


def test_lengths_around_every_tile_edge():
    lens = list(range(1, 34)) + [63, 64, 65, 127, 128, 129, 191, 192, 193, 255, 256, 257]
    for d, h, h_kv in ((64, 2, 1), (128, 4, 4)):
        c = Paged([1] * len(lens), lens, h, h_kv, d, 32, BF16, seed=d)
        check_attention(c, attend(c), d ** -0.5)
        c = Paged(lens, lens, h, h_kv, d, 32, F16, seed=d + 1)
        check_attention(c, attend(c), d ** -0.5)
    clean()


def test_rows_that_see_nothing():
    """Sequences without rows, without new tokens, and with more new tokens
    than rows (the first of them stand before row 0)."""
    news, lens = [2, 0, 9, 1, 0, 140], [0, 33, 4, -3, 0, 20]
    for h, h_kv, d in ((6, 2, 64), (4, 4, 128)):
        c = Paged(news, lens, h, h_kv, d, 16, F16, seed=9)
        out, lse = attend(c, return_lse=True)
        check_attention(c, out, d ** -0.5, True, lse)
        assert not out[:2].any() and not out[2:7].any() and out[7:11].any(-1).all()
        out, lse = attend(c, causal=False, return_lse=True)
        check_attention(c, out, d ** -0.5, False, lse)
    clean()


@pytest.mark.parametrize("n", [1, 4, 200])
def test_long_cache(n):
    c = Paged([n, 1], [30011, 5], 14, 2, 64, 64, F16, seed=n)
    check_attention(c, attend(c), 0.125)
    c = Paged([n], [20000], 8, 2, 128, 128, BF16, seed=n + 1)
    check_attention(c, attend(c), 128 ** -0.5)
    clean()


def test_many_sequences():
    g = torch.Generator().manual_seed(0)
    lens = torch.randint(0, 300, (700,), generator=g).tolist()
    c = Paged([1] * 700, lens, 4, 2, 64, 32, F16, seed=2)
    check_attention(c, attend(c), 0.125)
    news = [min(x, int(y)) for x, y in zip(lens, torch.randint(0, 40, (700,), generator=g))]
    c = Paged(news, lens, 4, 2, 64, 32, F16, seed=3)
    check_attention(c, attend(c), 0.125)
    clean()


@pytest.mark.parametrize("scale,sharp", [(0.125, 40.0), (-0.125, 1.0), (0.0, 1.0), (1e-6, 1.0)])
def test_scales(scale, sharp):
    """Sharp rows (scores of a few hundred, the softmax nearly one-hot: the
    score's own fp32 rounding, 2^-22 of it, is within the tolerance), and
    scales that are negative or nothing."""
    for news, lens in (([1, 1], [300, 1000]), ([150, 20], [300, 1000])):
        c = Paged(news, lens, 6, 2, 64, 16, F16, sharp=sharp, seed=4)
        out = flashattn_cuda.attend_paged(c.q, c.starts, c.kp, c.vp, c.table, c.seq_lens, scale)
        check_attention(c, out, scale)
    clean()


def test_views_of_q_and_tables():
    c = Paged([1, 60, 2], [100, 260, 90], 6, 2, 128, 16, BF16, seed=5)
    want = attend(c)
    fused = torch.randn(63, 10, 128, device="cuda").bfloat16()
    fused[:, 2:8] = c.q
    wide = torch.full((6, c.table.shape[1] + 3), -7, device="cuda", dtype=torch.int32)
    wide[::2, :c.table.shape[1]] = c.table
    pools = torch.stack((c.kp, c.vp), 1)  # (pages, 2, heads, rows, dim)
    got = flashattn_cuda.attend_paged(fused[:, 2:8], c.starts, pools[:, 0], pools[:, 1],
                                      wide[::2], c.seq_lens, 128 ** -0.5)
    assert torch.equal(got, want)
    check_attention(c, got, 128 ** -0.5)
    clean()


def test_capacity_of_the_table_bounds_the_rows():
    """seq_lens past the table's capacity: the rows there are attended, and
    the tokens keep their positions."""
    c = Paged([2, 2], [64, 40], 4, 2, 64, 16, F16, seed=6)
    longer = c.seq_lens + torch.tensor([5, 0], device="cuda", dtype=torch.int32)
    out = flashattn_cuda.attend_paged(c.q, c.starts, c.kp, c.vp, c.table, longer, 0.125)
    c.lens = [64, 40]
    want, _, _ = c.exact(0.125, causal=False)
    assert (out[:2].double() - want[:2]).abs().max() < 3e-3
    check_tail, _, _ = c.exact(0.125)
    assert (out[2:].double() - check_tail[2:]).abs().max() < 3e-3
    clean()


@pytest.mark.parametrize("news", [[1, 1], [70, 3]])
def test_missing_pages_are_reported(news):
    c = Paged(news, [100, 90], 4, 2, 64, 16, F16, seed=7)
    for entry in (-1, c.kp.shape[0], 2 ** 31 - 1):
        table = c.table.clone()
        table[0, 1] = entry
        out = flashattn_cuda.attend_paged(c.q, c.starts, c.kp, c.vp, table, c.seq_lens, 0.125)
        assert flashattn_cuda.take_device_error() == 4
        want, _, _ = c.exact(0.125)  # the other sequence is whole
        assert (out[news[0]:].double() - want[news[0]:]).abs().max() < 3e-3
    clean()


def test_tokens_of_no_sequence_are_left_alone():
    c = Paged([3, 40], [30, 60], 4, 2, 64, 16, F16, seed=8)
    q = torch.cat((c.q, torch.full((5, 4, 64), float("nan"), device="cuda").half()))
    out = flashattn_cuda.attend_paged(q, c.starts, c.kp, c.vp, c.table, c.seq_lens, 0.125)
    check_attention(c, out[:43], 0.125)
    clean()


def test_repeated_calls_streams_and_graphs_agree():
    c = Paged([1, 90, 1, 0, 4], [5000, 900, 17, 3, 333], 8, 2, 128, 64, F16, seed=10)
    want = attend(c)
    for _ in range(20):
        assert torch.equal(attend(c), want)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        q = c.q * 1
        got = flashattn_cuda.attend_paged(q, c.starts, c.kp, c.vp, c.table, c.seq_lens,
                                          128 ** -0.5)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            replayed = attend(c)
        g.replay()
    s.synchronize()
    assert torch.equal(got, want) and torch.equal(replayed, want)
    # another step through the same graph: shorter lengths, other starts
    d = Paged([40, 0, 50, 5, 1], [77, 2, 800, 30, 256], 8, 2, 128, 64, F16, seed=11)
    pages = min(c.kp.shape[0], d.kp.shape[0])
    assert d.kp.shape[0] <= pages and d.table.shape[1] <= c.table.shape[1]
    c.kp[:pages] = d.kp
    c.vp[:pages] = d.vp
    c.table[:, :d.table.shape[1]] = d.table
    c.q.copy_(d.q)
    c.starts.copy_(d.starts)
    c.seq_lens.copy_(d.seq_lens)
    g.replay()
    torch.cuda.synchronize()
    check_attention(d, replayed, 128 ** -0.5)
    clean()


def test_one_sequence_equals_prefill_and_decode():
    """The same rows in one contiguous cache through prefill() and decode()."""
    for d in (64, 128):
        c = Paged([500], [500], 8, 2, d, 64, F16, seed=12)
        k, v = (x[0].transpose(0, 1)[None].contiguous() for x in (c.k, c.v))
        q = c.q.transpose(0, 1)[None].contiguous()
        want = flashattn_cuda.prefill(q, k, v, True, d ** -0.5)[0].transpose(0, 1)
        assert (attend(c).float() - want.float()).abs().max() <= 4e-3
        one = flashattn_cuda.attend_paged(
            c.q[-1:], torch.tensor([0, 1], device="cuda", dtype=torch.int32), c.kp, c.vp,
            c.table, c.seq_lens, d ** -0.5)
        want = flashattn_cuda.decode(q[:, :, -1:].contiguous(), k, v, c.seq_lens, d ** -0.5)
        assert (one[0].float() - want[0, :, 0].float()).abs().max() <= 4e-3
    clean()


def test_nothing_to_do():
    c = Paged([0, 0], [3, 40], 4, 2, 64, 16, F16)
    out, lse = attend(c, return_lse=True)
    assert out.shape == (0, 4, 64) and lse.shape == (0, 4)


# ------------------------------------------------------------------- append
def append_case(dtype=F16, d=64, h=6, h_kv=2, page=16, token_major=False, news=None,
                lens=None, seed=0):
    news, lens = news or [1, 30, 0, 5], lens or [1, 77, 20, 133]
    c = Paged(news, lens, h, h_kv, d, page, dtype, token_major, seed=seed)
    t = sum(news)
    fused = torch.randn(t, h + 2 * h_kv, d, device="cuda").to(dtype)
    c.fused = fused
    c.q, c.kn, c.vn = fused[:, :h], fused[:, h:h + h_kv], fused[:, h + h_kv:]
    rows = [torch.arange(x - n, x) for n, x in zip(news, lens)]
    c.rows = torch.cat(rows).to(torch.int32).cuda()
    c.seq = torch.cat([torch.full((n,), b) for b, n in enumerate(news)]).cuda()
    return c


def packed(x):  # (tokens, heads, d) as rope() sees it
    return x.transpose(0, 1)[None]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d,rot,page,token_major", [
    (64, 64, 16, False), (128, 128, 64, True), (128, 32, 8, False), (64, 20, 256, True)])
@pytest.mark.parametrize("news,lens", [([1], [1]), ([1, 30, 0, 5], [1, 77, 20, 133]),
                                       ([900, 1], [1000, 300])])
def test_append_stores_and_rotates(dtype, interleaved, d, rot, page, token_major, news, lens):
    c = append_case(dtype, d, page=page, token_major=token_major, news=news, lens=lens)
    freqs, _ = flashattn_cuda.rope_frequencies(rot)
    want_k, want_v = c.kp.clone(), c.vp.clone()
    qo = flashattn_cuda.append_paged(c.kn, c.vn, c.starts, c.kp, c.vp, c.table, c.seq_lens,
                                     q=c.q, freqs=freqs, interleaved=interleaved,
                                     amplitude=1.5)
    kw = dict(amplitude=1.5)
    check_rope(packed(qo).contiguous(), packed(c.q), c.rows, freqs, interleaved, **kw)
    pages = c.table[c.seq, (c.rows // page).long()].long()
    stored = c.kp[pages, :, (c.rows % page).long()]
    check_rope(packed(stored).contiguous(), packed(c.kn), c.rows, freqs, interleaved, **kw)
    # V whole, and no other row of the pools
    want_k[pages, :, (c.rows % page).long()] = stored
    want_v[pages, :, (c.rows % page).long()] = c.vn
    same = lambda a, b: torch.equal(a.contiguous().view(torch.int16),
                                    b.contiguous().view(torch.int16))
    assert same(c.kp, want_k) and same(c.vp, want_v)
    clean()


def test_append_without_rotation_and_with_positions():
    c = append_case()
    assert flashattn_cuda.append_paged(c.kn, c.vn, c.starts, c.kp, c.vp, c.table,
                                       c.seq_lens) is None
    pages = c.table[c.seq, (c.rows // 16).long()].long()
    assert torch.equal(c.kp[pages, :, (c.rows % 16).long()], c.kn)
    assert torch.equal(c.vp[pages, :, (c.rows % 16).long()], c.vn)
    freqs, _ = flashattn_cuda.rope_frequencies(64)
    positions = torch.randint(0, 100000, c.rows.shape, device="cuda", dtype=torch.int32)
    qo = flashattn_cuda.append_paged(c.kn, c.vn, c.starts, c.kp, c.vp, c.table, c.seq_lens,
                                     q=c.q, freqs=freqs, positions=positions)
    check_rope(packed(qo).contiguous(), packed(c.q), positions, freqs, False)
    check_rope(packed(c.kp[pages, :, (c.rows % 16).long()]).contiguous(), packed(c.kn),
               positions, freqs, False)
    clean()


def test_append_of_unaligned_rows():
    c = append_case(d=64)
    odd = torch.zeros(36, 3, 67, device="cuda").half()[:, 1:, 1:65]
    odd.copy_(c.kn)
    freqs, _ = flashattn_cuda.rope_frequencies(64)
    flashattn_cuda.append_paged(c.kn, c.vn, c.starts, c.kp, c.vp, c.table, c.seq_lens,
                                freqs=freqs)
    want = c.kp.clone()
    c.kp[c.table[c.seq, (c.rows // 16).long()].long(), :, (c.rows % 16).long()] = 0
    flashattn_cuda.append_paged(odd, c.vn, c.starts, c.kp, c.vp, c.table, c.seq_lens,
                                freqs=freqs)
    assert torch.equal(c.kp.view(torch.int16), want.view(torch.int16))
    clean()


def test_append_stores_nothing_outside():
    """Tokens before row 0, past the table's capacity, of no sequence, and of
    a page that is none: not stored, and only the last is an error."""
    c = append_case(news=[3, 4], lens=[2, 32])
    kp, vp = c.kp.clone(), c.vp.clone()
    starts = torch.tensor([0, 3, 6], device="cuda", dtype=torch.int32)
    lens = torch.tensor([2, 34], device="cuda", dtype=torch.int32)  # capacity 32
    c.kp.zero_()
    c.vp.zero_()
    flashattn_cuda.append_paged(c.kn, c.vn, starts, c.kp, c.vp, c.table, lens)
    clean()
    stored = c.kp.abs().sum((1, 3)).nonzero().tolist()
    assert sorted(stored) == sorted([[int(c.table[0, 0]), 0], [int(c.table[0, 0]), 1],
                                     [int(c.table[1, 1]), 15]])
    table = c.table.clone()
    table[0, 0] = -1
    c.kp.copy_(kp)
    c.vp.copy_(vp)
    flashattn_cuda.append_paged(c.kn[:3], c.vn[:3], starts[:2], c.kp, c.vp, table[:1], lens[:1])
    assert flashattn_cuda.take_device_error() == 4
    assert torch.equal(c.kp.view(torch.int16), kp.view(torch.int16))
    assert torch.equal(c.vp.view(torch.int16), vp.view(torch.int16))
    clean()


def test_append_then_attend_reads_what_was_stored():
    c = append_case(d=128, h=8, news=[1, 40, 130], lens=[300, 40, 200], page=32)
    freqs, _ = flashattn_cuda.rope_frequencies(128)
    q = flashattn_cuda.append_paged(c.kn, c.vn, c.starts, c.kp, c.vp, c.table, c.seq_lens,
                                    q=c.q, freqs=freqs)
    lo = 0
    for b, n in enumerate(c.news):  # the oracle's own copy of the rows
        k, _ = flashattn_cuda.rope(packed(c.kn[lo:lo + n]), None, c.rows[lo:lo + n], freqs)
        c.k[b][c.lens[b] - n:] = k[0].transpose(0, 1)
        c.v[b][c.lens[b] - n:] = c.vn[lo:lo + n]
        lo += n
    c.q = q
    check_attention(c, attend(c), 128 ** -0.5)
    clean()


# ----------------------------------------------------------------- refusals
def test_refusals():
    c = append_case()
    freqs, _ = flashattn_cuda.rope_frequencies(64)
    good = dict(q=c.q, starts=c.starts, k_pages=c.kp, v_pages=c.vp, page_table=c.table,
                seq_lens=c.seq_lens, scale=0.125)

    def attend_refuses(match, **kw):
        with pytest.raises(RuntimeError, match=match):
            flashattn_cuda.attend_paged(**{**good, **kw})

    attend_refuses("CUDA", q=c.q.cpu())
    attend_refuses("fp16 or bf16", q=c.q.float())
    attend_refuses("3-D", q=c.q[None])
    attend_refuses("same dtype", q=c.q.bfloat16())
    attend_refuses("same head_dim", q=torch.zeros(36, 6, 128, device="cuda").half())
    attend_refuses("identical shapes", v_pages=c.vp[1:])
    attend_refuses("head_dim", q=c.q[..., :32], k_pages=c.kp[..., :32], v_pages=c.vp[..., :32])
    attend_refuses("multiple of 8 rows", k_pages=c.kp[:, :, :12], v_pages=c.vp[:, :, :12])
    attend_refuses("starts must be 1-D", starts=c.starts[:-1])
    attend_refuses("starts must be int32", starts=c.starts.long())
    attend_refuses("seq_lens must be int32", seq_lens=c.seq_lens.long())
    attend_refuses("seq_lens must be 1-D", seq_lens=c.seq_lens[None])
    attend_refuses("page_table must be", page_table=c.table[:2])
    attend_refuses("page_table must be", page_table=c.table.T.contiguous().T)
    attend_refuses("multiple \\(at most 128 times\\)", q=c.q[:, :5])
    attend_refuses("finite", scale=math.nan)
    attend_refuses("16-byte aligned", q=torch.zeros(36, 6, 68, device="cuda").half()[..., 4:])
    attend_refuses("contiguous along head_dim", q=c.q.transpose(1, 2).contiguous().transpose(1, 2))

    add = dict(k_new=c.kn, v_new=c.vn, starts=c.starts, k_pages=c.kp, v_pages=c.vp,
               page_table=c.table, seq_lens=c.seq_lens)

    def append_refuses(match, **kw):
        with pytest.raises(RuntimeError, match=match):
            flashattn_cuda.append_paged(**{**add, **kw})

    append_refuses("k_new and v_new must agree", v_new=c.vn[:3])
    append_refuses("head count", k_new=c.kn[:, :1], v_new=c.vn[:, :1])
    append_refuses("freqs must be given", q=c.q)
    append_refuses("q must be", q=c.q[:3], freqs=freqs)
    append_refuses("float64", q=c.q, freqs=freqs.float())
    append_refuses("positions must be", freqs=freqs, positions=c.rows[:3])
    append_refuses("amplitude", freqs=freqs, amplitude=math.inf)
    clean()


@pytest.mark.parametrize("kw", [dict(), dict(page_rows=24, heads=8, kv_heads=8, dim=128, steps=6)])
def test_server_loop_matches_whole_sequences(kw):
    """paged_serving.py: chunks and single tokens through pages, against rope()
    and prefill(). Both sides round the attention's output to bf16 and carry it
    through two products: a relative difference of a few 2^-8 at most."""
    import paged_serving

    assert paged_serving.main(**kw) <= 4 * 2.0 ** -8


def test_groups_that_share_the_keys_of_one_tile():
    """At head_dim 64 an item of one query tile has its key tiles split between
    two softmax groups: odd and even counts, rows that one group's tiles show
    nothing, parts of long items."""
    for news, lens in (([20], [129]), ([20], [385]), ([128], [128]), ([100, 3], [612, 1025]),
                       ([40], [30]), ([17], [30000]), ([128, 128], [257, 20000])):
        for dtype in (F16, BF16):
            c = Paged(news, lens, 2, 2, 64, 64, dtype, seed=len(news) + news[0])
            for causal in (True, False):
                out, lse = attend(c, causal=causal, return_lse=True)
                check_attention(c, out, 0.125, causal, lse)
    # a wide group: one token is a tile's worth of rows
    c = Paged([1, 1, 1], [700, 5000, 90], 40, 2, 64, 16, F16, seed=1)
    check_attention(c, attend(c), 0.125)
    clean()


@pytest.mark.parametrize("h,h_kv", [(128, 1), (100, 1), (66, 2), (17, 1)])
def test_wide_groups(h, h_kv):
    for d, news, lens in ((64, [1, 3], [300, 77]), (128, [2, 1], [700, 33])):
        c = Paged(news, lens, h, h_kv, d, 32, BF16, seed=h)
        check_attention(c, attend(c), d ** -0.5)
    clean()


def test_special_values_in_the_cache():
    """A NaN or an infinity of a row that a token sees reaches it; one past what
    the sequence holds, or in another sequence, does not."""
    for news in ([1, 1], [40, 3]):
        for d in (64, 128):
            c = Paged(news, [300, 200], 4, 2, d, 16, F16, seed=d)
            clean_out = attend(c, causal=False)
            c.kp[c.table[0, 7].long(), 0, 3, 5] = float("nan")
            out = attend(c, causal=False)
            n = news[0]
            assert out[:n, :2].isnan().all()
            assert torch.equal(out[:n, 2:], clean_out[:n, 2:])
            assert torch.equal(out[n:], clean_out[n:])
            c.kp[c.table[0, 7].long(), 0, 3, 5] = 0
            c.vp[c.table[0, 7].long(), 1, 3, 5] = float("inf")
            out = attend(c, causal=False)
            assert (out[:n, 2:, 5] == float("inf")).all()
            assert out[:n, :2].isfinite().all() and torch.equal(out[n:], clean_out[n:])
    clean()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("n", [1, 40])
def test_small_probabilities_keep_their_precision(dtype, n):
    """One row far above all others, whose values are zero: the result is the
    others' weights alone, about e^-13 each, below fp16's normal numbers."""
    for d in (64, 128):
        c = Paged([n], [500], 4, 2, d, 16, dtype)
        c.q.zero_()[..., 0] = 1
        for pages, rows in ((c.kp, c.k[0]), (c.vp, c.v[0])):
            rows.zero_()
            rows[1:, :, 0] = -13 if rows is c.k[0] else 1
            pages.zero_()
            for r0 in range(0, 500, 16):
                m = min(16, 500 - r0)
                pages[c.table[0, r0 // 16].long(), :, :m] = rows[r0:r0 + m].transpose(0, 1)
        out = flashattn_cuda.attend_paged(c.q, c.starts, c.kp, c.vp, c.table, c.seq_lens, 1.0)
        check_attention(c, out, 1.0)
    clean()


@pytest.mark.parametrize("n", [1, 50])
def test_calls_in_a_row_wait_for_one_another(n):
    """A chain in which every call reads what the one before it wrote (rows
    appended, queries made from the last output): the same bits with and
    without a synchronisation after each."""
    h, h_kv, d, steps, b = 8, 2, 64, 40, 3
    freqs, _ = flashattn_cuda.rope_frequencies(d)
    torch.manual_seed(n)
    first = torch.randn(b * n, h + 2 * h_kv, d, device="cuda").half()
    starts = torch.arange(0, b * n + 1, n, device="cuda", dtype=torch.int32)
    pages = steps * n // 16 + 1
    table = torch.randperm(b * pages, device="cuda", dtype=torch.int32).view(b, pages)

    def chain(wait):
        kp = torch.zeros(b * pages, h_kv, 16, d, device="cuda").half()
        vp = torch.zeros_like(kp)
        x, outs = first, []
        lens = torch.zeros(b, device="cuda", dtype=torch.int32)
        for _ in range(steps):
            lens += n
            q = flashattn_cuda.append_paged(x[:, h:h + h_kv], x[:, h + h_kv:], starts, kp, vp,
                                            table, lens, q=x[:, :h], freqs=freqs)
            wait()
            o = flashattn_cuda.attend_paged(q, starts, kp, vp, table, lens, 0.125)
            wait()
            o = flashattn_cuda.attend_paged(o * 4, starts, kp, vp, table, lens, 0.125)
            wait()
            x = (x * 0.5 + torch.cat((o, o[:, :2 * h_kv]), 1)).clamp(-3, 3)  # stays finite
            outs.append(o)
        torch.cuda.synchronize()
        return torch.stack(outs), kp, vp

    want = chain(torch.cuda.synchronize)
    assert want[0].isfinite().all()
    for _ in range(3):
        for a, c in zip(chain(lambda: None), want):
            assert torch.equal(a, c)
    clean()
