"""Paged caches on the GPU: the plan of a batch (exact), the write of keys and values (exact) and the
attention of single tokens against a plain implementation in 64 bits (tests/ops_oracle.py)."""

import pytest
import torch

import ops_oracle as oracle
from causal_conv1d_triton.paged import paged_attention, paged_cache_write, paged_plan

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, HF, F = torch.bfloat16, torch.float16, torch.float32


# ------------------------------------------------------------------------------------------ plan


def check_plan(cached, new, tables, free, num_free, ps, N):
    i32 = lambda t: torch.as_tensor(t).to(torch.int32)  # noqa: E731
    cached, new, tables, free = map(i32, (cached, new, tables, free))
    want = oracle.plan(cached, new, tables, free, num_free, ps, N)
    dev = tables.to(DEV)
    got = paged_plan(cached.to(DEV), new.to(DEV), dev, free.to(DEV),
                     torch.tensor([num_free], dtype=torch.int32, device=DEV), ps, N)
    for k, v in got._asdict().items():
        assert torch.equal(v.cpu().long(), want[k]), k
    assert torch.equal(dev.cpu().long(), want["tables"])
    return got


def requests(seed, R, most, new_most, ps, spare=64, slack=0):
    g = torch.Generator().manual_seed(seed)
    cached = torch.randint(0, most + 1, (R,), generator=g)
    new = torch.randint(0, new_most + 1, (R,), generator=g)
    have = (cached + ps - 1) // ps
    M = max(1, int(((cached + new + ps - 1) // ps).max()) - slack)
    total = int(have.sum())
    pages = torch.randperm(total + spare, generator=g)
    tables = torch.full((R, M), -1)
    at = 0
    for r in range(R):
        n = min(int(have[r]), M)
        tables[r, :n] = pages[at:at + n]
        at += int(have[r])
    return cached, new, tables, pages[total:]


@pytest.mark.parametrize("R", [1, 2, 15, 64, 255, 256, 257, 1024, 1025, 3000])
@pytest.mark.parametrize("ps", [1, 16, 7])
def test_plan(R, ps):
    cached, new, tables, free = requests(R, R, 40, 12, ps, spare=R * 13)
    N = int(new.sum())
    for extra in (0, 5, 1500):
        check_plan(cached, new, tables, free, len(free), ps, N + extra)


def test_plan_of_decode_and_of_long_prompts():
    cached, _, tables, free = requests(1, 33, 100, 1, 16)
    check_plan(cached, torch.ones(33), torch.cat([tables, tables[:, :1]], 1), free, len(free), 16, 40)
    check_plan([0, 5, 0], [5000, 0, 3000], torch.full((3, 400), -1), torch.arange(600), 600, 16, 8192)


@pytest.mark.parametrize("free", [0, 1, 7, 60])
def test_plan_short_of_pages_or_table_rows(free):
    """Requests are refused from the first that the free list cannot serve; those that need no page,
    and those before, go on; a row of the table that is too short refuses its own request alone."""
    cached, new, tables, pages = requests(2, 50, 60, 20, 8, spare=400)
    check_plan(cached, new, tables, pages, free, 8, int(new.sum()) + 3)
    cached, new, tables, pages = requests(3, 50, 60, 20, 8, spare=400, slack=3)
    check_plan(cached, new, tables, pages, free, 8, int(new.sum()) + 3)


def test_plan_edges():
    check_plan([], [], torch.empty(0, 4), [3, 4], 2, 16, 5)  # no requests
    check_plan([3], [0], [[9, -1]], [3, 4], 2, 16, 0)  # no tokens, no places
    check_plan([-4, 2], [-1, 3], [[-1], [8]], [3], 1, 16, 6)  # negative lengths count as zero
    check_plan([0], [4], [[-1]], [3, 4], 50, 16, 4)  # more free than listed
    check_plan([0], [4], [[-1]], [3, 4], -3, 16, 4)
    check_plan([20], [4], [[-1, -1]], [3, 4], 2, 16, 4)  # a cached page that is not there
    check_plan([0], [4], [[-1]], [], 0, 16, 4)
    check_plan([0, 0], [9, 9], [[-1], [-1]], [3, 4], 2, 16, 11)  # fewer places than tokens
    check_plan([2 ** 31 - 1, 0], [2 ** 31 - 2, 1], [[-1], [-1]], [3, 4], 2, 16, 8)  # the sums' limit


def test_plan_leaves_cached_pages_and_strided_tables():
    cached, new, tables, free = requests(4, 20, 60, 20, 8, spare=400)
    wide = torch.full((20, tables.shape[1] + 5), 77, dtype=torch.int32, device=DEV)
    view = wide[:, 2:2 + tables.shape[1]]
    view.copy_(tables)
    want = oracle.plan(cached, new, tables, free, len(free), 8, 100)
    paged_plan(cached.int().to(DEV), new.int().to(DEV), view, free.int().to(DEV),
               torch.tensor([len(free)], dtype=torch.int32, device=DEV), 8, 100)
    assert torch.equal(view.cpu().long(), want["tables"])
    assert (wide[:, :2] == 77).all() and (wide[:, 2 + tables.shape[1]:] == 77).all()


# ----------------------------------------------------------------------------------------- write


@pytest.mark.parametrize("dtype", [BF, HF, F])
@pytest.mark.parametrize("H,Dh", [(1, 1), (2, 8), (8, 128), (3, 20), (5, 33), (16, 256)])
def test_write(dtype, H, Dh):
    g = torch.Generator().manual_seed(H)
    N, P, ps = 37, 9, 7
    qkv = torch.randn(N, 3 * H, Dh, generator=g).to(dtype)
    kc, vc = (torch.randn(P, ps, H, Dh, generator=g).to(dtype) for _ in range(2))
    slots = torch.randperm(P * ps, generator=g)[:N]
    slots[::5] = -1
    slots[3], slots[4] = P * ps, 2 ** 40
    wk, wv = kc.clone(), vc.clone()
    for t, s in enumerate(slots.tolist()):
        if 0 <= s < P * ps:
            wk[s // ps, s % ps], wv[s // ps, s % ps] = qkv[t, H:2 * H], qkv[t, 2 * H:]
    d = qkv.to(DEV)
    a, b = kc.to(DEV), vc.to(DEV)
    paged_cache_write(d[:, H:2 * H], d[:, 2 * H:], a, b, slots.to(DEV))
    assert torch.equal(a.cpu(), wk) and torch.equal(b.cpu(), wv)
    # keys and values in one tensor, heads before tokens, an odd start; slots as int32
    both = torch.zeros(P, 2, H, ps, Dh + 3, dtype=dtype, device=DEV)
    a, b = (both[:, j].transpose(1, 2)[..., 1:1 + Dh] for j in (0, 1))
    a.copy_(kc)
    b.copy_(vc)
    paged_cache_write(d[:, H:2 * H], d[:, 2 * H:], a, b, slots.clamp(max=P * ps).int().to(DEV))
    assert torch.equal(a.cpu(), wk) and torch.equal(b.cpu(), wv)
    assert not both[..., 0].any() and not both[..., 1 + Dh:].any()


def test_write_nothing():
    kc = torch.zeros(2, 4, 2, 8, device=DEV)
    z = torch.zeros(0, 2, 8, device=DEV)
    paged_cache_write(z, z, kc, kc.clone(), torch.zeros(0, dtype=torch.int64, device=DEV))
    assert not kc.any()


# ------------------------------------------------------------------------------------- attention


def caches(seed, lens, H, Dh, ps, dtype, extra=2):
    g = torch.Generator().manual_seed(seed)
    have = [-(-max(0, n) // ps) for n in lens]
    P, M = sum(have) + extra, max(have + [1]) + 1
    order = torch.randperm(P, generator=g)
    tables, at = torch.full((len(lens), M), -1, dtype=torch.int32), 0
    for r, n in enumerate(have):
        tables[r, :n] = order[at:at + n]
        at += n
    kc, vc = (torch.randn(P, ps, H, Dh, generator=g).to(dtype) for _ in range(2))
    return kc, vc, tables


def check_attn(seed, lens, Hq, H, Dh, ps, dtype, window=None, scale=None, amp=1.0, **kw):
    kc, vc, tables = caches(seed, lens, H, Dh, ps, dtype)
    g = torch.Generator().manual_seed(seed + 1)
    q = (amp * torch.randn(len(lens), Hq, Dh, generator=g)).to(dtype)
    lens = torch.tensor(lens, dtype=torch.int32)
    out, lse = paged_attention(q.to(DEV), kc.to(DEV), vc.to(DEV), tables.to(DEV), lens.to(DEV), scale,
                               window, return_lse=True, **kw)
    want, want_lse = oracle.attention(q, kc, vc, tables, lens, scale, window)
    oracle.assert_close(out, want, "out")
    finite = torch.isfinite(want_lse[0])
    assert torch.equal(torch.isfinite(lse.cpu()), finite)
    oracle.assert_close(lse.cpu()[finite], (want_lse[0][finite], want_lse[1][finite]), "lse")
    assert (lse.cpu()[~finite] == float("-inf")).all() and not out.cpu()[~finite].any()


LENS = [1, 0, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 100, 127, 128, 129, 255, 256, 257, 300, 513]


@pytest.mark.parametrize("dtype", [BF, HF, F])
@pytest.mark.parametrize("ps", [1, 3, 4, 16, 20, 32, 64, 100, 256])
def test_attention_lengths_and_pages(dtype, ps):
    check_attn(ps, LENS, 8, 2, 64, ps, dtype)


@pytest.mark.parametrize("dtype", [BF, HF, F])
@pytest.mark.parametrize("Dh", [8, 16, 24, 32, 40, 64, 72, 80, 96, 104, 112, 120, 128, 136, 160, 192,
                                200, 248, 256])
def test_attention_head_sizes(dtype, Dh):
    check_attn(Dh, [70, 5, 0, 161], 4, 2, Dh, 16, dtype)


@pytest.mark.parametrize("Hq,H", [(1, 1), (2, 1), (5, 5), (6, 2), (15, 1), (16, 1), (17, 1), (32, 1),
                                  (33, 3), (40, 1), (64, 8), (71, 1), (24, 8)])
@pytest.mark.parametrize("dtype", [BF, F])
def test_attention_heads(Hq, H, dtype):
    check_attn(Hq, [90, 300, 1], Hq, H, 64, 16, dtype)


@pytest.mark.parametrize("window", [1, 2, 16, 31, 32, 33, 100, 512, 100000])
@pytest.mark.parametrize("ps", [16, 5])
def test_attention_window(window, ps):
    check_attn(window, LENS, 4, 1, 128, ps, BF, window=window)
    check_attn(window, LENS[::3], 4, 1, 128, ps, F, window=window)


@pytest.mark.parametrize("window", [2 ** 31 - 32, 2 ** 31 - 1, 2 ** 31, 2 ** 63 - 31, 2 ** 63 - 1])
def test_attention_window_past_every_length(window):
    """Rows that are split, with a window that reaches past every length: the bits of no window."""
    lens = [1, 0, 5000, 129]
    kc, vc, tables = caches(8, lens, 2, 64, 16, BF)
    q = torch.randn(4, 4, 64, generator=torch.Generator().manual_seed(2)).to(BF).to(DEV)
    args = (q, kc.to(DEV), vc.to(DEV), tables.to(DEV), torch.tensor(lens, device=DEV))
    want = paged_attention(*args, return_lse=True)
    got = paged_attention(*args, window=window, return_lse=True)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("window", [1, 20, 31, 100, 700])
@pytest.mark.parametrize("cut", ["table", "max_seq_len"])
def test_attention_window_of_lengths_past_the_end(window, cut):
    """The window is the last of the length, not of what the table or max_seq_len leaves of it: a row sees
    [length - window, end), which is nothing where the window starts past the end."""
    end, ps = 480, 16
    lens = [n for o in (-1, 0, 1, 10, 19, 20, 21, 99, 100, 101, 699, 701, 2 ** 31 - 1 - end) for n in [end + o]]
    kc, vc, tables = caches(9, [end] * len(lens), 2, 64, ps, BF)
    kw = dict(window=window)
    if cut == "table":
        tables = tables[:, :end // ps].contiguous()
    else:
        kw["max_seq_len"] = end
    q = torch.randn(len(lens), 4, 64, generator=torch.Generator().manual_seed(2)).to(BF)
    out, lse = paged_attention(q.to(DEV), kc.to(DEV), vc.to(DEV), tables.to(DEV),
                               torch.tensor(lens, device=DEV), return_lse=True, **kw)
    for r, n in enumerate(lens):
        stop = min(n, end)
        start = max(0, n - window)
        if start >= stop:
            assert not out[r].any() and (lse[r] == float("-inf")).all(), n
            continue
        one = slice(r, r + 1)
        want, want_lse = oracle.attention(q[one], kc, vc, tables[one], torch.tensor([stop]), window=stop - start)
        oracle.assert_close(out[one], want, n)
        oracle.assert_close(lse[one], want_lse, n)


@pytest.mark.parametrize("dtype", [BF, HF, F])
def test_attention_long(dtype):
    """Lengths that are split over workgroups and joined, beside short ones."""
    check_attn(1, [5000, 3, 0, 9001], 8, 2, 128, 16, dtype)
    check_attn(2, [12345], 4, 1, 64, 64, dtype, max_seq_len=13000)
    check_attn(3, [7000, 100, 6999], 16, 1, 256, 32, dtype, window=4000)


@pytest.mark.parametrize("dtype", [BF, HF, F])
@pytest.mark.parametrize("Dh", [8, 16, 40, 64, 72, 96, 120, 128, 136, 192, 200, 256])
def test_attention_joined_head_sizes(dtype, Dh):
    check_attn(Dh + 1, [1300, 5, 0, 131, 700], 4, 2, Dh, 16, dtype)


@pytest.mark.parametrize("R,Dh,most", [(3, 128, 400), (3, 128, 401), (3, 64, 512), (3, 64, 513), (3, 256, 200),
                                       (3, 256, 201), (127, 64, 513), (128, 64, 513), (128, 64, 1055),
                                       (128, 64, 1056)])
def test_attention_whole_and_split_rows(R, Dh, most):
    """Either side of the sizes at which rows are split over workgroups."""
    lens = [most, 0, most - 1] + [n * 37 % 140 for n in range(R - 4)] + [most] * (R > 3)
    check_attn(most, lens, 4, 2, Dh, 16, BF, max_seq_len=most)
    if R > 3:
        check_attn(most + 1, lens, 4, 2, Dh, 20, HF, window=most - 300)


def test_attention_many_rows():
    check_attn(4, [n % 97 for n in range(700)], 4, 2, 64, 16, BF)


def test_attention_scale_and_large_scores():
    check_attn(5, [200, 33], 4, 2, 64, 16, BF, scale=0.02)
    check_attn(6, [200, 33], 4, 2, 64, 16, F, amp=30.0)  # the softmax is nearly a choice
    check_attn(7, [200, 33, 0], 4, 2, 64, 16, HF, scale=0.0)


@pytest.mark.parametrize("dtype", [BF, HF, F])
@pytest.mark.parametrize("low", [16.4, 20.4, 24.4, 25.3, 27.4])
def test_attention_beside_a_dominant_position(low, dtype):
    """Positions that take most of the weight and have values of zero, one in each wave, beside a tail at
    2^-low: the result is the tail's. Room: what the pieces of a weight leave out (2^-16 of it in bf16, 2^-22 of it or
    2^-32 of the largest in fp16, nothing in fp32) and a score's rounding, 2^-22 of 32 at most in its exponent."""
    ps, n, Dh = 16, 400, 64
    g = torch.Generator().manual_seed(int(low))
    kc, vc = torch.zeros(25, ps, 1, Dh).to(dtype), torch.zeros(25, ps, 1, Dh).to(dtype)
    score = -low + (torch.rand(n, generator=g) - 0.5) / 8
    sinks = torch.zeros(n, dtype=torch.bool)
    sinks[[0, 33, 70, 100]] = True
    score[sinks] = 0
    kc.view(n, Dh)[:, 0] = score.to(dtype)
    vc.view(n, Dh)[:] = (256 + 700 * torch.rand(n, Dh, generator=g)).to(dtype)
    vc.view(n, Dh)[sinks] = 0
    q = torch.zeros(1, 4, Dh, dtype=dtype)
    q[..., 0] = 1
    ln2 = 0.6931471805599453
    tables = torch.arange(25, dtype=torch.int32)[None]
    out, lse = paged_attention(q.to(DEV), kc.to(DEV), vc.to(DEV), tables.to(DEV), torch.tensor([n], device=DEV),
                               softmax_scale=ln2, return_lse=True)
    w = torch.exp2(kc.view(n, Dh)[:, 0].double())
    v = vc.view(n, Dh).double()
    lost = {BF: 2.0 ** -16 * w, HF: torch.clamp(2.0 ** -22 * w, min=2.0 ** -32), F: 0 * w}[dtype]
    want = (w @ v / w.sum()).expand(1, 4, Dh)
    room = ((lost + 2.0 ** -17 * w) @ v / w.sum()).expand(1, 4, Dh)
    oracle.assert_close(out, (want, room))
    oracle.assert_close(lse, (torch.log(w.sum()).expand(1, 4), torch.full((1, 4), 2.0 ** -20, dtype=torch.float64)))


@pytest.mark.parametrize("dtype", [BF, HF, F])
def test_attention_weights_keep_their_bits(dtype):
    """Six positions whose weighted values nearly cancel, so that the result shows how far the weights are off.
    Room, of the sum of the products' sizes: a score's rounding in its exponent (2 * 2^-23), the exponential's,
    the pieces' (2^-22 in fp16), the sums' and the division's, together below 2^-20."""
    R, n, Dh, ps = 40, 6, 64, 16
    g = torch.Generator().manual_seed(5)
    score = -torch.randint(0, 65, (R, n), generator=g) / 32
    w = torch.exp2(score.double())
    v = ((0.5 + 1.5 * torch.rand(R, n, Dh, generator=g)) * torch.sign(torch.randn(R, n, Dh, generator=g))).to(dtype)
    for j in (4, 5):  # the last two take back what the others sum to
        v[:, j] = 0
        v[:, j] = (-(w[:, :, None] * v.double())[:, :j].sum(1) / w[:, j, None]).to(dtype)
    kc, vc = torch.zeros(R, ps, 1, Dh).to(dtype), torch.zeros(R, ps, 1, Dh).to(dtype)
    kc[:, :n, 0, 0], vc[:, :n, 0] = score.to(dtype), v
    q = torch.zeros(R, 2, Dh, dtype=dtype)
    q[..., 0] = 1
    out = paged_attention(q.to(DEV), kc.to(DEV), vc.to(DEV), torch.arange(R, dtype=torch.int32, device=DEV)[:, None],
                          torch.full((R,), n, device=DEV), softmax_scale=0.6931471805599453)
    p = (w / w.sum(1, keepdim=True))[:, :, None]
    want, size = (p * v.double()).sum(1), (p * v.double().abs()).sum(1)
    oracle.assert_close(out, (want[:, None].expand(R, 2, Dh), 2.0 ** -20 * size[:, None].expand(R, 2, Dh)))


@pytest.mark.parametrize("dtype", [BF, F])
def test_attention_strides(dtype):
    """Heads before tokens in one tensor of keys and values, odd starts, a strided table and query."""
    H, Dh, ps, lens = 2, 64, 16, [100, 7, 0, 49]
    kc, vc, tables = caches(1, lens, H, Dh, ps, dtype)
    q = torch.randn(4, 6, Dh, generator=torch.Generator().manual_seed(2)).to(dtype)
    both = torch.full((kc.shape[0], 2, H, ps, Dh + 3), float("nan"), dtype=dtype, device=DEV)
    a, b = (both[:, j].transpose(1, 2)[..., 1:1 + Dh] for j in (0, 1))
    a.copy_(kc)
    b.copy_(vc)
    wide_t = torch.full((4, tables.shape[1] + 3), 10 ** 6, dtype=torch.int32, device=DEV)
    wide_t[:, 1:1 + tables.shape[1]] = tables.to(DEV)
    wide_q = torch.zeros(4, 9, Dh + 1, dtype=dtype, device=DEV)
    wide_q[:, 2:8, 1:] = q.to(DEV)
    out = paged_attention(wide_q[:, 2:8, 1:], a, b, wide_t[:, 1:1 + tables.shape[1]],
                          torch.tensor(lens, device=DEV))
    want, _ = oracle.attention(q, kc, vc, tables, torch.tensor(lens))
    oracle.assert_close(out, want)


def test_attention_of_a_prompt():
    """Several rows of one request, each up to its own position; padding rows are empty."""
    kc, vc, tables = caches(3, [40, 90], 2, 64, 16, BF)
    ids = torch.tensor([0] * 40 + [1] * 10 + [-1, 2, -7], dtype=torch.int32)
    lens = torch.tensor(list(range(1, 41)) + list(range(81, 91)) + [0, 5, 9], dtype=torch.int32)
    q = torch.randn(53, 4, 64, generator=torch.Generator().manual_seed(2)).to(BF)
    out = paged_attention(q.to(DEV), kc.to(DEV), vc.to(DEV), tables.to(DEV), lens.to(DEV),
                          request_ids=ids.to(DEV))
    want, _ = oracle.attention(q, kc, vc, tables, lens, ids=ids)
    oracle.assert_close(out, want)
    assert not out[-3:].any()


def test_attention_reads_no_other_row():
    """NaN and infinities in every cache row that a request does not see, its page's end included."""
    lens, ps = [33, 1, 70, 0], 16
    for dtype, window in ((BF, None), (BF, 20), (F, None), (F, 20)):
        kc, vc, tables = caches(5, lens, 2, 64, ps, dtype)
        q = torch.randn(4, 4, 64, generator=torch.Generator().manual_seed(2)).to(dtype)
        seen = torch.zeros(kc.shape[:2], dtype=torch.bool)
        for r, n in enumerate(lens):
            for p in range(max(0, n - window) if window else 0, n):
                seen[tables[r, p // ps], p % ps] = True
        args = (tables.to(DEV), torch.tensor(lens, device=DEV), None, window)
        clean = paged_attention(q.to(DEV), kc.to(DEV), vc.to(DEV), *args)
        for bad in (float("nan"), float("inf"), float("-inf"), torch.finfo(dtype).min):
            k2, v2 = kc.clone(), vc.clone()
            k2[~seen], v2[~seen] = bad, bad
            assert torch.equal(paged_attention(q.to(DEV), k2.to(DEV), v2.to(DEV), *args), clean), bad


def test_attention_pages_outside_the_cache():
    kc, vc, tables = caches(6, [100, 64], 2, 64, 16, BF)
    tables[0, 2], tables[0, 4], tables[1, :] = -1, kc.shape[0], 2 ** 31 - 1
    q = torch.randn(2, 4, 64, generator=torch.Generator().manual_seed(2)).to(BF)
    lens = torch.tensor([100, 64])
    out, lse = paged_attention(q.to(DEV), kc.to(DEV), vc.to(DEV), tables.to(DEV), lens.to(DEV),
                               return_lse=True)
    want, want_lse = oracle.attention(q, kc, vc, tables, lens)
    oracle.assert_close(out, want)
    assert not out[1].any() and (lse[1] == float("-inf")).all()
    # a length past the table's end stops there
    out = paged_attention(q.to(DEV), kc.to(DEV), vc.to(DEV), tables[:, :2].to(DEV), lens.to(DEV))
    want, _ = oracle.attention(q, kc, vc, tables[:, :2], lens)
    oracle.assert_close(out, want)


@pytest.mark.parametrize("dtype", [BF, F])
def test_attention_of_scores_without_a_finite_maximum(dtype):
    """Keys of -infinity give weights of zero; where all are, the row is empty."""
    kc, vc, tables = caches(7, [40, 40], 1, 64, 16, dtype)
    q = torch.rand(2, 1, 64, generator=torch.Generator().manual_seed(2)).to(dtype) + 0.5
    kc[tables[0, 0].item(), 3:9] = float("-inf")
    for p in range(3):
        kc[tables[1, p].item()] = float("-inf")
    lens = torch.tensor([40, 40])
    out, lse = paged_attention(q.to(DEV), kc.to(DEV), vc.to(DEV), tables.to(DEV), lens.to(DEV),
                               return_lse=True)
    keep = torch.tensor([p for p in range(40) if not 3 <= p < 9])
    k = kc[tables[0, keep // 16].long(), keep % 16, 0].double()
    v = vc[tables[0, keep // 16].long(), keep % 16, 0].double()
    w = torch.softmax(k @ q[0, 0].double() / 8, 0)
    oracle.assert_close(out[0, 0], (w @ v, 2.0 ** -14 * (w @ v.abs())))
    assert not out[1].any() and lse[1, 0] == float("-inf")


@pytest.mark.parametrize("dtype", [BF, HF, F])
@pytest.mark.parametrize("Dh", [64, 40, 256])
@pytest.mark.parametrize("lens", [[40, 1, 33], [3000, 7, 1500]])
def test_attention_of_infinite_values(dtype, Dh, lens):
    """An infinite value that a row sees is its element's result, two of both signs or a NaN make it no number;
    the other elements, heads and rows keep their bits."""
    kc, vc, tables = caches(11, lens, 2, Dh, 16, dtype)
    q = (0.3 * torch.randn(len(lens), 4, Dh, generator=torch.Generator().manual_seed(2))).to(dtype)
    args = (q.to(DEV), kc.to(DEV))
    rest = (tables.to(DEV), torch.tensor(lens, device=DEV))
    clean = paged_attention(*args, vc.to(DEV), *rest).cpu()
    want = clean.float()
    inf, nan = float("inf"), float("nan")
    bad = vc.clone()
    for r, p, h, d, v, res in ((0, 0, 0, 3, inf, inf), (0, lens[0] - 1, 0, 7, -inf, -inf), (0, 5, 1, 8, inf, nan),
                               (0, 37, 1, 8, -inf, nan), (0, 20, 1, 11, nan, nan), (1, 0, 1, 0, -inf, -inf),
                               (2, 30, 0, Dh - 1, inf, inf), (2, 31, 0, Dh - 1, inf, inf),
                               (2, 32, 0, 2, inf, nan), (2, 9, 0, 2, nan, nan)):
        bad[tables[r, p // 16], p % 16, h, d] = v
        want[r, 2 * h:2 * h + 2, d] = res
    got = paged_attention(*args, bad.to(DEV), *rest).cpu().float()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(got.nan_to_num(123.0, inf, -inf), want.nan_to_num(123.0, inf, -inf))


def test_attention_offsets_past_32_bits():
    """A cache of more than 2^32 elements, its last pages in use."""
    ps, H, Dh = 64, 8, 128
    P = (2 ** 32) // (ps * H * Dh) + 8
    k = torch.zeros(P, ps, H, Dh, dtype=BF, device=DEV)
    g = torch.Generator().manual_seed(1)
    pages = torch.tensor([[P - 1, P - 3, 5]], dtype=torch.int32)
    rows = torch.randn(3, ps, H, Dh, generator=g).to(BF)
    n = 2 * ps + 9
    slots = (pages[0].long()[:, None] * ps + torch.arange(ps)).reshape(-1)
    v = torch.zeros_like(k)
    flat = rows.reshape(-1, H, Dh).to(DEV)
    paged_cache_write(flat, flat.flip(0), k, v, slots.to(DEV))
    assert torch.equal(k[P - 1].cpu(), rows[0])
    q = torch.randn(1, 16, Dh, generator=g).to(BF)
    out = paged_attention(q.to(DEV), k, v, pages.to(DEV), torch.tensor([n], device=DEV))
    small = torch.tensor([[0, 1, 2]], dtype=torch.int32)
    want, _ = oracle.attention(q, rows, rows.reshape(-1, H, Dh).flip(0).reshape(rows.shape), small,
                               torch.tensor([n]))
    oracle.assert_close(out, want)


def test_empty_calls():
    kc = torch.zeros(2, 16, 2, 64, dtype=BF, device=DEV)
    t = torch.zeros(0, 4, dtype=torch.int32, device=DEV)
    out = paged_attention(torch.zeros(0, 4, 64, dtype=BF, device=DEV), kc, kc, t,
                          torch.zeros(0, dtype=torch.int32, device=DEV))
    assert out.shape == (0, 4, 64)
    q = torch.ones(2, 4, 64, dtype=BF, device=DEV)
    out, lse = paged_attention(q, kc, kc, torch.zeros(2, 0, dtype=torch.int32, device=DEV),
                               torch.tensor([5, 6], device=DEV), return_lse=True)
    assert not out.any() and (lse == float("-inf")).all()
    out = paged_attention(q, kc[:0], kc[:0], torch.zeros(2, 3, dtype=torch.int32, device=DEV),
                          torch.tensor([5, 6], device=DEV))
    assert not out.any()


def test_a_step_in_a_graph_on_another_stream():
    """Plan, write and attention of one step captured once and replayed over changing lengths, with
    eager work between: the eager results each time."""
    H, Dh, ps, R = 2, 64, 16, 5
    g = torch.Generator().manual_seed(1)
    kc, vc = (torch.randn(80, ps, H, Dh, generator=g).to(BF).to(DEV) for _ in range(2))
    tables = torch.randperm(80, generator=g)[:60].reshape(R, 12).int().to(DEV)
    cached = torch.tensor([0, 15, 16, 100, 31], dtype=torch.int32, device=DEV)
    ones = torch.ones_like(cached)
    free = torch.arange(60, 80, dtype=torch.int32, device=DEV)
    num = torch.tensor([20], dtype=torch.int32, device=DEV)
    qkv = torch.randn(R, 8, Dh, generator=g).to(BF).to(DEV)

    def step(kc, vc, tables):
        plan = paged_plan(cached, ones, tables, free, num, ps, 8)
        paged_cache_write(qkv[:, 4:6], qkv[:, 6:], kc, vc, plan.slot_mapping[:R])
        return paged_attention(qkv[:, :4], kc, vc, tables, plan.seq_lens)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(kc.clone(), vc.clone(), tables.clone())
    torch.cuda.current_stream().wait_stream(side)
    ck, cv, ct = kc.clone(), vc.clone(), tables.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = step(ck, cv, ct)
    for i in range(4):
        cached.copy_(torch.tensor([i, 15 + 16 * i, 16 + i, 100 - i, 31], device=DEV))
        for a, b in ((ck, kc), (cv, vc), (ct, tables)):
            a.copy_(b)
        out.fill_(9)
        graph.replay()
        torch.cuda.synchronize()
        e = [t.clone() for t in (kc, vc, tables)]
        assert torch.equal(out, step(*e)), i
        assert torch.equal(ck, e[0]) and torch.equal(cv, e[1]) and torch.equal(ct, e[2])
