"""The serving operators on the GPU against float64: the paged cache (int8 codes against the formula, read back), decode
attention against the oracle's full-sequence forward, the shared prefix, the verification of drafts.

Tolerances, from the arithmetic. fp16: P is rounded to fp16 (2^-11 relative, so at most 2^-11 max|v| in the weighted
mean) and so is the output (2^-11 |o|); 10 % on top for the float32 logits: 1.1 * 2^-10 max|v|. float32: a logit's
float32 error is at most about D 2^-24 sum|q k| / sqrt(D), 2e-4 at D = 256 and unit inputs, and scales the weights by as
much: 2e-4 max|v|, the framework's float32 tolerance."""
import numpy as np
import pytest
import torch

from first_passage_attention_b200 import FPACache, LaunchStats, first_passage_attention, first_passage_decode, verify_draft
from oracle import fpa_oracle as O

pytestmark = pytest.mark.gpu

TOL = {torch.float16: 1.1 * 2.0 ** -10, torch.float32: 2e-4}
F16, F32, I8 = torch.float16, torch.float32, torch.int8


@pytest.fixture(autouse=True)
def need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA GPU")


def quantise(x):
    """Codes, scales and values by the cache's formula, in float32 (NumPy)."""
    x = x.float().numpy()
    top = np.maximum(np.abs(x).max(-1, keepdims=True), np.float32(127 * 2.0 ** -90))
    codes = np.rint((x * np.float32(127)) / top).astype(np.int8)
    scale = (top / np.float32(127)).astype(np.float32)
    return torch.from_numpy(codes), torch.from_numpy(scale[..., 0]), torch.from_numpy(codes * scale)


def sequence(B, H, T, D, dtype, seed, walk=0.5):
    g = torch.Generator().manual_seed(seed)
    q, k, v = (torch.randn(B, H, T, D, generator=g).to(dtype) for _ in range(3))
    w = (walk * torch.randn(B, H, T, generator=g)).cumsum(-1)
    phi, psi = w + torch.randn(B, H, T, generator=g), w + torch.randn(B, H, T, generator=g)
    return q, k, v, phi, psi


def tables(lens, page, extra=3, seed=0):
    """Shuffled pages, one table row per length, -1 where a row has no page."""
    need = [-(-x // page) for x in lens]
    perm = torch.randperm(sum(need) + extra, generator=torch.Generator().manual_seed(seed)).tolist()
    rows, at = [], 0
    for x in need:
        rows.append(perm[at:at + x] + [-1] * (max(max(need), 1) - x))
        at += x
    return torch.tensor(rows, dtype=torch.int32, device="cuda"), sum(need) + extra


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def poison(cache):
    """Everything a sequence has not written is NaN (255 in the codes' bytes)."""
    for x in (cache.k, cache.v, cache.phi, cache.psi, cache.phi_min, cache.k_scale, cache.v_scale):
        if x is not None:
            x.fill_(255 if x.dtype == torch.uint8 else float("nan"))


def fill(cache, table, lens, k, v, phi, psi):
    cache.append(k.cuda(), v.cuda(), phi.cuda(), psi.cuda(), table, i32([0] * len(lens)), i32(lens))


def expected(q, k, v, phi, psi, beta, n, storage):
    """Rows T - n .. T - 1 of one sequence ([H, T, ...] tensors) in float64, on the values that the cache holds."""
    if storage == I8:
        k, v = quantise(k)[2], quantise(v)[2]
    q, k, v, phi, psi, beta = (x.double().cuda() for x in (q, k, v, phi, psi, beta))
    T, out = k.shape[1], []
    for t in range(T - n, T):
        least = phi[:, 1:t + 1].flip(-1).cummin(-1).values.flip(-1)  # min over s < u <= t, for s < t
        z = (k[:, :t + 1] @ q[:, t, :, None])[..., 0] / q.shape[-1] ** 0.5
        z[:, :t] += beta[:, None] * (least - psi[:, :t]).clamp(max=0)
        out.append((z.softmax(-1)[:, None] @ v[:, :t + 1])[:, 0])
    return torch.stack(out, 1).cpu()


def test_expected_rows_are_the_oracles():
    q, k, v, phi, psi = sequence(1, 2, 70, 32, F32, seed=20)
    beta = torch.tensor([0.7, -0.4])
    want = O.forward(*(x.double().numpy() for x in (q, k, v, phi, psi)), beta.double().numpy())[0][0][:, -9:]
    got = expected(q[0], k[0], v[0], phi[0], psi[0], beta, 9, None)
    assert (got - torch.from_numpy(want)).abs().max().item() <= 1e-12


def assert_close(got, want, vmax, dtype, what=""):
    err = (got.double().cpu() - want).abs().max().item()
    assert err <= TOL[dtype] * vmax, (what, err, TOL[dtype] * vmax)


# -------------------------------------------------------------------------------------------------- the cache ----

@pytest.mark.parametrize("dtype,storage", [(F16, None), (F16, I8), (F32, None), (F32, I8)])
@pytest.mark.parametrize("D,page", [(16, 32), (64, 64), (128, 128), (256, 256), (32, 64)])
def test_append_and_read(dtype, storage, D, page):
    """Two appends, the second from the middle of a page on, ragged counts; layouts of a fused projection."""
    B, H, T = 3, 3, 2 * page + 37
    _, k, v, phi, psi = sequence(B, H, T, D, dtype, seed=D)
    k[0, 0, 5] = 0  # a row of zeros: the smallest scale
    lens, first = [T, page + 1, 7], [page - 3, page, 0]
    table, n_pages = tables(lens, page)
    cache = FPACache(n_pages, H, D, page, dtype, storage)
    poison(cache)
    qkv = torch.stack([k, k, v]).permute(1, 3, 0, 2, 4).contiguous().cuda()   # [B, T, 3, H, D]
    _, kk, vv = qkv.permute(2, 0, 3, 1, 4)
    assert not kk.is_contiguous()
    ph, ps = (x.permute(2, 0, 1).contiguous().permute(1, 2, 0).cuda() for x in (phi, psi))
    cache.append(kk, vv, ph, ps, table, i32([0, 0, 0]), i32(first))
    for b in range(B):  # each sequence's rest, from where it stopped
        n = lens[b] - first[b]
        sl = slice(first[b], lens[b])
        cache.append(kk[b:b + 1, :, sl], vv[b:b + 1, :, sl], ph[b:b + 1, :, sl], ps[b:b + 1, :, sl], table[b:b + 1],
                     i32([first[b]]), i32([n]))
    cache.check()
    start = [0, 2, 1]
    got = cache.read(table, i32(start), T, i32(lens))
    for b in range(B):
        c = lens[b] - start[b]
        for x, y in zip(got[:2], (k, v)):
            y = y[b, :, start[b]:lens[b]]
            want = (quantise(y)[2] if storage == I8 else y).to(dtype)
            assert torch.equal(x[b, :, :c].cpu(), want)
            assert (x[b, :, c:] == 0).all()
        for x, y in zip(got[2:], (phi, psi)):
            assert torch.equal(x[b, :, :c].cpu(), y[b, :, start[b]:lens[b]]) and (x[b, :, c:] == 0).all()
        for i in range(-(-lens[b] // page)):
            want = phi[b, :, i * page:min((i + 1) * page, lens[b])].amin(-1)
            assert torch.equal(cache.phi_min[table[b, i]].cpu(), want), (b, i)
    if storage == I8:
        codes, scale, _ = quantise(k[0, :, :page])
        assert torch.equal(cache.k[table[0, 0]].cpu().int() - 128, codes.int())
        assert torch.equal(cache.k_scale[table[0, 0]].cpu(), scale)


def test_append_odd_layouts():
    """Rows that no 16-byte load can take: an innermost stride of two, a base off by one element."""
    B, H, n, D = 2, 2, 5, 32
    _, k, v, phi, psi = sequence(B, H, n, D, F16, seed=1)
    table, n_pages = tables([n, n], 32)
    want = FPACache(n_pages, H, D, 32, F16, I8)
    fill(want, table, [n, n], k, v, phi, psi)
    wide = torch.zeros(B, H, n, 2 * D, dtype=F16, device="cuda")
    wide[..., ::2] = k.cuda()
    off = torch.zeros(B * H * n * D + 1, dtype=F16, device="cuda")
    off[1:] = v.cuda().flatten()
    got = FPACache(n_pages, H, D, 32, F16, I8)
    got.append(wide[..., ::2], off[1:].view(B, H, n, D), phi.cuda(), psi.cuda(), table, i32([0, 0]))
    shared = FPACache(n_pages, H, D, 32, F16, I8)   # one head's keys broadcast over the heads
    shared.append(k[:, :1].cuda().expand(B, H, n, D), v.cuda(), phi.cuda(), psi.cuda(), table, i32([0, 0]))
    for name in ("k", "v", "k_scale", "v_scale", "phi", "psi", "phi_min"):
        assert torch.equal(getattr(got, name), getattr(want, name)), name
    assert torch.equal(shared.k[table[1, 0], 1, :n].cpu().int() - 128, quantise(k[1, 0])[0].int())


def test_append_takes_back_refused_tokens():
    """Writing from an earlier position drops what the sequence held from there on, the page's minimum included."""
    H, D, page = 2, 16, 32
    _, k, v, phi, psi = sequence(1, H, page, D, F32, seed=2)
    phi[..., 20:] -= 100
    table, n_pages = tables([page], page)
    cache = FPACache(n_pages, H, D, page, F32)
    fill(cache, table, [page], k, v, phi, psi)
    phi2 = phi[..., :12] + 1
    cache.append(k[:, :, :12].cuda(), v[:, :, :12].cuda(), phi2.cuda(), psi[..., :12].cuda(), table, i32([20]))
    want = torch.cat([phi[..., :20], phi2], -1).amin(-1)[0]
    assert torch.equal(cache.phi_min[table[0, 0]].cpu(), want)


def test_extreme_rows():
    """Rows of the smallest and largest fp16 magnitudes beside ordinary ones: their codes, and attention over them."""
    H, D, T = 1, 64, 40
    q, k, v, phi, psi = sequence(1, H, T, D, F16, seed=3)
    v[0, 0, 3] *= 1e-6
    v[0, 0, 4] = 0
    v[0, 0, 5] = v[0, 0, 5] / v[0, 0, 5].abs().max() * 60000
    k[0, 0, 6] = 0
    table, n_pages = tables([T], 64)
    for t_last in (T, 5):  # with and without the large row
        cache = FPACache(n_pages, H, D, 64, F16, I8)
        fill(cache, table, [t_last], k, v, phi, psi)
        got = first_passage_decode(q[:, :, t_last - 1:t_last].cuda(), cache, table, i32([t_last]), torch.ones(1, device="cuda"))
        want = expected(q[0, :, :t_last], k[0, :, :t_last], v[0, :, :t_last], phi[0, :, :t_last], psi[0, :, :t_last], torch.ones(1), 1, I8)
        assert_close(got[0], want, v[0, 0, :t_last].abs().max().item(), F16)
    # Values of 1e-6 throughout: P' stays in range because V's scale is in the exponent.
    v = (v.clamp(-3, 3) * 1e-5).to(F16)
    cache = FPACache(n_pages, H, D, 64, F16, I8)
    fill(cache, table, [T], k, v, phi, psi)
    got = first_passage_decode(q[:, :, -1:].cuda(), cache, table, i32([T]), torch.ones(1, device="cuda"))
    want = expected(q[0], k[0], v[0], phi[0], psi[0], torch.ones(1), 1, I8)
    err = (got[0].double().cpu() - want).abs().max().item()
    assert err <= TOL[F16] * v.abs().max().item() + 2.0 ** -25  # half a step of fp16's subnormals


# ------------------------------------------------------------------------------------------------------ decode ----

LENS = [[0, 1, 2, 33, 64], [31, 32, 63, 65, 97], [129, 500, 0, 1000, 257]]


def run_decode(lens, n, H, D, page, dtype, storage, seed, P=0, beta=None, walk=0.5):
    B, T = len(lens), max(max(lens), n)
    q, k, v, phi, psi = sequence(B, H, T, D, dtype, seed, walk)
    beta = 0.5 + torch.rand(H, generator=torch.Generator().manual_seed(seed)) if beta is None else beta
    table, n_pages = tables(lens + [P], page, seed=seed)
    table, ptable = table[:-1], table[-1, :-(-P // page)].contiguous()
    cache = FPACache(n_pages, H, D, page, dtype, storage)
    poison(cache)
    fill(cache, table, lens, k, v, phi, psi)
    kw, pre = {}, None
    if P:
        pre = [x[0] for x in sequence(1, H, P, D, dtype, seed + 1, walk)]
        fill(cache, ptable[None], [P], *(x[None] for x in pre[1:]))
        kw = dict(prefix_table=ptable, prefix_len=P)
    qn = torch.zeros(B, H, n, D, dtype=dtype)
    for b, L in enumerate(lens):
        c = min(n, L)
        qn[b, :, n - c:] = q[b, :, L - c:L]
        if c < n:
            qn[b, :, :n - c] = 7  # rows that stand before the sequence's first token
    got = first_passage_decode(qn.cuda(), cache, table, i32(lens), beta.cuda(), **kw)
    cache.check()
    assert got.dtype == dtype and got.shape == (B, H, n, D) and torch.isfinite(got).all()
    for b, L in enumerate(lens):
        c = min(n, L)
        assert (got[b, :, :n - c] == 0).all()
        if not c:
            continue
        seq = [x[b, :, :L] for x in (q, k, v, phi, psi)]
        if P:
            seq = [torch.cat([x, y], 1) for x, y in zip(pre, seq)]
        want = expected(*seq, beta, c, storage)
        assert_close(got[b, :, n - c:], want, seq[2].abs().max().item(), dtype, (b, L))
    return cache, table, qn, beta, got, kw


@pytest.mark.parametrize("dtype,storage", [(F16, None), (F16, I8), (F32, None), (F32, I8)])
@pytest.mark.parametrize("D", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("n", [1, 3, 8, 16])
def test_decode(dtype, storage, D, n):
    for i, lens in enumerate(LENS):
        run_decode(lens, n, 2, D, (32, 64, 128)[i], dtype, storage, seed=D + n + i)


@pytest.mark.parametrize("dtype,storage", [(F16, None), (F16, I8), (F32, None), (F32, I8)])
@pytest.mark.parametrize("n", [1, 2, 5, 9, 13])
def test_decode_row_counts(dtype, storage, n):
    run_decode([n, n + 1, n - 1, 40 + n], n, 3, 64, 32, dtype, storage, seed=n)


@pytest.mark.parametrize("B,H,n,D,dtype,storage,P", [(64, 12, 1, 16, F16, I8, 0), (33, 24, 5, 64, F16, None, 0), (2, 400, 3, 16, F32, None, 0),
                                                     (50, 24, 1, 64, F16, I8, 40), (65, 12, 2, 32, F16, I8, 0)])
def test_decode_more_pairs_than_run_at_once(B, H, n, D, dtype, storage, P):
    """The CTAs take the sequences in the order of their lengths: many equal ones, empty ones, the longest last."""
    lens = [min(i * 37 % 150, 101) for i in range(B - 1)] + [160]
    cache, table, qn, beta, got, kw = run_decode(lens, n, H, D, 32, dtype, storage, seed=B, P=P)
    bad = list(lens)
    bad[1] = table.shape[1] * 32 + 1  # beyond the table: the page ids there are -1, so nothing outside is read
    bad[0] = -7
    out = first_passage_decode(qn.cuda(), cache, table, i32(bad), beta.cuda(), **kw)
    with pytest.raises(ValueError):
        cache.check()
    assert torch.equal(out[2:], got[2:])


@pytest.mark.parametrize("B,H,n,D,dtype,storage,P", [(64, 12, 1, 16, F16, I8, 0), (40, 12, 3, 64, F16, None, 0), (64, 12, 1, 32, F16, I8, 50),
                                                     (15, 64, 2, 64, F16, I8, 0), (62, 16, 1, 32, F32, None, 0)])
def test_decode_in_two_launches(B, H, n, D, dtype, storage, P):
    """Long tables, a few sequences more than one round of CTAs holds. What follows on the stream waits for both."""
    lens = [min(i * 37 % 150, 101) for i in range(B - 3)] + [1030, 3, 640]
    cache, table, qn, beta, got, kw = run_decode(lens, n, H, D, 64, dtype, storage, seed=B, P=P)
    q, lengths, beta = qn.cuda(), i32(lens), beta.cuda()
    LaunchStats.reset()
    assert torch.equal(first_passage_decode(q, cache, table, lengths, beta, **kw), got)
    assert LaunchStats.kernels == (4 if P else 2) or dtype == F32
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = first_passage_decode(q, cache, table, lengths, beta, **kw)
    graph.replay()
    assert torch.equal(out, got)
    # Calls in a row, the newest token rewritten before each: every call sees its own.
    last = i32([max(x - 1, 0) for x in lens])
    _, k, v, phi, psi = (x.cuda() for x in sequence(B, H, 2, D, dtype, seed=9))
    outs = [[], []]
    for i in range(20):
        j = i & 1
        cache.append(k[:, :, j:j + 1], v[:, :, j:j + 1], phi[..., j:j + 1], psi[..., j:j + 1], table, last, (lengths > 0).int())
        outs[j].append(first_passage_decode(q, cache, table, lengths, beta, **kw))
    assert all(torch.equal(x, y[0]) for y in outs for x in y) and not torch.equal(outs[0][0], outs[1][0])


@pytest.mark.parametrize("B,H,n,D,storage,P", [(40, 16, 1, 32, None, 0), (40, 16, 2, 64, I8, 0), (40, 16, 2, 128, None, 0), (55, 12, 2, 32, None, 50)])
def test_float32_decode_in_two_launches(B, H, n, D, storage, P):
    """As above, for float32 queries: 592 places (296 at D = 128) and a few sequences more than a round of them holds."""
    lens = [min(i * 37 % 150, 101) for i in range(B - 3)] + [1030, 3, 640]
    cache, table, qn, beta, got, kw = run_decode(lens, n, H, D, 64, F32, storage, seed=B, P=P)
    q, lengths, beta = qn.cuda(), i32(lens), beta.cuda()
    LaunchStats.reset()
    assert torch.equal(first_passage_decode(q, cache, table, lengths, beta, **kw), got)
    assert LaunchStats.kernels == (4 if P else 2)
    last = i32([max(x - 1, 0) for x in lens])
    _, k, v, phi, psi = (x.cuda() for x in sequence(B, H, 2, D, F32, seed=9))
    outs = [[], []]
    for i in range(20):
        j = i & 1
        cache.append(k[:, :, j:j + 1], v[:, :, j:j + 1], phi[..., j:j + 1], psi[..., j:j + 1], table, last, (lengths > 0).int())
        outs[j].append(first_passage_decode(q, cache, table, lengths, beta, **kw))
    assert all(torch.equal(x, y[0]) for y in outs for x in y) and not torch.equal(outs[0][0], outs[1][0])


@pytest.mark.parametrize("beta", [-0.7, 0.0, 3.0])
@pytest.mark.parametrize("dtype,storage", [(F16, I8), (F32, None)])
def test_decode_beta_and_wide_fields(beta, dtype, storage):
    run_decode([300, 41], 4, 2, 32, 64, dtype, storage, seed=5, beta=torch.full((2,), beta))
    if beta >= 0:
        run_decode([300, 41], 4, 2, 32, 64, dtype, storage, seed=6, beta=torch.full((2,), beta), walk=40.0)


@pytest.mark.parametrize("dtype,storage", [(F16, None), (F16, I8), (F32, I8)])
@pytest.mark.parametrize("D,n,P", [(64, 1, 1), (64, 1, 33), (16, 5, 128), (128, 3, 1000), (256, 2, 200), (32, 16, 517)])
def test_prefix(dtype, storage, D, n, P):
    run_decode([n, 0, 70, 200, 1], n, 2, D, 64, dtype, storage, seed=P, P=P)


@pytest.mark.parametrize("B,n", [(1, 1), (9, 1), (33, 2), (70, 4), (20, 16)])
@pytest.mark.parametrize("storage", [None, I8])
def test_prefix_many_rows(B, n, storage):
    run_decode([(7 * b) % 90 for b in range(B)], n, 1, 64, 32, F16, storage, seed=B, P=300)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("storage", [None, I8])
@pytest.mark.parametrize("B,n,P,page", [(17, 1, 1, 32), (8, 4, 128, 64), (11, 3, 257, 128), (16, 4, 640, 256), (13, 5, 1000, 32),
                                        (40, 3, 129, 64), (43, 3, 2100, 128), (9, 15, 127, 32)])
def test_prefix_on_the_tensor_cores(D, storage, B, n, P, page):
    """17 to 135 rows: a quarter, half or all of the 128 lanes, and a second row tile; prefixes around tile ends."""
    run_decode([(11 * b) % 50 for b in range(B)], n, 2, D, page, F16, storage, seed=B + P, P=P)


@pytest.mark.parametrize("B,n", [(3, 4), (6, 9), (9, 10)])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("storage", [None, I8])
def test_prefix_ahead_of_the_rows_minima(D, storage, B, n):
    """Four and more tiles of the prefix in a CTA, and long own histories in small pages: the rows' minima come late, so
    the loads run as far ahead as the ring lets them. Many calls in a row give the same bits."""
    lens = [2000 - 100 * b for b in range(B)]
    cache, table, qn, beta, got, kw = run_decode(lens, n, 9, D, 32, F16, storage, seed=B, P=7345)
    q, beta = qn.cuda(), beta.cuda()
    for _ in range(50):
        assert torch.equal(first_passage_decode(q, cache, table, i32(lens), beta, **kw), got)
    cache.check()


def test_prefix_rows_far_apart():
    """Rows whose scores differ by thousands beside ordinary ones, and a falling field: maxima that grow late."""
    B, n, D, P = 30, 2, 64, 700
    for beta, walk in ((4.0, 20.0), (-0.5, 3.0)):
        run_decode([(5 * b) % 40 for b in range(B)], n, 2, D, 64, F16, I8, seed=17, P=P, beta=torch.full((2,), beta), walk=walk)


def test_prefix_equals_whole_sequences():
    """The same tokens stored once as a prefix, or in front of every sequence: equal to rounding."""
    H, D, P, lens, n = 2, 64, 320, [65, 130], 2
    q, k, v, phi, psi = sequence(2, H, P + 130, D, F32, seed=8)
    for x in (k, v, phi, psi):
        x[1, :, :P] = x[0, :, :P]
    whole = [P + x for x in lens]
    table, n_pages = tables(whole, 64)
    a = FPACache(n_pages, H, D, 64, F32)
    fill(a, table, whole, k, v, phi, psi)
    beta = torch.ones(H, device="cuda")
    qn = torch.stack([q[b, :, P + L - n:P + L] for b, L in enumerate(lens)]).cuda()
    x = first_passage_decode(qn, a, table, i32(whole), beta)
    # The same pages, seen through tables that start behind the prefix.
    y = first_passage_decode(qn, a, table[:, P // 64:], i32(lens), beta, prefix_table=table[0, :P // 64].contiguous(), prefix_len=P)
    assert (x - y).abs().max().item() <= 1e-5 * v.abs().max().item()


def test_decode_matches_the_training_operator():
    B, H, T, D = 2, 3, 700, 64
    q, k, v, phi, psi = (x.cuda() for x in sequence(B, H, T, D, F16, seed=9))
    beta = torch.ones(H, device="cuda")
    want = first_passage_attention(q, k, v, phi, psi, beta)
    table, n_pages = tables([T, T], 64)
    cache = FPACache(n_pages, H, D)
    cache.append(k, v, phi, psi, table, i32([0, 0]))
    qkv = torch.stack([q, k, v]).permute(1, 3, 0, 2, 4).contiguous()  # queries as views of a fused projection
    for L in (1, 64, 65, 700):
        got = first_passage_decode(qkv.permute(2, 0, 3, 1, 4)[0][:, :, L - 1:L], cache, table, i32([L, L]), beta)
        # each side within its tolerance of the exact rows
        assert (got - want[:, :, L - 1:L]).abs().max().item() <= (TOL[F16] + 2e-3) * v.abs().max().item()


def test_query_layouts():
    """Queries whose elements lie two apart, or at odd addresses, and an output as it comes."""
    cache, table, qn, beta, got, _ = run_decode([100, 37], 2, 2, 64, 64, F16, I8, seed=10)
    wide = torch.zeros(*qn.shape[:3], 128, dtype=F16, device="cuda")
    wide[..., ::2] = qn.cuda()
    off = torch.zeros(qn.numel() + 1, dtype=F16, device="cuda")
    off[1:] = qn.cuda().flatten()
    for q in (wide[..., ::2], off[1:].view(qn.shape)):
        assert torch.equal(first_passage_decode(q, cache, table, i32([100, 37]), beta.cuda()), got)


def test_repeat_runs_streams_and_graphs():
    """The same bits on every run, on another stream, and replayed from a CUDA graph with new lengths and queries."""
    lens = [900, 300, 1, 0]
    cache, table, qn, beta, got, kw = run_decode(lens, 3, 2, 64, 64, F16, I8, seed=11, P=200)
    q, beta, L = qn.cuda(), beta.cuda(), i32(lens)
    torch.cuda.synchronize()
    for _ in range(3):
        assert torch.equal(first_passage_decode(q, cache, table, L, beta, **kw), got)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        o = first_passage_decode(q, cache, table, L, beta, **kw)
    side.synchronize()
    assert torch.equal(o, got)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = first_passage_decode(q, cache, table, L, beta, **kw)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(o, got)
    L.copy_(i32([5, 0, 1, 0]))
    q.mul_(0.5)
    graph.replay()
    assert torch.equal(o, first_passage_decode(q, cache, table, L, beta, **kw))


def test_large_pool_offsets():
    """Pages beyond 2^31 elements of the pool."""
    H, D, page = 16, 256, 256
    n_pages = 2 ** 31 // (H * D * page) + 20
    free, _ = torch.cuda.mem_get_info()
    if free < 8 * 2 ** 30:
        pytest.skip("needs 8 GiB of free device memory")
    cache = FPACache(n_pages, H, D, page, F16, I8)
    T, n = 300, 2
    q, k, v, phi, psi = sequence(1, H, T, D, F16, seed=12)
    table = i32([[n_pages - 1, n_pages - 2]])
    fill(cache, table, [T], k, v, phi, psi)
    got = first_passage_decode(q[:, :, -n:].cuda(), cache, table, i32([T]), torch.ones(H, device="cuda"))
    want = expected(q[0], k[0], v[0], phi[0], psi[0], torch.ones(H), n, I8)
    assert_close(got[0], want, v.abs().max().item(), F16)
    back = cache.read(table, None, T, i32([T]))
    assert torch.equal(back[0].cpu(), quantise(k)[2].to(F16))


def test_long_context():
    """16383 tokens, many pages per warp: rows against the oracle's single-row evaluation."""
    H, D, T, n = 2, 128, 16383, 2
    q, k, v, phi, psi = sequence(1, H, T, D, F16, seed=13, walk=0.05)
    table, n_pages = tables([T], 128)
    cache = FPACache(n_pages, H, D, 128, F16)
    fill(cache, table, [T], k, v, phi, psi)
    beta = torch.ones(H)
    got = first_passage_decode(q[:, :, -n:].cuda(), cache, table, i32([T]), beta.cuda())
    for r in range(n):
        t = T - n + r
        for h in range(H):
            low = torch.cat([phi[0, h, 1:t + 1].double().flip(0).cummin(0).values.flip(0), torch.full((1,), float("inf"), dtype=torch.float64)])
            z = k[0, h, :t + 1].double() @ q[0, h, t].double() / D ** 0.5 + (low - psi[0, h, :t + 1].double()).clamp(max=0)
            z[t] = k[0, h, t].double() @ q[0, h, t].double() / D ** 0.5
            want = z.softmax(0) @ v[0, h, :t + 1].double()
            assert_close(got[0, h, r], want, v.abs().max().item(), F16)


def test_bad_tables_are_reported_and_not_touched():
    """Page ids outside the pool, lengths beyond the table, negative starts: skipped, recorded, raised by check()."""
    H, D = 1, 16
    cache = FPACache(2, H, D, 32, F16, I8)
    cache.check()
    _, k, v, phi, psi = (x.cuda() for x in sequence(1, H, 40, D, F16, seed=14))
    before = [x.clone() for x in (cache.k, cache.v, cache.phi, cache.phi_min)]
    for table, start in (([[5, 9]], 0), ([[-1, -7]], 0), ([[0, 1]], -3), ([[0, 1]], 64)):
        cache.append(k, v, phi, psi, i32(table), i32([start]))
        with pytest.raises(ValueError, match="outside"):
            cache.check()
        assert all(torch.equal(x, y) for x, y in zip(before, (cache.k, cache.v, cache.phi, cache.phi_min)))
    cache.append(k[:, :, :32], v[:, :, :32], phi[..., :32], psi[..., :32], i32([[0]]), i32([0]))
    cache.check()
    q = torch.ones(1, H, 1, D, dtype=F16, device="cuda")
    beta = torch.ones(H, device="cuda")
    for table, length in (([[0, 2]], 40), ([[-1, 0]], 40), ([[0]], 33)):
        o = first_passage_decode(q, cache, i32(table), i32([length]), beta)
        assert torch.isfinite(o).all()
        with pytest.raises(ValueError, match="outside"):
            cache.check()
    cache.read(i32([[0, 7]]), None, 64)
    with pytest.raises(ValueError, match="outside"):
        cache.check()
    cache.check()


def test_refusals():
    cache = FPACache(4, 2, 32, 32)
    t, n, b = i32([[0, 1]]), i32([3]), torch.ones(2, device="cuda")
    q = torch.zeros(1, 2, 1, 32, dtype=F16, device="cuda")
    f = torch.zeros(1, 2, 1, device="cuda")
    bad = [
        (lambda: first_passage_decode(q.float(), cache, t, n, b), "must be torch.float16"),
        (lambda: first_passage_decode(q[..., :16], cache, t, n, b), "q must have shape"),
        (lambda: first_passage_decode(q.expand(1, 2, 17, 32), cache, t, n, b), "between 1 and 16"),
        (lambda: first_passage_decode(q, cache, t.long(), n, b), "block_table must be an int32"),
        (lambda: first_passage_decode(q, cache, t[0], n, b), "block_table must have shape"),
        (lambda: first_passage_decode(q, cache, t, n.cpu(), b), "lengths must be an int32 tensor on"),
        (lambda: first_passage_decode(q, cache, t, i32([1, 2]), b), "lengths must be contiguous with shape"),
        (lambda: first_passage_decode(q, cache, t, n, b[:1]), "beta must be"),
        (lambda: first_passage_decode(q, cache, t, n, b, prefix_len=3), "needs a prefix_table"),
        (lambda: first_passage_decode(q, cache, t, n, b, prefix_table=i32([2]), prefix_len=33), "longer than the pages"),
        (lambda: cache.append(q, q[:, :1], f, f, t, n), "k and v must have shape"),
        (lambda: cache.append(q.float(), q.float(), f, f, t, n), "k and v must be torch.float16"),
        (lambda: cache.append(q, q, f[:, :1], f, t, n), "phi and psi must have shape"),
        (lambda: cache.append(q, q, f.half(), f, t, n), "phi and psi must be float32"),
        (lambda: cache.append(q, q, f.cpu(), f, t, n), "cache's device"),
        (lambda: cache.append(q, q, f, f, t, n, counts=n.long()), "counts must be an int32"),
        (lambda: cache.read(t, None, -1), "must not be negative"),
    ]
    for call, message in bad:
        with pytest.raises(ValueError, match=message):
            call()
    LaunchStats.reset()
    cache.append(q[:, :, :0], q[:, :, :0], f[..., :0], f[..., :0], t, n)     # nothing to do
    assert cache.read(t, None, 0)[0].shape == (1, 2, 0, 32)
    assert first_passage_decode(q[:0], cache, t[:0], n[:0], b).shape == (0, 2, 1, 32)
    assert LaunchStats.kernels == 0


# ------------------------------------------------------------------------- keys that are not there, or not finite ----

FORMS = [(F16, None), (F16, I8), (F32, None), (F32, I8)]


def expected_rows(q, k, v, phi, psi, beta, n, storage, gone):
    """As `expected`, without the keys that `gone` [T] marks; rows that see no key at all are zeros."""
    if storage == I8:
        k, v = quantise(k)[2], quantise(v)[2]
    q, k, v, phi, psi, beta = (x.double().cuda() for x in (q, k, v, phi, psi, beta))
    gone = gone.cuda()
    phi = torch.where(gone, torch.inf, phi)
    T, out = k.shape[1], []
    for t in range(T - n, T):
        least = phi[:, 1:t + 1].flip(-1).cummin(-1).values.flip(-1)
        z = (k[:, :t + 1] @ q[:, t, :, None])[..., 0] / q.shape[-1] ** 0.5
        z[:, :t] += beta[:, None] * (least - psi[:, :t]).clamp(max=0)
        z = torch.where(gone[:t + 1], -torch.inf, z)
        o = (z.softmax(-1)[:, None] @ v[:, :t + 1])[:, 0]
        out.append(torch.zeros_like(o) if bool(gone[:t + 1].all()) else o)
    return torch.stack(out, 1).cpu()


@pytest.mark.parametrize("dtype,storage", FORMS)
@pytest.mark.parametrize("D,page,L,n,P", [(64, 32, 1000, 1, 0), (64, 64, 1000, 3, 0), (128, 64, 333, 16, 0), (256, 32, 200, 2, 0), (16, 128, 900, 5, 0),
                                          (64, 32, 150, 5, 700), (128, 64, 150, 6, 700), (32, 32, 40, 3, 300), (64, 32, 33, 1, 150)])
def test_keys_behind_bad_pages_are_skipped(dtype, storage, D, page, L, n, P):
    """Table entries outside the pool: the result is that of the remaining keys, whatever the sequence is split into. A
    row that sees none is zero."""
    H, B = 2, 5
    q, k, v, phi, psi = sequence(B, H, L, D, dtype, seed=D + n)
    table, n_pages = tables([L] * B + [P], page, seed=L)
    table, ptable = table[:-1], table[-1, :-(-P // page)].contiguous()
    cache = FPACache(n_pages, H, D, page, dtype, storage)
    poison(cache)
    fill(cache, table, [L] * B, k, v, phi, psi)
    pages, npre = -(-L // page), ptable.numel()
    bad = [[pages // 2], [0, pages - 1], list(range(pages // 3, pages - 1)), [pages - 1], list(range(pages))]
    kw, pre, pgone = {}, None, torch.zeros(0, dtype=torch.bool)
    if P:
        pre = [x[0] for x in sequence(1, H, P, D, dtype, 7)]
        fill(cache, ptable[None], [P], *(x[None] for x in pre[1:]))
        pgone = torch.zeros(P, dtype=torch.bool)
        for i, x in ((npre // 2, -5), (npre - 1, n_pages)):
            ptable[i] = x
            pgone[i * page:(i + 1) * page] = True
        kw = dict(prefix_table=ptable, prefix_len=P)
    gone = torch.zeros(B, L, dtype=torch.bool)
    for b, drop in enumerate(bad):
        for i in drop:
            table[b, i] = (-1, n_pages, -2 ** 31, 2 ** 31 - 1)[(b + i) % 4]
            gone[b, i * page:(i + 1) * page] = True
    beta = torch.tensor([0.8, 1.3])
    got = first_passage_decode(q[:, :, L - n:].cuda(), cache, table, i32([L] * B), beta.cuda(), **kw)
    with pytest.raises(ValueError, match="outside"):
        cache.check()
    for b in range(B):
        seq = [x[b] for x in (q, k, v, phi, psi)]
        if P:
            seq = [torch.cat([x, y], 1) for x, y in zip(pre, seq)]
        want = expected_rows(*seq, beta, n, storage, torch.cat([pgone, gone[b]]))
        assert torch.isfinite(got[b]).all()
        assert_close(got[b], want, seq[2].abs().max().item(), dtype, b)


@pytest.mark.parametrize("dtype,storage", FORMS)
@pytest.mark.parametrize("D,n,P", [(64, 2, 0), (128, 5, 0), (256, 3, 0), (32, 3, 400), (256, 2, 300), (64, 5, 700), (128, 3, 700)])
@pytest.mark.parametrize("offset,slope,sign", [(1e6, 0.0, 1), (-1e6, 0.0, -1), (0.0, -4.0, 1), (3e5, -1.0, 1)])
def test_a_walk_far_from_zero(dtype, storage, D, n, P, offset, slope, sign):
    """The bias depends on differences of the field only: a walk that starts far from zero or falls steadily costs no
    accuracy (an offset of 1e6 is held in steps of 1/16, a logit off by such a step would show at 6e-2)."""
    H, lens = 2, [700, 33, 64, 500, 150, 9]
    B, T = len(lens), max(lens)
    drift = offset + slope * torch.arange(P + T, dtype=torch.float32)
    q, k, v, phi, psi = sequence(B, H, T, D, dtype, seed=D + n)
    phi, psi = phi + drift[P:], psi + drift[P:]
    table, n_pages = tables(lens + [P], 64, seed=n)
    table, ptable = table[:-1], table[-1, :-(-P // 64)].contiguous()
    cache = FPACache(n_pages, H, D, 64, dtype, storage)
    fill(cache, table, lens, k, v, phi, psi)
    kw, pre = {}, None
    if P:
        pre = [x[0] for x in sequence(1, H, P, D, dtype, 5)]
        pre[3], pre[4] = pre[3] + drift[:P], pre[4] + drift[:P]
        fill(cache, ptable[None], [P], *(x[None] for x in pre[1:]))
        kw = dict(prefix_table=ptable, prefix_len=P)
    beta = sign * torch.tensor([0.8, 1.3])
    newest = torch.stack([q[b, :, L - n:L] for b, L in enumerate(lens)]).cuda()
    got = first_passage_decode(newest, cache, table, i32(lens), beta.cuda(), **kw)
    for b, L in enumerate(lens):
        seq = [x[b, :, :L] for x in (q, k, v, phi, psi)]
        if P:
            seq = [torch.cat([x, y], 1) for x, y in zip(pre, seq)]
        assert_close(got[b], expected(*seq, beta, n, storage), seq[2].abs().max().item(), dtype, (b, L))


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("D,P", [(64, 0), (128, 0), (16, 0), (64, 300), (128, 300), (256, 200)])
def test_int8_rows_that_are_not_finite(dtype, D, P):
    """A row of keys or values with a NaN or an infinity has no codes: it reads back as NaN, and what attends to it is NaN.
    Other rows, sequences and heads are as they were."""
    H, L, n, page = 2, 100, 3, 32
    q, k, v, phi, psi = sequence(6, H, L, D, dtype, seed=D)
    table, n_pages = tables([L] * 6 + [P], page)
    table, ptable = table[:-1], table[-1, :-(-P // page)].contiguous()
    cache = FPACache(n_pages, H, D, page, dtype, I8)
    kw, pre = {}, None
    if P:
        pre = [x[0] for x in sequence(1, H, P, D, dtype, 3)]
        fill(cache, ptable[None], [P], *(x[None] for x in pre[1:]))
        kw = dict(prefix_table=ptable, prefix_len=P)
    nan, inf = float("nan"), float("inf")
    bad = {0: (k, 40, nan), 1: (v, 41, nan), 2: (k, 42, inf), 3: (v, 43, -inf)}
    for b, (x, s, value) in bad.items():
        x[b, 0, s, (7 * b) % D] = value
    fill(cache, table, [L] * 6, k, v, phi, psi)
    back = cache.read(table, None, L)
    for b, (x, s, _) in bad.items():
        r = back[0 if x is k else 1][b].cpu()
        assert torch.isnan(r[0, s]).all()
        keep = torch.ones(H, L, dtype=torch.bool)
        keep[0, s] = False
        assert torch.equal(r[keep], quantise(x[b][keep])[2].to(dtype))
    beta = torch.tensor([0.0, 1.0])  # head 0 without the bias: every key counts
    got = first_passage_decode(q[:, :, L - n:].cuda(), cache, table, i32([L] * 6), beta.cuda(), **kw)
    for b in range(6):
        seq = [x[b] for x in (q, k, v, phi, psi)]
        if P:
            seq = [torch.cat([x, y], 1) for x, y in zip(pre, seq)]
        heads = slice(1, 2) if b in bad else slice(0, 2)
        if b in bad:
            assert torch.isnan(got[b, 0]).all(), b
        want = expected(*(x[heads] for x in seq), beta[heads], n, I8)
        assert_close(got[b, heads], want, max(x[heads].abs().max().item() for x in seq[2:3]), dtype, b)
    if P:  # a value of the prefix that is not finite reaches every row
        pre[2][0, 77, 1] = nan
        fill(cache, ptable[None], [P], *(x[None] for x in pre[1:]))
        got = first_passage_decode(q[:, :, L - n:].cuda(), cache, table, i32([L] * 6), beta.cuda(), **kw)
        assert torch.isnan(got[:, 0]).all() and torch.isfinite(got[:, 1]).all()


def test_int8_rows_near_the_end_of_float32():
    """127 x overflows from 2.7e36 on; the codes do not."""
    H, D, n = 2, 32, 6
    _, k, v, phi, psi = sequence(1, H, n, D, F32, seed=4)
    for i, top in enumerate((3.0e38, 1e37, 3e36, 2e36, 1.3e30, 1.2e30)):
        k[0, :, i] = k[0, :, i] / k[0, :, i].abs().amax(-1, keepdim=True) * top
        v[0, :, i] = v[0, :, i] / v[0, :, i].abs().amax(-1, keepdim=True) * top
    table, n_pages = tables([n], 32)
    cache = FPACache(n_pages, H, D, 32, F32, I8)
    fill(cache, table, [n], k, v, phi, psi)
    for x, pool, scales in ((k, cache.k, cache.k_scale), (v, cache.v, cache.v_scale)):
        top = x[0].double().abs().amax(-1, keepdim=True)
        exact = x[0].double() * 127 / top
        codes = pool[table[0, 0], :, :n].cpu().double() - 128
        # A code next to the exact quotient; the nearest one unless the quotient is within float32 rounding of a half.
        assert ((codes - exact).abs() <= 0.5 + 1e-4).all()
        assert (scales[table[0, 0], :, :n].cpu().double() * 127 / top[..., 0] - 1).abs().max().item() <= 2.0 ** -22


@pytest.mark.parametrize("dtype,storage", FORMS)
@pytest.mark.parametrize("D,n,P", [(16, 5, 0), (64, 5, 0), (128, 16, 0), (256, 7, 0), (32, 2, 0), (64, 6, 300), (64, 9, 0)])
def test_new_tokens_that_are_not_finite_stay_behind_the_mask(dtype, storage, D, n, P):
    """A drafted token whose key, value or field is NaN or infinite does not reach the rows before it, which cannot see
    it; what its value does to the other columns of the rows that see it is nothing either."""
    H, L, page = 2, 70, 32
    nan, inf = float("nan"), float("inf")
    at = L - n + n // 2  # the token, and a later one for n > 2
    cases = [("k", nan), ("k", inf), ("v", nan), ("v", inf), ("v", -inf), ("phi", nan), ("phi", -inf), ("psi", nan), ("psi", inf)]
    B = len(cases)
    q, k, v, phi, psi = sequence(B, H, L, D, dtype, seed=n)
    names = dict(k=k, v=v, phi=phi, psi=psi)
    for b, (name, value) in enumerate(cases):
        if name in "kv":
            names[name][b, :, at, 3] = value
            names[name][b, :, L - 1, D - 1] = value
        else:
            names[name][b, :, at] = value
    table, n_pages = tables([L] * B + [P], page)
    table, ptable = table[:-1], table[-1, :-(-P // page)].contiguous()
    cache = FPACache(n_pages, H, D, page, dtype, storage)
    poison(cache)
    kw, pre = {}, None
    if P:
        pre = [x[0] for x in sequence(1, H, P, D, dtype, 3)]
        fill(cache, ptable[None], [P], *(x[None] for x in pre[1:]))
        kw = dict(prefix_table=ptable, prefix_len=P)
    fill(cache, table, [L] * B, k, v, phi, psi)
    beta = torch.tensor([0.8, 1.3])
    got = first_passage_decode(q[:, :, L - n:].cuda(), cache, table, i32([L] * B), beta.cuda(), **kw)
    rows = at - (L - n)  # rows before the token
    for b, (name, value) in enumerate(cases):
        seq = [x[b, :, :at] for x in (q, k, v, phi, psi)]
        if P:
            seq = [torch.cat([x, y], 1) for x, y in zip(pre, seq)]
        want = expected(*seq, beta, rows, storage)
        assert torch.isfinite(got[b, :, :rows]).all(), (name, value)
        assert_close(got[b, :, :rows], want, seq[2].abs().max().item(), dtype, (name, value))
        if name == "v" and storage is None:
            # The rows from it on: not finite in its column, as they were in the others.
            rest = got[b, :, rows:n - 1].float().cpu()
            assert not torch.isfinite(rest[..., 3]).any()
            finite = v[b:b + 1, :, :].clone()
            finite[0, :, at, 3] = finite[0, :, L - 1, D - 1] = 0
            for r in range(rows, n - 1):
                T = L - n + r + 1
                seq = [x[b, :, :T] for x in (q, k)] + [finite[0, :, :T], phi[b, :, :T], psi[b, :, :T]]
                if P:
                    seq = [torch.cat([x, y], 1) for x, y in zip(pre, seq)]
                want = expected(*seq, beta, 1, storage)[:, 0]
                others = [d for d in range(D) if d != 3]
                assert_close(got[b, :, r][:, others], want[:, others], seq[2].abs().max().item(), dtype, (name, value, r))
        elif name in "kv" and not (storage is None and value == inf):  # an infinite product may be -inf, which is no weight
            assert not torch.isfinite(got[b, :, rows:].float()).all(-1).any()


def test_lengths_at_the_end_of_32_bits():
    """A table of 2^31 positions, all in one page: lengths end where rounding up to a page stays within 32 bits."""
    H, D, page = 1, 16, 256
    q, k, v, phi, psi = sequence(1, H, page, D, F16, seed=15)
    cache = FPACache(1, H, D, page, F16)
    table = torch.zeros(1, 2 ** 31 // page, dtype=torch.int32, device="cuda")
    cache.append(k.cuda(), v.cuda(), phi.cuda(), psi.cuda(), table, i32([0]))
    for length, ok in ((2 ** 31 - 256, True), (2 ** 31 - 1, False)):
        got = first_passage_decode(q[:, :, :1].cuda(), cache, table, i32([length]), torch.ones(H, device="cuda"))
        assert torch.isfinite(got).all()
        if ok:
            cache.check()
        else:
            with pytest.raises(ValueError, match="outside"):
                cache.check()


def test_gradients_are_refused_not_lost():
    """Forward only: a tensor that wants a gradient is refused while gradients are recorded."""
    cache = FPACache(4, 2, 32, 32)
    t, n, beta = i32([[0, 1]]), i32([1]), torch.ones(2, device="cuda")
    x = torch.zeros(1, 2, 1, 32, dtype=F16, device="cuda")
    f = torch.zeros(1, 2, 1, device="cuda")
    leaf = lambda y: y.clone().requires_grad_()  # noqa: E731
    cache.append(x, x, f, f, t, i32([0]))
    for call in (lambda: first_passage_decode(leaf(x), cache, t, n, beta), lambda: first_passage_decode(x, cache, t, n, leaf(beta)),
                 lambda: cache.append(leaf(x), x, f, f, t, i32([0])), lambda: cache.append(x, leaf(x), f, f, t, i32([0])),
                 lambda: cache.append(x, x, leaf(f), f, t, i32([0])), lambda: cache.append(x, x, f, leaf(f), t, i32([0]))):
        with pytest.raises(RuntimeError, match="forward only"):
            call()
        with torch.no_grad():
            call()


# ------------------------------------------------------------------------------------------------ verification ----

def verify_oracle(p, q, draft, u, noise, lens=None):
    """The definition, one sequence after the other, float32 operations rounded once each."""
    p, q, u, noise = (x.float().cpu().numpy() for x in (p, q, u, noise))
    draft = draft.cpu().numpy()
    B, n, V = q.shape
    accepted, tokens = [], []
    for b in range(B):
        k = n if lens is None else int(lens[b])
        a = 0
        while a < k:
            x = draft[b, a]
            if not (0 <= x < V) or not np.float32(u[b, a] * q[b, a, x]) < p[b, a, x]:
                break
            a += 1
        w = p[b, a] - (q[b, a] if a < k else np.float32(0))
        if not (w > 0).any():
            w = p[b, a]
        with np.errstate(divide="ignore", invalid="ignore"):
            score = np.where(w > 0, w / noise[b], np.float32(-1))
        accepted.append(a)
        tokens.append(list(draft[b, :a]) + [int(score.argmax())] + [-1] * (n - a))
    return torch.tensor(accepted, dtype=torch.int32), torch.tensor(np.array(tokens, dtype=np.int64).reshape(B, n + 1))


def draft_case(B, n, V, dtype, seed, close=0.5):
    g = torch.Generator().manual_seed(seed)
    logits = 2 * torch.randn(B, n + 1, V, generator=g)
    q = logits[:, :n].softmax(-1).to(dtype)
    p = (logits + close * torch.randn(B, n + 1, V, generator=g)).softmax(-1).to(dtype)
    draft = torch.multinomial(q.float().reshape(B * n, V), 1, generator=g).view(B, n) if n else torch.zeros(B, 0, dtype=torch.long)
    u = torch.rand(B, n, generator=g)
    noise = torch.empty(B, V).exponential_(generator=g)
    return [x.cuda() for x in (p, q, draft, u, noise)]


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("B,n,V", [(1, 4, 50304), (5, 1, 1), (3, 0, 7), (64, 7, 1000), (2, 16, 4097), (300, 3, 513), (4, 40, 33)])
def test_verify(dtype, B, n, V):
    args = draft_case(B, n, V, dtype, seed=B + n)
    got, want = verify_draft(*args), verify_oracle(*args)
    assert torch.equal(got[0].cpu(), want[0]) and torch.equal(got[1].cpu(), want[1])
    if n:
        lens = torch.randint(0, n + 1, (B,), generator=torch.Generator().manual_seed(n), dtype=torch.int32)
        got, want = verify_draft(*args, draft_lens=lens.cuda()), verify_oracle(*args, lens=lens)
        assert torch.equal(got[0].cpu(), want[0]) and torch.equal(got[1].cpu(), want[1])


def test_verify_edges():
    """Ties, an empty residual, zero probabilities, drafts outside the vocabulary, noise of zero, NaN, odd strides."""
    V, n = 40, 2
    p = torch.full((6, n + 1, V), 1 / V)
    q = torch.full((6, n, V), 1 / V)
    noise = torch.ones(6, V)
    draft = torch.zeros(6, n, dtype=torch.int64)
    u = torch.zeros(6, n)
    u[0, 0] = 1.0                    # refused at once with p == q: no residual, p's ties go to index 0
    p[1, 0, 0] = 0                   # the draft has no chance under p: refused even with u = 0
    draft[2, 1], draft[3, 0] = V, -1  # outside the vocabulary: refused
    noise[4, [7, 9]] = 0             # all accepted: the first infinite score
    p[5] = float("nan")              # nothing can be accepted or drawn: index 0
    args = [x.cuda() for x in (p, q, draft, u, noise)]
    accepted, tokens = verify_draft(*args)
    assert accepted.tolist() == [0, 0, 1, 0, 2, 0]
    want = verify_oracle(*(x[:5] for x in args))
    assert torch.equal(tokens[:5].cpu(), want[1])
    assert tokens[0].tolist() == [0, -1, -1] and tokens[4].tolist() == [0, 0, 7] and tokens[5].tolist() == [0, -1, -1]
    # The same through views: every other row of a wider batch, a transposed draft, rows that are not contiguous.
    wide = [torch.zeros((2 * x.shape[0],) + tuple(x.shape[1:]), dtype=x.dtype, device="cuda") for x in args]
    views = [w[::2] for w in wide]
    for w, x in zip(views, args):
        w.copy_(x)
    views[2] = args[2].t().contiguous().t()
    views[0] = args[0].transpose(1, 2).contiguous().transpose(1, 2)
    again = verify_draft(*views)
    assert torch.equal(again[0], accepted) and torch.equal(again[1], tokens)


def test_verified_tokens_have_the_targets_distribution():
    """The first token of 200000 verified drafts from q follows p: each frequency within 5 standard deviations."""
    V, N = 6, 200000
    g = torch.Generator(device="cuda").manual_seed(1)
    p = torch.tensor([0.05, 0.3, 0.1, 0.25, 0.0, 0.3], device="cuda")
    q = torch.tensor([0.3, 0.1, 0.1, 0.2, 0.2, 0.1], device="cuda")
    counts = torch.zeros(V, device="cuda")
    for _ in range(4):
        m = N // 4
        draft = torch.multinomial(q, m, replacement=True, generator=g)[:, None]
        u = torch.rand(m, 1, generator=g, device="cuda")
        noise = torch.empty(m, V, device="cuda").exponential_(generator=g)
        for lo in range(0, m, 50000):
            s = slice(lo, min(lo + 50000, m))
            _, tokens = verify_draft(p.expand(s.stop - lo, 2, V).contiguous(), q.expand(s.stop - lo, 1, V).contiguous(), draft[s], u[s], noise[s])
            counts += torch.bincount(tokens[:, 0], minlength=V)
    sd = (N * p * (1 - p)).sqrt()
    assert ((counts - N * p).abs() <= 5 * sd).all(), counts.tolist()


def test_verify_refusals():
    p, q, draft, u, noise = draft_case(2, 3, 11, F32, seed=0)
    for args, message in [
            ((p[:, :3], q, draft, u, noise), "p must have shape"), ((p.half(), q, draft, u, noise), "both be fp16 or both fp32"),
            ((p, q, draft.int(), u, noise), "draft must be"), ((p, q, draft, u[:, :2], noise), "u must be"),
            ((p, q, draft, u, noise.double()), "noise must be"), ((p, q, draft, u.cpu(), noise), "one CUDA device")]:
        with pytest.raises(ValueError, match=message):
            verify_draft(*args)
    with pytest.raises(ValueError, match="draft_lens"):
        verify_draft(p, q, draft, u, noise, draft_lens=torch.zeros(2, dtype=torch.int64, device="cuda"))
    assert verify_draft(p[:0], q[:0], draft[:0], u[:0], noise[:0])[1].shape == (0, 4)
