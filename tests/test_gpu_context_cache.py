"""The 8-bit context cache on the device against its definitions in 64 bits: codes, scales, bounds and chosen
blocks exactly, attention within bounds that follow from the roundings of its inputs.

Bounds of the attention (U = 2^-23, a unit of fp32 with room for sums that truncate).  A score is a sum of Dh products
of a query in two halves (22 bits) with an exact code, scaled twice: off by at most (Dh + 8) U A, A the largest
sum_d |q_d k_d| * scale.  Twice that is the relative error of a weight.  Weights in two halves, exponentials, the sums over 64
rows, blocks and partial results: another (N / 64 + 100) U.  One-part weights (bf16 queries) add 2^-11, the output's own type
half a step of it.  The log-sum-exp takes the score's error once and rounds a few times in its own magnitude."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -23
BLOCK = 64
ROWS = [16 * s + 8 * h + 2 * t + e for t in range(4) for s in range(4) for h in range(2) for e in range(2)]


def cc():
    from ar_tabpfn.model import context_cache
    return context_cache


@pytest.fixture(params=["by_cost", "few_rows", "row_tiles", "tensor_tiles"])
def form(request):
    """Attention by the kernels that their cost picks, and by each kind whatever the sizes."""
    from ar_tabpfn import _lib
    lib = _lib.lib()
    _lib.check(lib.artab_debug_set(_lib.DEBUG_CACHE_FORM, ("by_cost", "few_rows", "row_tiles", "tensor_tiles").index(request.param)))
    yield request.param
    lib.artab_debug_set(_lib.DEBUG_CACHE_FORM, 0)


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def rows(seed, G, H, N, D, dtype):
    g = gen(seed)
    spread = 0.3 + torch.rand(H, 1, D, device="cuda", generator=g)
    offset = torch.randn(H, 1, D, device="cuda", generator=g)
    return tuple((torch.randn(G, H, N, D, device="cuda", generator=g) * spread + offset).to(dtype) for _ in range(2))


# ------------------------------------------------------------------ definitions, 64 bits

def step(top):
    return (top / 127.0).float().double()


def quantized(k, v, lens, blocks):
    """codes as signed numbers [G,H,blocks,64,D] of keys and values, scales [G,H,blocks,2], live rows [G,blocks,64]."""
    G, H, N, D = k.shape
    live = (torch.arange(blocks * BLOCK, device=k.device) < lens[:, None]).view(G, 1, blocks, BLOCK, 1)
    codes, scales = [], []
    for x in (k, v):
        y = torch.zeros(G, H, blocks * BLOCK, D, dtype=torch.float64, device=k.device)
        y[:, :, :N] = x.double()
        y = torch.where(live, y.view(G, H, blocks, BLOCK, D), 0.0)
        s = step(y.abs().amax((-1, -2)))
        codes.append(torch.where(s[..., None, None] > 0, y / s[..., None, None], 0.0).round().clamp(-127, 127))
        scales.append(s)
    return codes[0], codes[1], torch.stack(scales, -1), live


def fields(cache):
    """The same from a cache's tensors."""
    G, H, nb = cache.scales.shape[:3]
    D = cache.head_dim
    c = cache.codes.double() - 128
    k = c[:, :, :, 0].reshape(G, H, nb, BLOCK, D)
    v = torch.empty_like(k)
    v[..., ROWS, :] = c[:, :, :, 1].reshape(G, H, nb, D, BLOCK).transpose(-1, -2)
    return k, v, cache.scales.double()


def check_fields(cache, ck, cv, scales, lens):
    G, H, nb = scales.shape[:3]
    live = (torch.arange(nb * BLOCK, device="cuda") < lens[:, None]).view(G, 1, nb, BLOCK, 1)
    k, v, s = fields(cache)
    used = live.any(3)                                               # [G,1,nb,1]
    assert torch.equal(torch.where(live, k, 0.0), torch.where(live, ck, 0.0).expand_as(k))
    assert torch.equal(torch.where(live, v, 0.0), torch.where(live, cv, 0.0).expand_as(v))
    assert torch.equal(torch.where(used, s, 0.0), torch.where(used, scales, 0.0))
    lo = torch.where(live, ck, 999.0).amin(3)
    hi = torch.where(live, ck, -999.0).amax(3)
    want = torch.stack([lo, hi], 3)
    got = cache.bounds.double()
    assert torch.equal(torch.where(used[..., None], got, 0.0), torch.where(used[..., None], want, 0.0))
    assert torch.equal(cache.lens.long(), lens.long())


def values(cache):
    k, v, s = fields(cache)
    return (k * s[..., :1, None]).flatten(2, 3), (v * s[..., 1:, None]).flatten(2, 3)


def attention(q, cache, scale, times=None):
    """out, lse in 64 bits, and what bounds the error: A and the largest value seen.  times [B,H,Lq,blocks]: how often a
    block counts."""
    k, v = values(cache)
    G, H, N, D = k.shape
    B, _, L, _ = q.shape
    live = torch.arange(N, device="cuda") < cache.lens[:, None]
    k, v = torch.where(live[:, None, :, None], k, 0.0).expand(B, -1, -1, -1), torch.where(live[:, None, :, None], v, 0.0).expand(B, -1, -1, -1)
    w = live.double().view(G, 1, 1, N).expand(B, H, L, N)
    if times is not None:
        w = w * times.double().repeat_interleave(BLOCK, 3)
    s = q.double() @ k.transpose(-1, -2) * scale + torch.log(w)
    A = float((q.double().abs() @ k.abs().transpose(-1, -2)).max()) * abs(scale)
    lse = torch.logsumexp(s, -1)
    p = torch.nan_to_num(torch.exp(s - lse[..., None]))
    return p @ v, lse, A, float(v.abs().max()), N


def check_attention(got, want, dtype, D):
    (out, lse), (o, l, A, vmax, N) = got, want
    assert out.dtype is dtype and lse.dtype is torch.float32
    rel = 2 * (D + 8) * U * A + (N / 64 + 100) * U
    tol = vmax * (rel + (2.0 ** -11 if dtype is torch.bfloat16 else 0.0)) + o.abs() * torch.finfo(dtype).eps / 2
    err = (out.double() - o).abs()
    assert bool((err <= tol).all()), (float(err.max()), float((err / tol).max()))
    nothing = torch.isinf(l)
    assert torch.equal(torch.isinf(lse), nothing) and bool((out[nothing] == 0).all())
    err = (lse.double() - l).abs()[~nothing]
    tol = ((D + 8) * U * A + (N / 64 + 100) * U + 4 * U * (l.abs() + A + 14))[~nothing]
    assert bool((err <= tol).all()), (float(err.max()), float((err / tol).max()))


def lens_of(kind, G, N, seed=0):
    if kind == "full":
        return torch.full((G,), N, dtype=torch.int32, device="cuda")
    lens = torch.randint(0, N + 1, (G,), device="cuda", generator=gen(seed)).int()
    lens[0] = 0                                       # a context of no rows, one of one, a full one
    if G > 1:
        lens[1] = 1
    if G > 2:
        lens[2] = N
    return lens


# ------------------------------------------------------------------ writing and reading

WRITES = [(1, 1, 16, 1), (1, 3, 32, 63), (2, 2, 64, 64), (3, 1, 32, 65), (4, 3, 16, 200), (5, 2, 64, 333), (1, 6, 32, 1025)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("shape", WRITES, ids=str)
@pytest.mark.parametrize("kind", ["full", "ragged"])
def test_written_cache_is_the_definition(shape, dtype, kind):
    G, H, D, N = shape
    k, v = rows(1, G, H, N, D, dtype)
    lens = lens_of(kind, G, N)
    cache = cc().quantize_context(k, v, lens=None if kind == "full" else lens, capacity=N + 70)
    ck, cv, s, _ = quantized(k, v, lens, cache.capacity // BLOCK)
    check_fields(cache, ck, cv, s, lens)
    unused = ~(torch.arange(cache.capacity // BLOCK, device="cuda") * BLOCK < lens[:, None])[:, None, :, None]
    assert not bool((cache.scales * unused).any()) and not bool((cache.bounds * unused[..., None]).any())
    want = [torch.where((torch.arange(N, device="cuda") < lens[:, None])[:, None, :, None], x[:, :, :N], 0.0) for x in values(cache)]
    for t in (torch.float32, torch.bfloat16):
        for got, x in zip(cc().read_context(cache, dtype=t), want):
            assert got.dtype is t and bool(((got.double() - x).abs() <= x.abs() * (2.0 ** -24 + (2.0 ** -8 if t is torch.bfloat16 else 0))).all())


def test_rows_by_strides_and_odd_addresses():
    """Views of other layouts: [N,H,D] tokens, a slice of a fused projection at an odd address, one row expanded."""
    c = cc()
    for dtype in (torch.float32, torch.bfloat16):
        big = rows(3, 1, 1, 130, 3 * 2 * 32 + 1, dtype)[0][0, 0]      # rows of odd pitch
        k, v = (big[:, 1 + i * 64:1 + (i + 1) * 64].unflatten(1, (2, 32)).transpose(0, 1) for i in (0, 1))
        for a, b in ((k, v), (k.transpose(-1, -2).contiguous().transpose(-1, -2), v), (k[:, :1].expand(2, 130, 32), v)):
            x, y = c.quantize_context(a, b), c.quantize_context(a.contiguous(), b.contiguous())
            assert torch.equal(x.codes, y.codes) and torch.equal(x.scales, y.scales) and torch.equal(x.bounds, y.bounds)


@pytest.mark.parametrize("size", [1e-44, 3e-39, 1e-30, 1.0, 3e38])
def test_every_magnitude(size):
    """Subnormal rows, whose step has few bits, to the largest; a block of zeros beside them."""
    k, v = rows(4, 1, 2, 128, 32, torch.float32)
    k, v = ((x / x.abs().max()).double().mul(size).float() for x in (k, v))
    k[:, 0, 64:] = 0
    cache = cc().quantize_context(k, v)
    ck, cv, s, _ = quantized(k, v, cache.lens, 2)
    check_fields(cache, ck, cv, s, cache.lens)
    assert bool((cache.scales[:, 0, 1, 0] == 0).all())


def test_rounding_at_ties_and_next_to_them():
    """A largest magnitude of 127 makes the step 1: halves are ties (to even), their neighbours are not."""
    half = torch.arange(-126, 126, device="cuda").float() + 0.5
    x = torch.cat([half, torch.nextafter(half, half + 1), torch.nextafter(half, half - 1), half.new_tensor([127.0])])
    x = torch.nn.functional.pad(x, (0, 1024 - x.numel())).view(1, 1, 64, 16)
    cache = cc().quantize_context(x, -x)
    k, v, s = fields(cache)
    assert bool((s == 1).all())
    assert torch.equal(k.view_as(x), x.double().round()) and torch.equal(v.view_as(x), -x.double().round())


def test_rows_behind_the_lengths_are_not_read_and_values_that_are_not_finite_show():
    c = cc()
    k, v = rows(5, 3, 2, 100, 32, torch.float32)
    lens = torch.tensor([100, 70, 64], dtype=torch.int32, device="cuda")
    want = c.quantize_context(k, v, lens=lens)
    k2, v2 = k.clone(), v.clone()
    for g in (1, 2):
        k2[g, :, int(lens[g]):], v2[g, :, int(lens[g]):] = float("nan"), float("inf")
    got = c.quantize_context(k2, v2, lens=lens)
    assert torch.equal(got.codes[0], want.codes[0]) and torch.equal(got.scales, want.scales) and torch.equal(got.bounds, want.bounds)
    q = torch.randn(3, 2, 1, 32, device="cuda", generator=gen(1))
    assert all(torch.equal(a, b) for a, b in zip(c.context_cache_attention(q, got), c.context_cache_attention(q, want)))
    k2 = k.clone()
    k2[0, 1, 80, 3] = float("inf")
    v2 = v.clone()
    v2[1, 0, 2, 0] = float("nan")
    bad = c.quantize_context(k2, v2, lens=lens)
    nan = torch.isnan(bad.scales)
    assert bool(nan[0, 1, 1, 0]) and bool(nan[1, 0, 0, 1]) and int(nan.sum()) == 2
    out, lse = c.context_cache_attention(q, bad)
    ref, rlse = c.context_cache_attention(q, want)
    wrong = torch.zeros(3, 2, dtype=torch.bool, device="cuda")
    wrong[0, 1] = wrong[1, 0] = True
    assert bool(torch.isnan(out[wrong]).all()) and torch.equal(out[~wrong], ref[~wrong])
    assert bool(torch.isnan(lse[0, 1]).all()) and torch.equal(lse[1], rlse[1])
    assert c.select_context_blocks(q, bad, 1)[0, 1].item() == 1          # a block that is wrong ranks first
    c.append_context(bad, k[:, :, :1], v[:, :, :1], start=lens)
    assert torch.equal(torch.isnan(bad.scales), nan)


def _append_reference(state, k, v, start, counts, cap):
    """state: ck, cv, scales (64 bits), lens; rows start[g] .. take the first counts[g] new rows."""
    ck, cv, s, lens = (x.clone() for x in state)
    G, H, n, D = k.shape
    for g in range(G):
        a = int(start[g])
        e = min(a + int(counts[g]), cap)
        for b in range(a // BLOCK, (e + BLOCK - 1) // BLOCK if e > a else 0):
            lo, hi = max(a, b * BLOCK), min(e, (b + 1) * BLOCK)
            for i, (c, x) in enumerate(((ck, k), (cv, v))):
                new = x[g, :, lo - a:hi - a].double()                              # [H, rows, D]
                was = s[g, :, b, i] if lo > b * BLOCK else torch.zeros_like(s[g, :, b, i])
                now = torch.maximum(was, step(new.abs().amax((-1, -2))))
                div = torch.where(now > 0, now, 1.0)[:, None, None]
                old = c[g, :, b, :lo - b * BLOCK]
                c[g, :, b, :lo - b * BLOCK] = (old * was[:, None, None] / div).round().clamp(-127, 127)
                c[g, :, b, lo - b * BLOCK:hi - b * BLOCK] = (new / div).round().clamp(-127, 127)
                s[g, :, b, i] = now
        lens[g] = e
    return ck, cv, s, lens


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("shape", [(1, 1, 16), (3, 2, 32), (4, 3, 64)], ids=str)
def test_rows_appended_step_by_step(shape, dtype):
    """One row, none, several blocks at once, different counts, rows taken back, up to and over the capacity."""
    c = cc()
    G, H, D = shape
    cap = 320
    k, v = rows(6, G, H, 40, D, dtype)
    lens = lens_of("ragged", G, 40) if G > 1 else lens_of("full", G, 40)
    cache = c.quantize_context(k, v, lens=lens, capacity=cap)
    ck, cv, s, _ = quantized(k, v, lens, cap // BLOCK)
    state = (ck, cv, s, lens.long())
    g = torch.Generator().manual_seed(2)
    for i, n in enumerate((1, 1, 130, 0, 23, 1, 64, 7, 100, 200)):
        k, v = rows(10 + i, G, H, n, D, dtype)
        k, v = k * (1 + 0.3 * i), v * (1 - 0.05 * i)             # scales that rise, scales that stay
        counts = torch.randint(0, n + 1, (G,), generator=g).cuda() if i % 3 == 2 else torch.full((G,), n, device="cuda")
        start = None
        if i in (4, 7, 9):
            start = (state[3].cpu() * torch.rand(G, generator=g)).long().cuda() if i != 9 else state[3]
        if start is None and int((state[3] + counts).max()) > cap:
            start = state[3] // 2
        c.append_context(cache, k.to(dtype), v.to(dtype), counts=counts if i % 3 == 2 else None, start=start)
        if n or start is not None:
            state = _append_reference(state, k.to(dtype), v.to(dtype), state[3] if start is None else start, counts, cap)
        check_fields(cache, *state)
        assert int(state[3].max()) <= cache.length


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("shape", [(1, 1, 16), (7, 3, 32), (5, 2, 64), (1, 16, 64), (3, 17, 32)], ids=str)
def test_single_rows_one_after_another(shape, dtype):
    """The step of a decode over more than two blocks: scales that rise and stay, contexts that take no row, rows that
    are taken back, rows of zeros, from strided tensors; the last rows one beyond the capacity."""
    c = cc()
    G, H, D = shape
    cap = 192
    k, v = rows(100, G, H, 50, D, dtype)
    lens = torch.arange(G, device="cuda").int() * 13 % 50
    cache = c.quantize_context(k, v, lens=lens, capacity=cap)
    ck, cv, s, _ = quantized(k, v, lens, cap // BLOCK)
    state = (ck, cv, s, lens.long())
    kn, vn = rows(101, G, H, 150, D, dtype)
    grow = (1 + torch.arange(150, device="cuda") / 60)[:, None]
    kn, vn = (kn * grow).to(dtype), (vn / grow).to(dtype)
    kn[:, :, 20] = 0
    g = torch.Generator().manual_seed(3)
    for i in range(150):
        counts = torch.randint(0, 4, (G,), generator=g).clamp(max=1).cuda() if i % 5 == 3 else torch.ones(G, dtype=torch.long, device="cuda")
        start = (state[3] - 2).clamp(min=0) if i % 17 == 16 else None
        if int((state[3] if start is None else start).max()) + 1 > cap:
            start = state[3] if i % 2 else state[3] // 3
        c.append_context(cache, kn[:, :, i:i + 1], vn[:, :, i:i + 1], counts=counts, start=start)
        state = _append_reference(state, kn[:, :, i:i + 1], vn[:, :, i:i + 1], state[3] if start is None else start, counts, cap)
        if i % 7 == 0 or i > 120 or start is not None:
            check_fields(cache, *state)


def test_a_full_cache_refuses_rows_and_looks_its_lengths_up_before():
    c = cc()
    k, v = rows(7, 2, 2, 100, 32, torch.float32)
    cache = c.quantize_context(k, v, lens=[100, 3], capacity=128)
    for _ in range(40):                                      # the host's bound passes the capacity, the rows do not
        c.append_context(cache, k[:, :, :1], v[:, :, :1], counts=[0, 1])
    assert cache.lens.tolist() == [100, 43]
    before = cache.codes.clone()
    with pytest.raises(ValueError, match="capacity"):
        c.append_context(cache, k[:, :, :29], v[:, :, :29])
    with pytest.raises(ValueError, match="capacity"):
        c.append_context(cache, k[:, :, :29], v[:, :, :29], counts=[29, 0])
    assert cache.lens.tolist() == [100, 43] and torch.equal(before, cache.codes)
    c.append_context(cache, k[:, :, :28], v[:, :, :28])
    assert cache.lens.tolist() == [128, 71]
    c.append_context(cache, k[:, :, :50], v[:, :, :50], counts=cache.lens // 100, start=cache.lens)   # [1, 0] rows: one beyond
    assert cache.lens.tolist() == [128, 71]
    c.append_context(cache, k, v, counts=cache.lens, start=torch.zeros_like(cache.lens))
    assert cache.lens.tolist() == [100, 71]                  # counts beyond the rows given are cut


def test_rows_read_from_anywhere():
    c = cc()
    k, v = rows(8, 3, 2, 300, 64, torch.bfloat16)
    cache = c.quantize_context(k, v, lens=[300, 130, 0], capacity=400)
    whole = c.read_context(cache, n=1000)
    assert torch.equal(whole[0], torch.nn.functional.pad(c.read_context(cache)[0], (0, 0, 0, 700)))
    for n in (1, 5, 64, 65, 200):
        for start in ([0, 0, 0], [63, 64, 1], [250, 129, 399], [299, 700, 5000]):
            for got, x in zip(c.read_context(cache, start=start, n=n), whole):
                x = torch.nn.functional.pad(x, (0, 0, 0, 6000))
                assert torch.equal(got, torch.stack([x[g, :, a:a + n] for g, a in enumerate(start)]))
    empty = c.quantize_context(k[:, :, :0], v[:, :, :0], capacity=10)
    assert empty.capacity == 64 and empty.length == 0 and c.read_context(empty)[0].shape == (3, 2, 0, 64)
    c.append_context(empty, k[:, :, :9], v[:, :, :9])
    assert empty.lens.tolist() == [9, 9, 9]


# ------------------------------------------------------------------ attention

# shared, B, H, D, N, Lq
ATTENTION = [(True, 1, 1, 16, 1, 1), (True, 3, 2, 32, 63, 1), (False, 3, 2, 32, 64, 2), (True, 2, 3, 64, 65, 5),
             (False, 5, 2, 16, 200, 1), (False, 9, 1, 64, 333, 9), (True, 17, 2, 32, 1000, 1), (True, 1, 2, 32, 5003, 1),
             (False, 2, 1, 64, 4100, 3), (True, 40, 6, 32, 700, 2), (True, 300, 2, 32, 450, 1), (True, 70, 1, 64, 1500, 3),
             (True, 1, 2, 64, 20000, 300), (True, 257, 1, 16, 130, 2), (False, 3, 2, 32, 900, 150),
             (True, 1100, 2, 32, 1500, 2), (False, 6, 3, 16, 1700, 500), (True, 900, 1, 64, 4100, 3)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("case", ATTENTION, ids=str)
def test_attention_over_the_cache(case, dtype, form):
    shared, B, H, D, N, L = case
    G = 1 if shared else B
    k, v = rows(20, G, H, N, D, dtype)
    lens = lens_of("full" if shared else "ragged", G, N)
    cache = cc().quantize_context(k, v, lens=lens, capacity=N + 100)
    q = torch.randn(B, H, L, D, device="cuda", generator=gen(21)).to(dtype)
    check_attention(cc().context_cache_attention(q, cache), attention(q, cache, D ** -0.5), dtype, D)


@pytest.mark.parametrize("B", [2, 200])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_scales_of_scores_and_magnitudes(dtype, B, form):
    """Any factor of the scores, negative and zero too; scores far apart between blocks; values and queries of extreme size."""
    c = cc()
    k, v = rows(22, 1, 2, 500, 32, dtype)
    q = torch.randn(B, 2, 3, 32, device="cuda", generator=gen(23)).to(dtype)
    cache = c.quantize_context(k, v)
    for scale in (-0.4, 0.0, 1e-3, 2.5):
        check_attention(c.context_cache_attention(q, cache, scale=scale), attention(q, cache, scale), dtype, 32)
    steps = torch.repeat_interleave(torch.tensor([1e-3, 30.0, 0.1, 200.0, 1.0, 5.0, 0.0, 9.0], device="cuda"), 64)[:500, None]
    for a, b, m in ((k * steps, v * steps, 1.0), (k, v * 1e-30, 1.0), (k * 1e-30, v * 1e30, 1e30), (k * 1e20, v, 1e-20)):
        cache = c.quantize_context(a.to(dtype), b.to(dtype))
        x = (q.double() * m).to(dtype)
        check_attention(c.context_cache_attention(x, cache), attention(x, cache, 32 ** -0.5), dtype, 32)


@pytest.mark.parametrize("B", [2, 100])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_values_that_are_not_finite_leave_the_weights_sound(dtype, B, form):
    c = cc()
    k, v = rows(28, 1, 3, 300, 32, dtype)
    q = torch.randn(B, 3, 1, 32, device="cuda", generator=gen(29)).to(dtype)
    sound = c.quantize_context(k, v)
    want = attention(q, sound, 32 ** -0.5)
    v[0, 1, 200, 3], k[0, 2, 0, 0] = float("nan"), float("-inf")
    out, lse = c.context_cache_attention(q, c.quantize_context(k, v))
    # the value scales of a head are factors of its numerators, taken out of their sum again: not the same bits as with
    # sound values, but the same bound.  Head 1's outputs are NaN, so the sound ones stand in for them here.
    assert bool(torch.isnan(out[:, 1:]).all()) and bool(torch.isnan(lse[:, 2]).all())
    mixed = torch.where(torch.isnan(out), want[0].to(dtype), out), torch.where(torch.isnan(lse), want[1].float(), lse)
    check_attention(mixed, want, dtype, 32)
    v[0, 1], k[0, 2] = v[0, 1] * 0, k[0, 2] * 0               # a head of zero values, one of zero keys
    v[0, 1, 200, 3] = k[0, 2, 0, 0] = 0.0
    cache = c.quantize_context(torch.nan_to_num(k), torch.nan_to_num(v))
    check_attention(c.context_cache_attention(q, cache), attention(q, cache, 32 ** -0.5), dtype, 32)


@pytest.mark.parametrize("D", [16, 32, 64])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_scores_that_rise_from_block_to_block_and_within(dtype, D, form):
    """Keys along one direction, longer from row to row, in steps far beyond the range of a half-precision numerator, up, down
    and in between; half of the queries point the other way."""
    c = cc()
    g = gen(36)
    N, B, H = 700, 200, 4
    axis = torch.randn(D, device="cuda", generator=g)
    axis = axis / axis.norm()
    n = torch.arange(N, device="cuda").float()
    length = torch.stack([n / 4, 175 - n / 4, 40 * torch.sin(n / 20), torch.where(n % 64 < 32, 0.0, n / 8)])       # [H,N]
    k = (length[None, :, :, None] * axis + 0.1 * torch.randn(1, H, N, D, device="cuda", generator=g)).to(dtype)
    v = torch.randn(1, H, N, D, device="cuda", generator=g).to(dtype)
    sign = torch.where(torch.arange(B, device="cuda") % 2 == 0, 1.0, -1.0)[:, None, None, None]
    q = (sign * axis * (0.5 + torch.rand(B, H, 1, 1, device="cuda", generator=g)) * D ** 0.5
         + 0.1 * torch.randn(B, H, 1, D, device="cuda", generator=g)).to(dtype)
    cache = c.quantize_context(k, v)
    check_attention(c.context_cache_attention(q, cache), attention(q, cache, D ** -0.5), dtype, D)
    few = c.context_cache_attention(q[:3], cache)
    check_attention(few, attention(q[:3], cache, D ** -0.5), dtype, D)


@pytest.mark.parametrize("B", [3, 130])
def test_queries_by_strides_and_odd_addresses(B, form):
    c = cc()
    for dtype in (torch.float32, torch.bfloat16):
        k, v = rows(24, 1, 2, 300, 32, dtype)
        cache = c.quantize_context(k, v)
        base = torch.randn(B, 4, 2 * 32 + 1, device="cuda", generator=gen(25)).to(dtype)
        q = base[:, :, 1:].unflatten(2, (2, 32)).transpose(1, 2)              # token-major, odd pitch and address
        blocks = c.select_context_blocks(q.contiguous(), cache, 2)
        for x in (q, q.transpose(-1, -2).contiguous().transpose(-1, -2), q[:1].expand(B, -1, -1, -1)):
            y = x.contiguous()
            assert all(torch.equal(a, b) for a, b in zip(c.context_cache_attention(x, cache), c.context_cache_attention(y, cache)))
            assert torch.equal(c.select_context_blocks(x, cache, 2), c.select_context_blocks(y, cache, 2))
            assert all(torch.equal(a, b) for a, b in zip(c.block_context_attention(x, cache, blocks), c.block_context_attention(y, cache, blocks)))


def test_a_query_that_is_not_finite_stays_in_its_row(form):
    c = cc()
    for B in (4, 200):
        for dtype in (torch.float32, torch.bfloat16):
            k, v = rows(26, 1, 2, 300, 32, dtype)
            cache = c.quantize_context(k, v)
            q = torch.randn(B, 2, 1, 32, device="cuda", generator=gen(27)).to(dtype)
            bad = q.clone()
            bad[1, 0, 0, 5] = float("nan")
            bad[2, 1, 0, 7] = float("inf")
            want, got = c.context_cache_attention(q, cache), c.context_cache_attention(bad, cache)
            hit = torch.zeros(B, 2, 1, dtype=torch.bool, device="cuda")
            hit[1, 0] = hit[2, 1] = True
            for a, b in zip(want, got):
                assert torch.equal(a[~hit], b[~hit]) and not bool(torch.isfinite(b[1, 0]).any())
            index, ref = c.select_context_blocks(bad, cache, 2), c.select_context_blocks(q, cache, 2)
            assert torch.equal(index[~hit], ref[~hit]) and bool((index[hit] == torch.tensor([0, 1], device="cuda")).all())


# ------------------------------------------------------------------ selection

def chosen(q, cache, n):
    G, H, nb = cache.scales.shape[:3]
    B, _, L, D = q.shape
    x = q.double()
    r = step(x.abs().amax(-1, keepdim=True))
    qi = torch.where(r > 0, x / r, 0.0).round().clamp(-127, 127)[:, :, :, None]                   # [B,H,L,1,D]
    lo, hi = (cache.bounds[..., i, :].double().expand(B, H, nb, D)[:, :, None] for i in (0, 1))
    score = (torch.maximum(qi * lo, qi * hi).sum(-1).float() * cache.scales[..., 0].expand(B, H, nb)[:, :, None]).double()
    held = ((cache.lens + 63) // 64).expand(B)
    out = torch.full((B, H, L, n), -1, dtype=torch.int32)
    score, held = score.cpu(), held.cpu()
    for b in range(B):
        m = min(n, int(held[b]))
        if m:
            order = torch.sort(score[b, ..., :int(held[b])], dim=-1, descending=True, stable=True).indices[..., :m]
            out[b, ..., :m] = order.sort(-1).values.int()
    return out.cuda()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("case", [(True, 1, 1, 16, 1, 1), (False, 3, 2, 32, 640, 2), (True, 2, 3, 64, 2100, 5),
                                  (True, 40, 2, 32, 5000, 1), (False, 5, 2, 64, 1300, 17), (True, 1, 1, 32, 70000, 3)], ids=str)
def test_chosen_blocks(case, dtype):
    shared, B, H, D, N, L = case
    k, v = rows(30, 1 if shared else B, H, N, D, dtype)
    lens = lens_of("full" if shared else "ragged", 1 if shared else B, N)
    cache = cc().quantize_context(k, v, lens=lens, capacity=N + 100)
    q = torch.randn(B, H, L, D, device="cuda", generator=gen(31)).to(dtype)
    for n in (1, 2, 7, 33, 90):
        assert torch.equal(cc().select_context_blocks(q, cache, n), chosen(q, cache, n)), n


def test_equal_bounds_go_to_the_lower_index():
    c = cc()
    k, v = rows(32, 1, 2, 64, 32, torch.float32)
    cache = c.quantize_context(k.repeat(1, 1, 50, 1), v.repeat(1, 1, 50, 1))
    q = torch.randn(5, 2, 1, 32, device="cuda", generator=gen(33))
    q[0] = 0                                                  # and a query of zeros, for which all are equal
    for n in (1, 3, 40, 49):
        assert bool((c.select_context_blocks(q, cache, n) == torch.arange(n, device="cuda")).all())
    two = c.quantize_context(torch.cat([k, k * 0.5, k, k * 0.25, k], 2), torch.cat([v] * 5, 2))
    pos = (q @ k.transpose(-1, -2)).amax(-1) > 0
    got = c.select_context_blocks(q[1:], two, 2)
    assert torch.equal(got, chosen(q[1:], two, 2)) and bool((got[pos[1:]] == torch.tensor([0, 2], device="cuda")).all())


def test_the_largest_bound_is_a_bound():
    """No score of a row exceeds its block's bound by more than the rounding of the query (half a step of 1 / 127)."""
    k, v = rows(34, 1, 2, 640, 32, torch.float32)
    cache = cc().quantize_context(k, v)
    q = torch.randn(6, 2, 1, 32, device="cuda", generator=gen(35)).double()
    ck, _, s = fields(cache)
    r = step(q.abs().amax(-1, keepdim=True))
    qi = (q / r).round()
    lo, hi = (cache.bounds[..., i, :].double() for i in (0, 1))
    bound = torch.maximum(qi[:, :, 0, None] * lo, qi[:, :, 0, None] * hi).sum(-1)                # [B,H,blocks]
    score = torch.einsum("bhd,hnrd->bhnr", (q / r)[:, :, 0], ck[0])
    slack = 0.5 * ck[0].abs().sum(-1).amax(-1)
    assert bool((score.amax(-1) <= bound + slack).all())


# ------------------------------------------------------------------ attention over listed blocks

def times_of(blocks, nb):
    B, H, L, S = blocks.shape
    t = torch.zeros(B, H, L, nb + 1, device="cuda", dtype=torch.float64)
    i = torch.where((blocks < 0) | (blocks >= nb), nb, blocks).long()
    return t.scatter_add_(3, i, torch.ones_like(i, dtype=torch.float64))[..., :nb]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("case", [(True, 1, 1, 16, 1, 1, 1), (False, 4, 2, 32, 640, 2, 5), (True, 3, 3, 64, 2100, 5, 20),
                                  (True, 200, 6, 32, 3000, 2, 16), (False, 5, 2, 64, 1300, 1, 64), (True, 2, 1, 32, 5000, 1, 1),
                                  (False, 3, 2, 64, 900, 250, 7), (True, 700, 2, 16, 500, 1, 9), (True, 1, 1, 32, 64, 9000, 1)], ids=str)
def test_attention_over_listed_blocks(case, dtype, form):
    """Chosen blocks; any list: none (-1), indices that are no block in use, the same one twice."""
    c = cc()
    shared, B, H, D, N, L, S = case
    G = 1 if shared else B
    k, v = rows(40, G, H, N, D, dtype)
    lens = lens_of("full" if shared else "ragged", G, N)
    cache = c.quantize_context(k, v, lens=lens, capacity=N + 100)
    nb = cache.capacity // BLOCK
    q = torch.randn(B, H, L, D, device="cuda", generator=gen(41)).to(dtype)
    wild = torch.randint(-2, nb + 3, (B, H, L, S), device="cuda", generator=gen(42)).int()
    wild[0, 0, 0] = -1
    wild[-1, -1, -1] = 0
    for blocks in (c.select_context_blocks(q, cache, S), wild, wild + 2 ** 30):
        want = attention(q, cache, D ** -0.5, times_of(blocks, nb))
        check_attention(c.block_context_attention(q, cache, blocks), want, dtype, D)
    out, lse = c.block_context_attention(q, cache, wild[..., :0])
    assert not bool(out.any()) and bool((lse == float("-inf")).all())


# ------------------------------------------------------------------ together

@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("shared", [True, False])
def test_a_decode_step_on_a_growing_context(dtype, shared, form):
    """A cache is written, grows, its blocks are chosen, attended to and merged with private buffers: the attention
    over [listed rows of the cache, buffer rows] together."""
    from ar_tabpfn.model.triton_kernels import merge_attention_outputs, pytorch_buffer_attention
    c = cc()
    B, H, D, L, Nb = 6, 3, 32, 2, 20
    G = 1 if shared else B
    k, v = rows(50, G, H, 700, D, dtype)
    cache = c.quantize_context(k, v, lens=lens_of("full" if shared else "ragged", G, 700), capacity=1024)
    for i in range(3):
        c.append_context(cache, *rows(51 + i, G, H, 40 + i, D, dtype))
    q = torch.randn(B, H, L, D, device="cuda", generator=gen(55)).to(dtype)
    kb, vb = rows(56, B, H, Nb, D, dtype)
    blocks = c.select_context_blocks(q, cache, 4)
    part = c.block_context_attention(q, cache, blocks)
    got = merge_attention_outputs(*part, *pytorch_buffer_attention(q, kb, vb))
    o, l, A, vmax, N = attention(q, cache, D ** -0.5, times_of(blocks, cache.capacity // BLOCK))
    s = q.double() @ kb.double().transpose(-1, -2) * D ** -0.5
    lb = torch.logsumexp(s, -1)
    ob = torch.softmax(s, -1) @ vb.double()
    both = torch.logaddexp(l, lb)
    want = o * torch.exp(l - both)[..., None] + ob * torch.exp(lb - both)[..., None]
    # two partial results of the type (half a step each, and the buffer pass's own numerators), and the merged one's half
    big = max(vmax, float(vb.abs().max()))
    tol = big * (4 * torch.finfo(dtype).eps + 4 * (D + 8) * U * max(A, float(s.abs().max()) * 8) + 300 * U)
    assert bool(((got.double() - want).abs() <= tol).all()), float((got.double() - want).abs().max() / tol)
    full = c.context_cache_attention(q, cache)
    every = torch.arange(16, dtype=torch.int32, device="cuda").expand(B, H, L, 16)
    check_attention(c.block_context_attention(q, cache, every), attention(q, cache, D ** -0.5), dtype, D)
    check_attention(full, attention(q, cache, D ** -0.5), dtype, D)


def test_the_same_bits_again_on_another_stream_and_in_a_graph(form):
    """A decode step captured once and replayed: lengths grow on the device, the launches stay."""
    c = cc()
    B, H, D = 5, 2, 32
    k, v = rows(60, B, H, 130, D, torch.bfloat16)
    kn, vn = rows(61, B, H, 1, D, torch.bfloat16)
    q = torch.randn(B, H, 2, D, device="cuda", generator=gen(62)).bfloat16()

    def step_of(cache):
        c.append_context(cache, kn, vn)
        index = c.select_context_blocks(q, cache, 2)
        return (*c.context_cache_attention(q, cache), index, *c.block_context_attention(q, cache, index))
    eager, other, replayed = (c.quantize_context(k, v, capacity=256) for _ in range(3))
    want = [step_of(eager) for _ in range(70)]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = [step_of(other) for _ in range(70)]
    side.synchronize()
    for a, b in zip(want, got):
        assert all(torch.equal(x, y) for x, y in zip(a, b))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step_of(replayed)
    for i in range(70):
        graph.replay()
        assert all(torch.equal(x, y) for x, y in zip(want[i], out)), i
    assert torch.equal(replayed.codes, eager.codes) and replayed.lens.tolist() == [200] * B
    for _ in range(100):                                      # past the capacity: rows are left out, nothing else is written
        graph.replay()
    assert replayed.lens.tolist() == [256] * B


def test_a_cache_put_together_from_its_tensors():
    c = cc()
    k, v = rows(70, 2, 2, 500, 64, torch.float32)
    a = c.quantize_context(k, v, lens=[500, 77])
    b = c.ContextCache(a.codes.clone(), a.scales.clone(), a.bounds.clone(), a.lens.clone())
    assert b.length == b.capacity == 512
    q = torch.randn(2, 2, 3, 64, device="cuda", generator=gen(71))
    got, want = c.context_cache_attention(q, b), attention(q, a, 0.125)
    check_attention(got, want, torch.float32, 64)
    assert torch.equal(c.select_context_blocks(q, a, 3), c.select_context_blocks(q, b, 3))
    assert c.context_cache_attention(q[:, :, :0], a)[0].shape == (2, 2, 0, 64)


def test_offsets_beyond_32_bits():
    """A cache of more than 2^32 code bytes: the last context is where it should be."""
    c = cc()
    G, H, D, blocks = 70, 8, 64, 1000
    codes = torch.full((G, H, blocks, 2, 64 * D), 128, dtype=torch.uint8, device="cuda")
    assert codes.numel() > 2 ** 32
    cache = c.ContextCache(codes, torch.zeros(G, H, blocks, 2, device="cuda"),
                           torch.zeros(G, H, blocks, 2, D, dtype=torch.float16, device="cuda"),
                           torch.full((G,), blocks * 64, dtype=torch.int32, device="cuda"))
    k, v = rows(72, 1, H, 100, D, torch.bfloat16)
    small = c.quantize_context(k, v)
    at = torch.zeros(G, dtype=torch.int32, device="cuda")
    at[-1] = blocks * 64 - 128
    c.append_context(cache, k.expand(G, H, 100, D), v.expand(G, H, 100, D), start=at)
    assert cache.lens.tolist() == [100] * (G - 1) + [blocks * 64 - 28]
    assert torch.equal(cache.codes[-1, :, -2:], small.codes[0]) and torch.equal(cache.codes[0, :, :2], small.codes[0])
    got = c.read_context(cache, start=at, n=100)
    assert all(torch.equal(a[-1], b[0]) for a, b in zip(got, c.read_context(small)))
    q = torch.randn(G, H, 1, D, device="cuda", generator=gen(73)).bfloat16()
    index = torch.full((G, H, 1, 2), -1, dtype=torch.int32, device="cuda")
    index[-1] = torch.tensor([blocks - 2, blocks - 1], dtype=torch.int32, device="cuda")
    out, lse = c.block_context_attention(q, cache, index)
    ref, rlse = c.context_cache_attention(q[-1:], small)
    assert bool((out[:-1] == 0).all())
    U16 = 2.0 ** -8
    assert bool(((out[-1:] - ref).abs().float() <= 2 * U16 * ref.abs().float().clamp(min=float(v.abs().max()) * 2.0 ** -3)).all())
    assert bool(((lse[-1:] - rlse).abs() <= 1e-4).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("D", [16, 32, 64])
def test_a_wait_that_runs_out_gives_nan_and_the_next_call_is_right(D, dtype):
    """The tensor-core form of many queries with its "scores ready" signal withheld and a limit of 0.1 ms."""
    from ar_tabpfn import _lib
    c, lib = cc(), _lib.lib()
    k, v = rows(80, 1, 6, 6000, D, dtype)
    cache = c.quantize_context(k, v)
    q = torch.randn(3000, 6, 1, D, device="cuda", generator=gen(81)).to(dtype)   # far beyond the few-row kernel's range
    want = c.context_cache_attention(q, cache)
    try:
        _lib.check(lib.artab_debug_set(_lib.DEBUG_WAIT_CYCLES, 200_000))
        _lib.check(lib.artab_debug_set(_lib.DEBUG_DROP_SCORE_COMMITS, 1))
        out, lse = c.context_cache_attention(q, cache)
        torch.cuda.synchronize()
    finally:
        lib.artab_debug_set(_lib.DEBUG_DROP_SCORE_COMMITS, 0)
        lib.artab_debug_set(_lib.DEBUG_WAIT_CYCLES, 0)
    assert bool(torch.isnan(out).all()) and bool(torch.isnan(lse).all())
    assert all(torch.equal(a, b) for a, b in zip(want, c.context_cache_attention(q, cache)))


def test_two_graphs_with_workspaces_replayed_in_turn():
    """Attention over listed blocks by block, captured for two caches: each graph has its own partial results."""
    c = cc()
    outs, wants, graphs = [], [], []
    for seed in (90, 91):
        k, v = rows(seed, 1, 2, 1000, 32, torch.float32)
        cache = c.quantize_context(k, v)
        q = torch.randn(600, 2, 1, 32, device="cuda", generator=gen(seed))
        blocks = c.select_context_blocks(q, cache, 8)
        from ar_tabpfn import _lib
        assert _lib.lib().artab_cache_block_workspace(cache._ref, 600, 1, 8) > 0
        wants.append((blocks, c.block_context_attention(q, cache, blocks)))
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append((c.select_context_blocks(q, cache, 8), c.block_context_attention(q, cache, blocks), (cache, q)))
        graphs.append(g)
    for i in (0, 1, 1, 0, 1, 0):
        outs[i][1][0].zero_()
        graphs[i].replay()
        if i:
            graphs[0].replay()
        assert torch.equal(outs[i][0], wants[i][0]) and all(torch.equal(a, b) for a, b in zip(outs[i][1], wants[i][1]))


def test_many_rows_again_and_on_another_stream(form):
    """The forms of many queries: the same bits twice, and on a side stream while another call runs."""
    c = cc()
    for dtype in (torch.float32, torch.bfloat16):
        k, v = rows(95, 1, 3, 2500, 32, dtype)
        cache = c.quantize_context(k, v)
        q = torch.randn(700, 3, 2, 32, device="cuda", generator=gen(96)).to(dtype)
        want = c.context_cache_attention(q, cache)
        blocks = c.select_context_blocks(q, cache, 6)
        listed = c.block_context_attention(q, cache, blocks)
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in range(2)]
        got = []
        for s in streams * 3:
            with torch.cuda.stream(s):
                got.append((c.context_cache_attention(q, cache), c.block_context_attention(q, cache, blocks)))
        torch.cuda.synchronize()
        for a, b in got:
            assert all(torch.equal(x, y) for x, y in zip(a, want)) and all(torch.equal(x, y) for x, y in zip(b, listed))


# contexts x heads x rows for which few queries are spread in different ways: one warp a unit up to clusters of eight CTAs
SPREADS = [(512, 6, 200), (300, 8, 700), (64, 6, 700), (96, 4, 2000), (20, 8, 8000), (8, 8, 9000), (8, 6, 8192), (1, 6, 8192),
           (3, 2, 300), (12, 8, 4096), (16, 8, 9000), (64, 6, 8192)]


@pytest.mark.parametrize("D", [16, 32, 64])
@pytest.mark.parametrize("case", SPREADS, ids=str)
def test_few_queries_however_the_rows_are_spread(case, D):
    G, H, N = case
    c = cc()
    k, v = rows(110, G, H, N, D, torch.bfloat16)
    cache = c.quantize_context(k, v, lens=lens_of("ragged" if G > 1 else "full", G, N))
    del k, v
    for dtype, L in ((torch.float32, 1), (torch.bfloat16, 1), (torch.bfloat16, 5)):
        q = torch.randn(G, H, L, D, device="cuda", generator=gen(111)).to(dtype)
        check_attention(c.context_cache_attention(q, cache), attention(q, cache, D ** -0.5), dtype, D)


@pytest.mark.parametrize("D", [16, 32, 64])
@pytest.mark.parametrize("case", [(64, 6, 2000, 4, 8), (200, 8, 900, 1, 4), (8, 6, 8192, 1, 32), (1, 6, 16384, 1, 64), (1, 6, 5000, 1, 9)], ids=str)
def test_listed_blocks_however_they_are_spread(case, D):
    G, H, N, L, S = case
    c = cc()
    k, v = rows(112, G, H, N, D, torch.bfloat16)
    cache = c.quantize_context(k, v, lens=lens_of("ragged" if G > 1 else "full", G, N))
    for dtype in (torch.float32, torch.bfloat16):
        q = torch.randn(G, H, L, D, device="cuda", generator=gen(113)).to(dtype)
        blocks = c.select_context_blocks(q, cache, S)
        check_attention(c.block_context_attention(q, cache, blocks), attention(q, cache, D ** -0.5, times_of(blocks, cache.capacity // BLOCK)), dtype, D)


@pytest.mark.parametrize("D", [16, 32, 64])
@pytest.mark.parametrize("case", [(1, 100, 300), (1, 100, 640), (1, 100, 1280), (1, 100, 2500), (1, 100, 5100), (1, 100, 8000), (2, 700, 2560),
                                  (3, 1000, 5100), (6, 1000, 300)], ids=str)
def test_many_rows_however_the_context_is_split(case, D, form):
    """Clusters of one, two, four, five and eight CTAs, with shares of blocks that are not equal."""
    H, L, N = case
    c = cc()
    k, v = rows(114, 1, H, N, D, torch.bfloat16)
    cache = c.quantize_context(k, v)
    for dtype in (torch.float32, torch.bfloat16):
        q = torch.randn(1, H, L, D, device="cuda", generator=gen(115)).to(dtype)
        check_attention(c.context_cache_attention(q, cache), attention(q, cache, D ** -0.5), dtype, D)


@pytest.mark.parametrize("p", [-118, -60, 0, 90])
def test_every_quotient_of_bf16_magnitudes(p):
    """Blocks whose largest magnitude is b 2^p, b = 128 .. 255, with every a 2^(p - i) up to it: among the quotients are all the
    ties and near ties that bf16 rows can have."""
    c = cc()
    a = torch.arange(1, 256, device="cuda", dtype=torch.float64)
    x = (a[None] * 2.0 ** -torch.arange(16, device="cuda", dtype=torch.float64)[:, None]).flatten()        # 4080 numbers
    x = torch.cat([x, torch.zeros(16, device="cuda", dtype=torch.float64)])
    b = torch.arange(128, 256, device="cuda", dtype=torch.float64)
    k = torch.where(x[None] <= b[:, None], x[None], x[None] / 2) * torch.where(torch.arange(4096, device="cuda") % 2 == 0, 1.0, -1.0)
    k[:, -1] = b
    k = (k * 2.0 ** p).view(128, 1, 64, 64).bfloat16()
    v = (k.float() * 0.5).bfloat16().flip(0)
    lens = torch.full((128,), 64, dtype=torch.int32, device="cuda")
    ck, cv, scales, _ = quantized(k, v, lens, 1)
    check_fields(c.quantize_context(k, v), ck, cv, scales, lens)


# ------------------------------------------------------------------ value scales far apart

def far_apart(seed, B, H, D, dtype, ratio, gap):
    """A cache of 300 rows whose values are `ratio` of those of one block (the first of every other head, else the third), and
    queries that score the rows of that block some `gap` below the others."""
    g = gen(seed)
    N = 300
    axis = torch.randn(D, device="cuda", generator=g)
    axis = axis / axis.norm()
    large = torch.zeros(H, N, dtype=torch.bool, device="cuda")
    large[0::2, :64] = True
    large[1::2, 128:192] = True
    k = 0.5 * torch.randn(H, N, D, device="cuda", generator=g) - gap * large[..., None] * axis
    v = torch.randn(H, N, D, device="cuda", generator=g) * torch.where(large, 1.0, ratio)[..., None]
    q = axis * D ** 0.5 + 0.2 * torch.randn(B, H, 1, D, device="cuda", generator=g)
    q = q - ((q @ axis)[..., None] - D ** 0.5) * axis                  # along the axis all the same
    return cc().quantize_context(k.to(dtype), v.to(dtype)), q.to(dtype), large


@pytest.mark.parametrize("ratio", [1e-3, 1e-5, 1e-7, 1e-8, 1e-9, 1e-20])
@pytest.mark.parametrize("B", [3, 200])
@pytest.mark.parametrize("D", [16, 32, 64])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_values_far_below_those_of_a_block_that_nothing_attends(dtype, D, B, ratio, form):
    """The block of large values has weights of exp(-40) * ratio or less: what is left of it is far below the bounds, which
    are those of check_attention over the small rows alone.  Exponents of up to log2(1 / ratio) < 67 are sums of
    numbers of that size, a weight then off by another 2^-17; the log-sum-exp is a difference of such numbers."""
    cache, q, large = far_apart(120, B, 2, D, dtype, ratio, 40.0 - math.log(ratio))
    seen = torch.nn.functional.pad(~large, (0, 20), value=False)[:, ::BLOCK]                # [H,blocks]
    o, l, _, _, N = attention(q, cache, D ** -0.5, seen[None, :, None].expand(B, -1, 1, -1))
    k, v = values(cache)
    small = ~large[None, :, :, None]
    k, v = k[:, :, :300] * small, v[:, :, :300] * small
    A = float((q.double().abs() @ k.abs().transpose(-1, -2)).max()) * D ** -0.5
    out, lse = cc().context_cache_attention(q, cache)
    far = 2.0 ** -17
    rel = 2 * (D + 8) * U * A + (N / 64 + 100) * U + far + (2.0 ** -11 if dtype is torch.bfloat16 else 0.0)
    err = (out.double() - o).abs()
    tol = float(v.abs().max()) * rel + o.abs() * torch.finfo(dtype).eps / 2
    assert bool((err <= tol).all()), (float(err.max()), float((err / tol).max()))
    err = (lse.double() - l).abs()
    tol = (D + 8) * U * A + (N / 64 + 100) * U + 4 * U * (l.abs() + A + 14) + 2 * far
    assert bool((err <= tol).all()), (float(err.max()), float((err / tol).max()))


@pytest.mark.parametrize("ratio", [1e-2, 1e-4, 1e-6])
@pytest.mark.parametrize("B", [3, 200])
@pytest.mark.parametrize("D", [16, 32, 64])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_small_values_beside_large_ones_of_as_small_a_weight(dtype, D, B, ratio, form):
    """Both kinds of rows make up the output: every row's share w |v| of it may be off by its weight's relative error."""
    cache, q, _ = far_apart(121, B, 2, D, dtype, ratio, -math.log(ratio))
    k, v = (x[:, :, :300] for x in values(cache))
    s = q.double() @ k.transpose(-1, -2) * D ** -0.5
    p = torch.softmax(s, -1)
    o, share = p @ v, p @ v.abs()
    A = float((q.double().abs() @ k.abs().transpose(-1, -2)).max()) * D ** -0.5
    rel = 2 * (D + 8) * U * A + 105 * U + 2.0 ** -17 + (2.0 ** -11 if dtype is torch.bfloat16 else 0.0)
    out, _ = cc().context_cache_attention(q, cache)
    err = (out.double() - o).abs()
    tol = share * rel + o.abs() * torch.finfo(dtype).eps / 2
    assert bool((err <= tol).all()), (float(err.max()), float((err / tol).max()))


@pytest.mark.parametrize("B", [3, 200])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("N", [50, 64, 300, 1500])
def test_values_that_are_not_finite_show_beside_nothing_but_zeros(N, dtype, B, form):
    """No block has a value scale that is a positive number: the only block, every block, or one beside blocks of zeros is
    not finite.  Outputs are NaN, the weights and so the log-sum-exp are sound."""
    c = cc()
    k, v = rows(130, 1, 3, N, 32, dtype)
    v[0, 0, ::7, 3] = float("nan")                                     # in every block
    v[0, 1], v[0, 1, N // 2, 0] = 0.0, float("-inf")                   # in one, zeros in the others
    v[0, 2] = 0.0                                                      # nothing wrong
    q = torch.randn(B, 3, 1, 32, device="cuda", generator=gen(131)).to(dtype)
    cache = c.quantize_context(k, v)
    out, lse = c.context_cache_attention(q, cache)
    assert bool(torch.isnan(out[:, :2]).all()) and bool((out[:, 2] == 0).all())
    sound = c.quantize_context(k, torch.zeros_like(v))
    want = attention(q, sound, 32 ** -0.5)
    check_attention((torch.zeros_like(out), lse), want, dtype, 32)


@pytest.mark.parametrize("size", [1e-37, 1e31, 1e34, 1e36])
@pytest.mark.parametrize("B", [3, 200])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_attended_values_near_the_ends_of_the_range(dtype, B, size, form):
    """Thirty rows of values up to some 3 size: even all of them at their largest add up to a finite number."""
    c = cc()
    k, v = rows(140, 1, 2, 30, 32, torch.float32)
    cache = c.quantize_context(k.to(dtype), (v.double() * size).to(dtype))
    q = torch.randn(B, 2, 2, 32, device="cuda", generator=gen(141)).to(dtype)
    want = attention(q, cache, 32 ** -0.5)
    assert want[3] * 30 < 3e38
    check_attention(c.context_cache_attention(q, cache), want, dtype, 32)
    listed = torch.zeros(B, 2, 2, 2, dtype=torch.int32, device="cuda")
    listed[..., 1] = -1
    check_attention(c.block_context_attention(q, cache, listed), want, dtype, 32)


@pytest.mark.parametrize("rise", [20.0, 24.6, 30.0, 37.0])
@pytest.mark.parametrize("D", [16, 32, 64])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_a_maximum_that_rises_within_a_block_keeps_its_other_rows(dtype, D, rise, form):
    """One block has a row some 2^9 above the weights before it, and one 2^rise above them whose values are zero in half of
    the channels: there the output is made of the other rows.  A numerator is rounded to a multiple of 2^-24 (the smallest half)
    where the largest row's is 2^5 at least: each is off by at most 2^-25 / 2^5 = 2^-30 of the largest weight, and the output by
    that times the sum of all |v|, beside what the weights themselves are off by."""
    c = cc()
    g = gen(150)
    B, H, N = 200, 2, 40 * BLOCK
    axis = torch.randn(D, device="cuda", generator=g)
    axis = axis / axis.norm()
    length = torch.zeros(N, device="cuda")
    length[20 * BLOCK + 40], length[20 * BLOCK + 3] = 9 * math.log(2), rise * math.log(2)
    k = (length[:, None] * axis).expand(1, H, N, D).to(dtype)
    v = torch.randn(1, H, N, D, device="cuda", generator=g)
    v[:, :, 20 * BLOCK + 3, D // 2:] = 0
    q = (axis * D ** 0.5 * (1 + 0.02 * torch.rand(B, H, 1, 1, device="cuda", generator=g))).to(dtype)
    cache = c.quantize_context(k, v.to(dtype))
    kk, vv = values(cache)
    s = q.double() @ kk.transpose(-1, -2) * D ** -0.5
    p = torch.softmax(s, -1)
    o, share = p @ vv, p @ vv.abs()
    A = float((q.double().abs() @ kk.abs().transpose(-1, -2)).max()) * D ** -0.5
    rel = 2 * (D + 8) * U * A + (N / 64 + 100) * U + 2.0 ** -17 + (2.0 ** -11 if dtype is torch.bfloat16 else 0.0)
    out, _ = c.context_cache_attention(q, cache)
    err = (out.double() - o).abs()
    tol = share * rel + o.abs() * torch.finfo(dtype).eps / 2 + 2.0 ** -30 * vv.abs().sum(2, keepdim=True)
    assert bool((err <= tol).all()), (float(err.max()), float((err / tol).max()))


@pytest.mark.parametrize("p", [-133, -127, -126, -125, -124])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_ties_at_steps_near_the_smallest_normal_number(dtype, p):
    """Blocks whose largest magnitude is b 2^p, b = 128 .. 255: steps on either side of 2^-126 and 2^-125, where a step or its half
    has fewer bits.  Written at once, appended, and each first row by itself; queries of such a size choose blocks."""
    c = cc()
    a = torch.arange(1, 256, device="cuda", dtype=torch.float64)
    x = (a[None] * 2.0 ** -torch.arange(16, device="cuda", dtype=torch.float64)[:, None]).flatten()        # 4080 numbers
    x = torch.cat([x, torch.zeros(16, device="cuda", dtype=torch.float64)])
    b = torch.arange(128, 256, device="cuda", dtype=torch.float64)
    k = torch.where(x[None] <= b[:, None], x[None], x[None] / 2) * torch.where(torch.arange(4096, device="cuda") % 2 == 0, 1.0, -1.0)
    k[:, 63] = b                                             # in the first row, that all but it may be appended to
    k = (k * 2.0 ** p).view(128, 1, 64, 64).to(dtype)
    v = (k.double() * 0.5).to(dtype).flip(0)
    lens = torch.full((128,), 64, dtype=torch.int32, device="cuda")
    ck, cv, scales, _ = quantized(k, v, lens, 1)
    check_fields(c.quantize_context(k, v), ck, cv, scales, lens)
    cache = c.quantize_context(k[:, :, :1], v[:, :, :1], capacity=64)
    one = quantized(k[:, :, :1], v[:, :, :1], lens.clamp(max=1), 1)
    check_fields(cache, *one[:3], lens.clamp(max=1))
    zero = torch.zeros_like(lens)
    c.append_context(cache, k, v, start=zero)
    check_fields(cache, ck, cv, scales, lens)
    c.append_context(cache, k[:, :, :1], v[:, :, :1], start=zero)
    check_fields(cache, *one[:3], lens.clamp(max=1))
    c.append_context(cache, k[:, :, 1:], v[:, :, 1:])
    check_fields(cache, *_append_reference(one[:3] + (lens.clamp(max=1),), k[:, :, 1:], v[:, :, 1:], lens.clamp(max=1), lens - 1, 64))
    keys = torch.randn(1, 1, 640, 64, device="cuda", generator=gen(160))
    other = c.quantize_context(keys, keys)
    q = k.reshape(128 * 64, 1, 1, 64)[::7]
    assert torch.equal(c.select_context_blocks(q, other, 3), chosen(q, other, 3))
