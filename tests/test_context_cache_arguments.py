"""Arguments of the 8-bit context cache, checked before anything reaches the device: the native entry points see
addresses only.  Also the host's side of lengths and capacities.  Runs without a GPU."""
import pytest
import torch

from ar_tabpfn import _lib
from ar_tabpfn.model import context_cache as cc

G, H, D, N = 3, 2, 32, 100


class FakeLibrary:
    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def call(*args):
            self.calls.append((name, args))
            return 0
        return call


@pytest.fixture
def fake(monkeypatch):
    """Calls are recorded, and host tensors pass for device tensors."""
    lib = FakeLibrary()

    class Launch:
        def __init__(self, device):
            pass

        def __enter__(self):
            return lib, None

        def __exit__(self, *exc):
            return False
    monkeypatch.setattr(cc, "_Launch", Launch)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    return lib


def tensors(blocks=2, g=G, h=H, d=D):
    return dict(codes=torch.zeros(g, h, blocks, 2, 64 * d, dtype=torch.uint8), scales=torch.zeros(g, h, blocks, 2),
                bounds=torch.zeros(g, h, blocks, 2, d, dtype=torch.float16), lens=torch.zeros(g, dtype=torch.int32))


def cache(**kw):
    return cc.ContextCache(**tensors(**kw))


@pytest.mark.parametrize("change", [
    dict(codes=torch.zeros(G, H, 2, 2, 64 * D)), dict(codes=torch.zeros(G, H, 2, 64 * D, dtype=torch.uint8)),
    dict(codes=torch.zeros(G, H, 2, 2, 64 * D + 1, dtype=torch.uint8)), dict(codes=torch.zeros(G, H, 2, 2, 64 * 48, dtype=torch.uint8)),
    dict(codes=torch.zeros(G, H, 2, 1, 64 * D, dtype=torch.uint8)), dict(codes=torch.zeros(G, H, 0, 2, 64 * D, dtype=torch.uint8)),
    dict(codes=torch.zeros(H, G, 2, 2, 64 * D, dtype=torch.uint8).transpose(0, 1)), dict(scales=torch.zeros(G, H, 3, 2)),
    dict(scales=torch.zeros(G, H, 2, 2, dtype=torch.float16)), dict(bounds=torch.zeros(G, H, 2, 2, D)),
    dict(bounds=torch.zeros(G, H, 2, D, dtype=torch.float16)), dict(lens=torch.zeros(G, dtype=torch.int64)),
    dict(lens=torch.zeros(G + 1, dtype=torch.int32)), dict(lens=torch.zeros(2 * G, dtype=torch.int32)[::2]),
], ids=lambda c: next(f"{k}{tuple(v.shape)}{v.dtype}" for k, v in c.items()))
def test_tensors_that_are_no_cache(change):
    cache()
    with pytest.raises(ValueError, match="ContextCache"):
        cc.ContextCache(**(tensors() | change))


@pytest.mark.parametrize("k,v,kw", [
    ((H, N, D), (H, N + 1, D), {}), ((N, D), (N, D), {}), ((H, N, 24), (H, N, 24), {}), ((H, N, 128), (H, N, 128), {}),
    ((G, H, N, D), (H, N, D), {}), ((H, N, D), (H, N, D), dict(capacity=N - 1)), ((H, 0, D), (H, 0, D), {}),
    ((0, H, N, D), (0, H, N, D), {}), ((G, H, N, D), (G, H, N, D), dict(lens=[N] * (G + 1))),
    ((G, H, N, D), (G, H, N, D), dict(lens=torch.ones(G))), ((G, H, N, D), (G, H, N, D), dict(lens=torch.ones(1, G, dtype=torch.int32))),
], ids=str)
def test_contexts_that_do_not_fit(fake, k, v, kw):
    with pytest.raises(ValueError):
        cc.quantize_context(torch.zeros(k), torch.zeros(v), **kw)
    assert not fake.calls


def test_types(fake):
    x = torch.zeros(H, N, D)
    for k, v in ((x, x.bfloat16()), (x.half(), x.half()), (x.double(), x.double()), (x.int(), x.int())):
        with pytest.raises(ValueError):
            cc.quantize_context(k, v)
    with pytest.raises(ValueError):
        cc.read_context(cache(), dtype=torch.float16)
    for op in (lambda q: cc.context_cache_attention(q, cache()), lambda q: cc.select_context_blocks(q, cache(), 1)):
        with pytest.raises(ValueError):
            op(torch.zeros(G, H, 1, D).half())
    assert not fake.calls


@pytest.mark.parametrize("q", [(G, H, D), (G, H + 1, 1, D), (G, H, 1, 16), (G + 1, H, 1, D), (1, H, 1, D)], ids=str)
def test_queries_that_do_not_fit(fake, q):
    q = torch.zeros(q)
    blocks = torch.zeros(*q.shape[:3], 2, dtype=torch.int32) if q.dim() == 4 else torch.zeros(1, dtype=torch.int32)
    for op in (lambda: cc.context_cache_attention(q, cache()), lambda: cc.select_context_blocks(q, cache(), 3),
               lambda: cc.block_context_attention(q, cache(), blocks)):
        with pytest.raises(ValueError):
            op()
    assert not fake.calls


def test_blocks_that_do_not_fit(fake):
    q = torch.zeros(G, H, 2, D)
    for blocks in (torch.zeros(G, H, 2, 3), torch.zeros(G, H, 2, 3, dtype=torch.int64), torch.zeros(G, H, 1, 3, dtype=torch.int32),
                   torch.zeros(G, H, 2, dtype=torch.int32), torch.zeros(1, H, 2, 3, dtype=torch.int32)):
        with pytest.raises(ValueError, match="blocks"):
            cc.block_context_attention(q, cache(), blocks)
    for n in (0, -1):
        with pytest.raises(ValueError):
            cc.select_context_blocks(q, cache(), n)
    with pytest.raises(ValueError):
        cc.read_context(cache(), n=-1)
    assert not fake.calls


@pytest.mark.parametrize("shape", [(H, 1, D), (G, H, 1, 16), (G, H + 1, 1, D), (G + 1, H, 1, D)], ids=str)
def test_rows_that_do_not_fit_a_cache(fake, shape):
    with pytest.raises(ValueError):
        cc.append_context(cache(), torch.zeros(shape), torch.zeros(shape))
    x = torch.zeros(G, H, 1, D)
    for kw in (dict(counts=[1, 1]), dict(start=torch.zeros(G)), dict(start=torch.zeros(G, dtype=torch.bool))):
        with pytest.raises(ValueError):
            cc.append_context(cache(), x, x, **kw)
    assert not fake.calls


def test_room_is_counted_before_rows_are_written(fake, monkeypatch):
    c = cc.ContextCache(**tensors(), length=100)
    x = torch.zeros(G, H, 20, D)
    c.lens.fill_(100)
    cc.append_context(c, x, x)                              # the fake leaves lens as it is
    assert c.length == 120 and len(fake.calls) == 1
    c.lens.fill_(120)
    with pytest.raises(ValueError, match="capacity"):
        cc.append_context(c, x, x)
    with pytest.raises(ValueError, match="capacity"):
        cc.append_context(c, x, x, counts=[0, 0, 9])
    cc.append_context(c, x, x, counts=[0, 8, 8])
    cc.append_context(c, x, x, start=[0, 0, 0])
    cc.append_context(c, x[:, :, :0], x[:, :, :0])          # nothing to do
    assert len(fake.calls) == 3
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(ValueError, match="capture"):
        cc.append_context(c, x, x)
    assert len(fake.calls) == 3


def test_views_are_passed_by_their_strides(fake):
    x = torch.zeros(N, 3, H, D)
    k, v = x[:, 0].transpose(0, 1), x[:, 1].transpose(0, 1)
    cc.quantize_context(k, v)
    args = fake.calls[-1][1]
    assert args[1] == k.data_ptr() and list(args[2])[1:] == [D, 3 * H * D] and args[3] == v.data_ptr()
    q = torch.zeros(G, 2, H, D).transpose(1, 2)
    cc.context_cache_attention(q, cache())
    assert fake.calls[-1][1][1] == q.data_ptr() and list(fake.calls[-1][1][2]) == list(q.stride()[:3])


def test_no_device_no_result():
    if torch.cuda.is_available():
        x = torch.zeros(H, N, D)
        with pytest.raises(ValueError, match="CUDA"):
            cc.quantize_context(x, x)
    else:
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            cc.quantize_context(torch.zeros(H, N, D), torch.zeros(H, N, D))


def test_the_library_refuses_what_does_not_fit_without_a_device():
    """The C entry points: codes, never exceptions or aborts."""
    import ctypes as C
    lib = _lib.load_library()
    p = 4096
    st = (C.c_int64 * 3)(1, 1, 1)
    good = lambda **kw: _lib.Cache(**(dict(n_groups=2, n_heads=2, head_dim=32, n_blocks=2, codes=p, scales=p, bounds=p, lens=p) | kw))
    bad = [good(n_groups=0), good(n_groups=70000), good(n_heads=0), good(head_dim=48), good(n_blocks=0), good(n_blocks=1 << 25),
           good(codes=None), good(scales=None), good(bounds=None), good(lens=None), good(codes=p + 8), good(bounds=p + 2), good(scales=p + 4)]
    for c in bad:
        r = C.byref(c)
        assert lib.artab_cache_write(0, p, st, p, st, 4, None, None, 1, r, None) == -1
        assert lib.artab_cache_read(0, r, None, 4, p, p, None) == -1
        assert lib.artab_cache_attention(0, p, st, 2, 1, r, 0, 1.0, p, p, None) == -1
        assert lib.artab_cache_select(0, p, st, 2, 1, r, 0, 1, p, None) == -1
        assert lib.artab_cache_block_attention(0, p, st, 2, 1, r, p, 1, 1.0, p, p, None, 0, None) == -1
        assert lib.artab_cache_block_workspace(r, 4096, 2, 64) == 0
    r = C.byref(good())
    assert lib.artab_cache_write(7, p, st, p, st, 4, None, None, 1, r, None) == -1
    assert lib.artab_cache_write(0, None, st, p, st, 4, None, None, 1, r, None) == -1
    assert lib.artab_cache_write(0, p, st, p, st, 0, None, None, 1, r, None) == -1
    assert lib.artab_cache_write(0, p, st, p, st, 129, None, None, 1, r, None) == -2
    assert lib.artab_cache_write(0, p, st, p, st, 4, p, None, 1, r, None) == -1
    assert lib.artab_cache_write(0, p, st, p, st, 4, p + 4, None, 0, r, None) == -1       # start inside lens
    assert lib.artab_cache_write(0, p, st, p, st, 4, None, p + 4, 0, r, None) == -1
    assert lib.artab_cache_read(0, r, None, 0, p, p, None) == -1
    assert lib.artab_cache_read(0, r, None, 1, p + 4, p, None) == -1
    assert lib.artab_cache_attention(3, p, st, 2, 1, r, 0, 1.0, p, p, None) == -1
    assert lib.artab_cache_attention(0, p, st, 3, 1, r, 0, 1.0, p, p, None) == -1
    assert lib.artab_cache_attention(0, p, st, 2, 0, r, 0, 1.0, p, p, None) == -1
    assert lib.artab_cache_attention(0, p, st, 2, 1, r, 0, 1.0, None, p, None) == -1
    assert lib.artab_cache_select(0, p, st, 2, 1, r, 0, 0, p, None) == -1
    assert lib.artab_cache_select(0, p, st, 2, 1, C.byref(good(n_blocks=3457)), 0, 1, p, None) == -1
    assert lib.artab_cache_block_attention(0, p, st, 2, 1, r, None, 1, 1.0, p, p, None, 0, None) == -1
    assert lib.artab_cache_block_attention(0, p, st, 2, 1, r, p, 0, 1.0, p, p, None, 0, None) == -1
    one = C.byref(good(n_groups=1, n_blocks=16))
    need = lib.artab_cache_block_workspace(one, 4096, 2, 8)
    assert need == 4096 * 2 * 2 * 8 * (32 * 4 + 8)
    assert lib.artab_cache_block_attention(0, p, st, 4096, 2, one, p, 8, 1.0, p, p, p, need - 1, None) == -2
    assert lib.artab_cache_block_attention(0, p, st, 4096, 2, one, p, 8, 1.0, p, p, p + 4, need, None) == -1
    assert b"cache" in lib.artab_last_error()


def test_replayed_rows_are_counted_too(fake, monkeypatch):
    """A graph that appends moves lens, not what the host knows of it."""
    c = cc.ContextCache(**tensors(), length=80)
    x = torch.zeros(G, H, 10, D)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    cc.append_context(c, x, x)
    cc.append_context(c, x, x)                              # two steps of one graph
    assert c.length == 100 and len(fake.calls) == 2
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    c.lens.fill_(125)                                       # what replays have left
    with pytest.raises(ValueError, match="capacity"):
        cc.append_context(c, x, x)
    assert len(fake.calls) == 2
    assert cc.read_context(c)[0].shape[2] == 125
    c.lens.fill_(118)
    cc.append_context(c, x, x)
    assert c.length == 128 and len(fake.calls) == 4


def test_sizes_beyond_32_bits_are_refused(fake):
    c = cc.ContextCache(**tensors(), length=0)
    x = torch.zeros(1).expand(G, H, 2 ** 32 + 5, D)
    start = torch.zeros(G, dtype=torch.int32)
    q = torch.zeros(G, H, 1, D)
    listed = torch.zeros(1, dtype=torch.int32).expand(G, H, 1, 2 ** 32 + 1)
    for match, call in (("rows at once", lambda: cc.append_context(c, x, x, start=start)),
                        ("rows at once", lambda: cc.quantize_context(x, x)),
                        ("no room", lambda: cc.quantize_context(x[:, :, :4], x[:, :, :4], capacity=2 ** 32 + 64)),
                        ("4294967297 rows", lambda: cc.read_context(c, n=2 ** 32 + 1)),
                        ("4294967297 blocks", lambda: cc.select_context_blocks(q, c, 2 ** 32 + 1)),
                        ("4294967297 blocks", lambda: cc.block_context_attention(q, c, listed))):
        with pytest.raises(ValueError, match=match):
            call()
    assert not fake.calls
    counts = cc._lengths(torch.tensor([2 ** 32, -2 ** 40, 7]), G, q.device, "counts")
    assert counts.dtype is torch.int32 and counts[0] >= 2 ** 30 and counts[1] < 0 and counts[2] == 7


def test_lists_that_a_step_would_carry_beyond_32_bits_are_refused(fake):
    """Warps step through a list by up to 2048 entries: a list that ends less than that below 2^31 would be left at the
    wrong end, so lists are as long as a cache has rows at most."""
    q = torch.zeros(G, H, 1, D)
    most = 1 << 30
    for n in (most + 1, 2 ** 31 - 64, 2 ** 31 - 1):
        listed = torch.zeros(1, dtype=torch.int32).expand(G, H, 1, n)
        with pytest.raises(ValueError, match=f"{n} blocks"):
            cc.block_context_attention(q, cache(), listed)
        with pytest.raises(ValueError, match=f"{n} blocks"):
            cc.select_context_blocks(q, cache(), n)
    assert not fake.calls
    import ctypes as C
    lib, p = _lib.load_library(), 4096
    st = (C.c_int64 * 3)(1, 1, 1)
    r = C.byref(_lib.Cache(n_groups=1, n_heads=2, head_dim=32, n_blocks=2, codes=p, scales=p, bounds=p, lens=p))
    for n in (most + 1, 2 ** 31 - 1):
        assert lib.artab_cache_select(0, p, st, 1, 1, r, 0, n, p, None) == -1
        assert lib.artab_cache_block_attention(0, p, st, 1, 1, r, p, n, 1.0, p, p, None, 0, None) == -1


def test_a_length_that_bounds_nothing_is_refused():
    """`length` is what room is counted from: below zero it would let rows fall behind the capacity unseen."""
    for length in (-1, -2 ** 40):
        with pytest.raises(ValueError, match="length"):
            cc.ContextCache(**tensors(), length=length)
    assert cc.ContextCache(**tensors(), length=0).length == 0 and cc.ContextCache(**tensors(), length=10 ** 9).length == 128


def test_row_counts_are_whole_numbers_however_they_are_handed_over(fake):
    """Lists go the way of tensors: no fraction is cut off, what does not fit 32 bits stays out of range."""
    dev = torch.device("cpu")
    for x in ([1.5, 2, 3], [True, False, True], [1.0, 2.0, 3.0], torch.tensor([1, 2, 3], dtype=torch.uint64)):
        with pytest.raises(ValueError, match="whole numbers"):
            cc._lengths(x, G, dev, "counts")
    with pytest.raises(ValueError, match="whole numbers"):
        cc.quantize_context(torch.zeros(G, H, N, D), torch.zeros(G, H, N, D), lens=[99.7, 3, 4])
    assert not fake.calls
    for x in ([2 ** 40, -2 ** 40, 7], torch.tensor([2 ** 32 - 1, 0, 7], dtype=torch.uint32), (300, 0, 7),
              torch.tensor([200, 0, 7], dtype=torch.uint8)):
        got = cc._lengths(x, G, dev, "counts")
        assert got.dtype is torch.int32 and got[0] >= 200 and got[1] <= 0 and got[2] == 7
