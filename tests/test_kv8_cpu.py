"""The paged 8-bit K/V cache without a GPU: the C ABI's argument checks (before any
HIP call), the binding's, the layout helpers, and the 64-bit restatement itself."""
import numpy as np
import pytest
import torch

from csahca_amd import extension, kv8_layout, native
from oracle import kv8 as plain

E4M3, INT8 = torch.float8_e4m3fn, torch.int8


@pytest.fixture(scope="module")
def lib():
    if not native.library_path().exists():
        pytest.fail("libcsahca.so is not built (run python -m csahca_amd.build)")
    return native.lib()


def _error(lib):
    return lib.csahca_last_error().decode()


CACHE = dict(kc=16, vc=16, ks=16, vs=16, fmt=0, pages=4, page=64, table=16, blocks=2, tstride=2)


def _cache(a):
    return (a["kc"], a["vc"], a["ks"], a["vs"], a["fmt"], a["pages"], a["page"], a["table"], a["blocks"], a["tstride"])


def _write(lib, **over):
    a = dict(CACHE, k=16, v=16, dtype=2, st=(0, 0, 0), start=16, counts=None, B=1, H=2, N=1, D=128)
    a.update(over)
    return lib.csahca_kv8_write(a["k"], a["v"], a["dtype"], *a["st"], *a["st"], *_cache(a), a["start"], a["counts"],
                                a["B"], a["H"], a["N"], a["D"], None)


def _read(lib, **over):
    a = dict(CACHE, start=None, lens=16, ko=16, vo=16, dtype=2, B=1, H=2, N=1, D=128)
    a.update(over)
    return lib.csahca_kv8_read(*_cache(a), a["start"], a["lens"], a["ko"], a["vo"], a["dtype"], a["B"], a["H"], a["N"],
                               a["D"], None)


def _attend(lib, **over):
    a = dict(CACHE, q=16, out=16, dtype=2, B=1, Q=1, heads=4, H=2, D=128, lens=16, scale=0.1, ws=None, wsb=0)
    a.update(over)
    return lib.csahca_kv8_decode_forward(a["q"], a["out"], a["dtype"], a["B"], a["Q"], a["heads"], a["H"], a["D"],
                                         *_cache(a), a["lens"], a["scale"], a["ws"], a["wsb"], None)


def _csa(lib, **over):
    a = dict(CACHE, q=16, out=16, dtype=2, B=1, heads=4, H=2, D=128, lens=16, ids=16, idt=0, top_k=2, chunk=64, scale=0.1,
             ws=None, wsb=0)
    a.update(over)
    return lib.csahca_kv8_csa_decode_forward(a["q"], a["out"], a["dtype"], a["B"], a["heads"], a["H"], a["D"],
                                             *_cache(a), a["lens"], a["ids"], a["idt"], a["top_k"], a["chunk"],
                                             a["scale"], a["ws"], a["wsb"], None)


@pytest.mark.parametrize("call", [_write, _read, _attend, _csa])
def test_cache_argument_errors_before_any_launch(lib, call):
    for over, text in ((dict(fmt=2), "float8_e4m3fn or int8"), (dict(page=0), "multiple of 16"),
                       (dict(page=24), "multiple of 16"), (dict(page=272), "multiple of 16"),
                       (dict(D=0), "multiple of 32"), (dict(D=48), "multiple of 32"), (dict(D=288), "multiple of 32"),
                       (dict(pages=-1), "negative"), (dict(blocks=-1), "negative"), (dict(H=-1), "negative"),
                       (dict(B=-1), "negative"), (dict(tstride=1), "rows overlap"), (dict(pages=2 ** 40), "too large"),
                       (dict(blocks=2 ** 30, tstride=2 ** 30), "too large"),
                       (dict(dtype=3), "unsupported dtype"), (dict(dtype=9), "unsupported dtype"),
                       (dict(kc=None), "null tensor pointer"), (dict(table=None), "null tensor pointer"),
                       (dict(ks=None), "null tensor pointer"), (dict(kc=8), "16-byte aligned"),
                       (dict(vc=24), "16-byte aligned")):
        assert call(lib, **over) == 1 and text in _error(lib), (over, _error(lib))


def test_other_argument_errors_before_any_launch(lib):
    assert _write(lib, k=None) == 1 and _error(lib) == "null tensor pointer"
    assert _write(lib, start=None) == 1 and _error(lib) == "null tensor pointer"
    assert _write(lib, N=-1) == 1 and _write(lib, N=2 ** 40) == 1 and "too many tokens" in _error(lib)
    assert _write(lib, B=2 ** 20, N=2 ** 20) == 1 and "too many tokens" in _error(lib)
    assert _write(lib, B=0) == 0 and _write(lib, N=0) == 0 and _write(lib, H=0) == 0
    assert _write(lib, pages=0) == 0 and _write(lib, blocks=0, tstride=0) == 0
    assert _read(lib, ko=None) == 1 and _read(lib, lens=None) == 1 and _error(lib) == "null tensor pointer"
    assert _read(lib, B=2 ** 20, N=2 ** 20) == 1 and "too many tokens" in _error(lib)
    assert _read(lib, B=0) == 0 and _read(lib, N=0) == 0
    assert _attend(lib, heads=5) == 1 and "multiple of the cache's heads" in _error(lib)
    assert _attend(lib, H=0) == 1 and "multiple of the cache's heads" in _error(lib)
    assert _attend(lib, q=None) == 1 and _attend(lib, lens=None) == 1 and _error(lib) == "null tensor pointer"
    assert _attend(lib, Q=2 ** 20, B=2 ** 20) == 1 and "too many query rows" in _error(lib)
    assert _attend(lib, B=0) == 0 and _attend(lib, Q=0) == 0 and _attend(lib, heads=0) == 0
    assert _csa(lib, idt=2) == 1 and _error(lib) == "chunk_indices must be int32 or int64"
    assert _csa(lib, chunk=0) == 1 and _error(lib) == "chunk_size must be positive"
    assert _csa(lib, top_k=-1) == 1 and _csa(lib, ids=None) == 1 and _error(lib) == "null tensor pointer"
    assert _csa(lib, B=0) == 0 and _csa(lib, heads=0) == 0


def test_workspace_sizes(lib):
    big = 1 << 40
    f, g = lib.csahca_kv8_decode_workspace_bytes, lib.csahca_kv8_csa_decode_workspace_bytes
    assert f(2, -1, 1, 8, 8, 128, 64, 8) == f(2, 1, 1, 8, 0, 128, 64, 8) == f(2, 0, 1, 8, 8, 128, 64, 8) == 0
    assert g(2, 1, 8, 0, 128, 8, 64) == g(2, 1, 8, 8, 128, -8, 64) == g(2, 1, 8, 8, 128, 0, 64) == 0
    assert f(2, 1, 1, 8, 8, 128, 64, 16) == 0  # 1024 tokens: one part a sequence, nothing to join
    # parts of at least 4 tiles of 64 tokens: 32 for 8192 tokens, each a row of 128 values, two maxima and a sum (in four)
    assert f(2, 1, 1, 8, 8, 128, 64, 128) == 32 * 8 * 132 * 4
    assert f(2, big, big, big, 1, 128, 64, big) == 0 and g(2, big, big, 1, 128, big, big) == 0
    assert f(0, 4, 50, 64, 8, 256, 256, 4096) > 0 and g(2, 1, 8, 8, 128, 64, 64) > 0


def test_missing_workspace_is_reported(lib):
    assert _attend(lib, blocks=128, tstride=128) == 2 and "workspace too small" in _error(lib)
    assert _csa(lib, top_k=64) == 2 and "workspace too small" in _error(lib)
    assert _attend(lib, q=8) == 1 and "16-byte aligned" in _error(lib)
    enough = dict(wsb=1 << 60)
    assert _attend(lib, blocks=128, tstride=128, ws=8, **enough) == 1 and "workspace must be 16-byte" in _error(lib)
    assert _csa(lib, top_k=64, ws=24, **enough) == 1 and "workspace must be 16-byte" in _error(lib)


def test_calls_beyond_a_launch_are_refused(lib):
    """Grids of 2^32 threads and more, and sizes whose products pass 32 bits on the way."""
    huge = dict(ws=16, wsb=1 << 62)
    assert _attend(lib, B=1 << 25, blocks=128, tstride=128, **huge) == 1 and "too many query rows" in _error(lib)
    assert _write(lib, B=1 << 22, H=4) == 1 and "too many tokens" in _error(lib)
    assert _write(lib, B=1 << 14, N=1 << 20) == 1 and "too many tokens" in _error(lib)
    assert _read(lib, B=1 << 20, N=1 << 20) == 1 and "too many tokens" in _error(lib)
    assert _csa(lib, B=(1 << 31) - 1, heads=65534, top_k=1 << 20, **huge) == 1 and "too many query rows" in _error(lib)
    g = lib.csahca_kv8_csa_decode_workspace_bytes
    # a list is never divided further than it is long, however many sequences there are
    assert g(2, (1 << 31) - 1, 64, 32, 128, 1 << 20, 64) == 0 and g(2, 1 << 20, 8, 8, 128, 1 << 20, 64) == 0


def test_binding_rejects_cpu_tensors():
    cache = kv8_layout.empty_cache(2, 2, 16, 32, device="cpu")
    table, n = torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    q = torch.zeros(1, 2, 32)
    for f, args in ((extension.kv8_decode_forward, (q, *cache, table, n)),
                    (extension.kv8_csa_decode_forward, (q, *cache, table, n, torch.zeros(1, 2, 1, dtype=torch.int32), 16)),
                    (extension.kv8_read, (*cache, table, n, 4)),
                    (extension.kv8_write, (q.unsqueeze(2), q.unsqueeze(2), *cache, table, n))):
        with pytest.raises(RuntimeError, match="must be CUDA tensors"):
            f(*args)


def test_layout_helpers():
    c = kv8_layout.empty_cache(3, 2, 48, 96, dtype=INT8, device="cpu")
    assert c.k_cache.shape == (3, 2, 48, 96) and c.v_cache.shape == (3, 2, 3, 96, 16) and c.k_cache.dtype == INT8
    assert c.k_scale.shape == c.v_scale.shape == (3, 2) and c.k_scale.data_ptr() != c.v_scale.data_ptr()
    assert kv8_layout.num_blocks(0, 16) == 0 and kv8_layout.num_blocks(17, 16) == 2
    assert kv8_layout.LARGEST == plain.LARGEST


def test_restated_e4m3_is_torchs():
    codes = np.arange(256, dtype=np.uint8)
    want = torch.from_numpy(codes).view(E4M3).double().numpy()
    assert np.array_equal(plain.decode(codes, E4M3), want, equal_nan=True)
    x = np.concatenate([np.linspace(-448, 448, 40001), np.linspace(-0.1, 0.1, 4001), plain._MIDDLES, -plain._MIDDLES])
    x = x.astype(np.float32)
    want = torch.from_numpy(x).to(E4M3).view(torch.uint8).numpy()
    assert np.array_equal(plain.encode(x.astype(np.float64), E4M3), want)


def test_restated_write_and_read_agree():
    """What is written reads back within half a step of the page's scale."""
    g = torch.Generator().manual_seed(1)
    for fmt in (E4M3, INT8):
        cache = kv8_layout.empty_cache(4, 2, 16, 32, dtype=fmt, device="cpu")
        table = torch.tensor([[2, 0], [3, 1]], dtype=torch.int32)
        k, v = (torch.randn(2, 2, 20, 32, generator=g) for _ in range(2))
        cache = plain.write(k, v, cache, table, torch.tensor([0, 5], dtype=torch.int32))
        got = plain.read(cache, table, torch.tensor([20, 25]), 20, torch.tensor([0, 5]))
        for x, y in zip((k, v), got):
            x = x.double().numpy()
            # |x| < 8: an int8 scale of at most 2^-4, an e4m3 one of at most 2^-6 (steps of 2^-9 below 2^-6)
            half = 2.0 ** -5 if fmt == INT8 else np.maximum(np.abs(x) * 2.0 ** -4, 2.0 ** -16)
            assert np.all(np.abs(x - y) <= half)
