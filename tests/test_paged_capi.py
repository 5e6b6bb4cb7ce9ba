"""CPU checks of the paged cache's entry points: struct layout, refusals before anything runs."""
import copy
import ctypes
import dataclasses
import pickle
import weakref

import numpy as np
import pytest
import torch

import oracle.paged as OP
import slang_amd as sa
from slang_amd import _lib
from slang_amd._lib import G4ACfg, G4APaged

FAKE = 0x10000  # never dereferenced: every case fails validation first
E, U, W = -1, -2, -3


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def cfg(**kw):
    base = dict(n_q_heads=8, n_kv_heads=2, head_dim=256, window=0, flags=0, scale=1.0, eps=1e-6, out_q=0.0)
    base.update(kw)
    return G4ACfg(**base)


def paged(**kw):
    base = dict(k_pages=FAKE, v_pages=FAKE, page_table=FAKE, key_len=FAKE, n_pages=100, page_size=16, n_seq=4,
                table_cols=10, table_stride=10, max_key_len=160)
    base.update(kw)
    return G4APaged(**base)


def test_struct_layout():
    assert [f[0] for f in G4APaged._fields_] == ["k_pages", "v_pages", "page_table", "key_len", "n_pages", "page_size", "n_seq",
                                                 "table_cols", "table_stride", "max_key_len", "reserved"]
    assert ctypes.sizeof(G4APaged) == 64 and G4APaged.n_pages.offset == 32 and G4APaged.reserved.offset == 56


def write(lib, c=None, pg=None, n=8, cu=FAKE, k=FAKE, v=FAKE, ks=0.0, vs=0.0, kg=None, cos=None, sin=None):
    return lib.g4a_paged_write(ctypes.byref(c or cfg()), None if pg == 0 else ctypes.byref(pg or paged()), n, cu, k, v, ks, vs,
                               kg, cos, sin, None)


def decode(lib, c=None, pg=None, q=FAKE, qg=None, cos=None, sin=None, kn=None, vn=None, ks=0.0, vs=0.0, kg=None,
           out=0x4000000, ws=FAKE, n=1 << 30):
    return lib.g4a_paged_decode(ctypes.byref(c or cfg()), None if pg == 0 else ctypes.byref(pg or paged()), q, qg, cos, sin, kn,
                                vn, ks, vs, kg, out, ws, n, None)


def prefill(lib, c=None, pg=None, n=8, cu=FAKE, q=FAKE, qg=None, cos=None, sin=None, out=0x4000000, ws=FAKE, nb=1 << 40):
    return lib.g4a_paged_prefill(ctypes.byref(c or cfg()), None if pg == 0 else ctypes.byref(pg or paged()), n, cu, q, qg, cos,
                                 sin, out, ws, nb, None)


@pytest.mark.parametrize("call", [write, decode, prefill])
def test_cache_refusals(lib, call):
    assert call(lib, pg=0) == E
    for field in ("k_pages", "v_pages", "page_table", "key_len"):
        assert call(lib, pg=paged(**{field: None})) == E
    assert call(lib, pg=paged(k_pages=FAKE + 8)) == E
    assert call(lib, pg=paged(page_table=FAKE + 2)) == E
    for size in (0, -16, 1, 8, 24, 131072):
        assert call(lib, pg=paged(page_size=size)) == U, size
    for bad in (dict(n_pages=0), dict(n_seq=0), dict(n_seq=-1), dict(table_cols=0), dict(table_stride=9), dict(max_key_len=0),
                dict(max_key_len=161), dict(n_seq=40000), dict(table_cols=1 << 30, table_stride=1 << 30, max_key_len=(1 << 30) + 1)):
        assert call(lib, pg=paged(**bad)) == E, bad
    pg = paged()
    pg.reserved[1] = 1
    assert call(lib, pg=pg) == E
    assert call(lib, c=cfg(head_dim=128)) == U
    assert call(lib, c=cfg(n_q_heads=6, n_kv_heads=4)) == E
    assert call(lib, c=cfg(window=(1 << 30) + 1)) == E
    assert call(lib, cos=FAKE) == E and call(lib, sin=FAKE) == E
    assert call(lib, cos=FAKE + 4, sin=FAKE) == E


def test_write_refusals(lib):
    assert write(lib, n=0) == E and write(lib, n=-1) == E
    assert write(lib, cu=None) == E and write(lib, cu=FAKE + 1) == E
    assert write(lib, k=None) == E and write(lib, v=None) == E
    assert write(lib, k=FAKE + 8) == E and write(lib, kg=FAKE + 4) == E
    assert write(lib, ks=-1.0) == E and write(lib, vs=float("nan")) == E


def test_decode_refusals(lib):
    assert decode(lib, c=cfg(n_q_heads=24, n_kv_heads=2)) == E  # 12 query heads a kv head
    assert decode(lib, q=None) == E and decode(lib, out=None) == E
    assert decode(lib, q=FAKE + 4) == E and decode(lib, qg=FAKE + 4) == E and decode(lib, out=0x4000008) == E
    assert decode(lib, kn=FAKE) == E and decode(lib, vn=FAKE) == E
    assert decode(lib, kn=FAKE + 4, vn=FAKE) == E
    assert decode(lib, kn=FAKE, vn=FAKE, ks=-0.5) == E
    assert decode(lib, c=cfg(flags=_lib.IN_F16)) == U
    assert decode(lib, out=FAKE) == E  # over q
    far = 0x8000000
    assert decode(lib, q=far, kn=0x4000000, vn=far + 0x10000) == E and decode(lib, q=far, kn=far + 0x10000, vn=0x4000100) == E
    assert b"k_new" in lib.g4a_last_error()
    assert decode(lib, ws=None) == W and decode(lib, ws=FAKE + 16) == W and decode(lib, n=16) == W
    assert b"workspace" in lib.g4a_last_error()
    assert lib.g4a_paged_decode_ws_bytes(ctypes.byref(cfg()), ctypes.byref(paged())) > 0
    assert lib.g4a_paged_decode_ws_bytes(ctypes.byref(cfg()), ctypes.byref(paged(n_seq=0))) == 0


def test_prefill_refusals(lib):
    assert prefill(lib, n=0) == E and prefill(lib, n=1 << 30) == E
    assert prefill(lib, cu=None) == E and prefill(lib, q=None) == E and prefill(lib, out=None) == E
    assert prefill(lib, q=FAKE + 4) == E and prefill(lib, out=0x4000008) == E
    assert prefill(lib, c=cfg(flags=_lib.Q_HILO)) == U
    assert prefill(lib, out=FAKE + 4096) == E
    assert prefill(lib, ws=None) == W and prefill(lib, ws=FAKE + 16) == W and prefill(lib, nb=16) == W
    size = lambda n=8, c=None, **k: lib.g4a_paged_prefill_ws_bytes(ctypes.byref(c or cfg()), ctypes.byref(paged(**k)), n)  # noqa: E731
    assert size() > 0 and size(n=0) == 0 and size(n_pages=0) == 0


def test_host_refusals_without_a_gpu():
    """The host layer refuses CPU tensors and shapes that do not fit before it loads anything."""
    c = sa.AttnConfig(8, 2, 256)
    q, pages = torch.zeros(2, 8, 256), torch.zeros(4, 16, 2, 256, dtype=torch.float16)
    tab, kl = torch.zeros(2, 2, dtype=torch.int32), torch.ones(2, dtype=torch.int32)
    for call in (lambda: sa.paged_decode(q, pages, pages, tab, kl, c),
                 lambda: sa.paged_prefill(q, pages, pages, tab, kl, torch.zeros(3, dtype=torch.int32), c, workspace=None),
                 lambda: sa.paged_write(q[:, :2], q[:, :2], pages, pages, tab, kl, torch.zeros(3, dtype=torch.int32), c),
                 lambda: sa.paged_decode(q[:, :4], pages, pages, tab, kl, c)):
        with pytest.raises(ValueError):
            call()


def test_used_configs_are_copied_and_pickled():
    c = sa.AttnConfig(8, 2, 256, window=100, scale=0.5)
    c.c_ref(3)
    for x in (copy.copy(c), copy.deepcopy(c), pickle.loads(pickle.dumps(c)), dataclasses.replace(c)):
        assert x == c and hash(x) == hash(c) and x.c(3).window == 100
        assert ctypes.cast(x.c_ref(3), ctypes.POINTER(G4ACfg)).contents.scale == 0.5


def test_workspace_sizes(lib):
    c = sa.AttnConfig(8, 2, 256)
    assert sa.paged_decode_ws_bytes(16, 4096, c, page_size=16) > 0
    assert sa.paged_prefill_ws_bytes(100, 16, 4096, c, page_size=64) > 0
    assert sa.paged_prefill_ws_bytes(100, 16, 4096, c, page_size=64, kv_f32=True) > 0
    with pytest.raises(_lib.G4AError):
        sa.paged_decode_ws_bytes(16, 4096, c, page_size=20)
    with pytest.raises(_lib.G4AError):
        sa.paged_prefill_ws_bytes(0, 16, 4096, c, page_size=64)


@pytest.mark.parametrize("kvh,hd,window", [(1, 256, 512), (2, 256, 0), (8, 256, 0), (2, 512, 0), (1, 512, 4096)])
@pytest.mark.parametrize("kv_f32", [False, True])
def test_a_workspace_holds_every_smaller_call(kvh, hd, window, kv_f32):
    """Sizes grow with tokens, sequences and the bound of the keys: one reserved for the largest call does."""
    c, kw = sa.AttnConfig(8, kvh, hd, window), dict(page_size=16, kv_f32=kv_f32)
    seqs, keys = [1, 2, 3, 7, 16, 33, 64, 65, 200, 300, 1000, 4000], [1, 16, 128, 129, 320, 321, 600, 4096, 8192, 30000, 131072]
    tokens = [1, 5, 33, 100, 1000, 3000, 10000, 30000, 100000]
    dec = np.array([[sa.paged_decode_ws_bytes(n, k, c, **kw) for k in keys] for n in seqs])
    assert (np.diff(dec, axis=0) >= 0).all() and (np.diff(dec, axis=1) >= 0).all()
    pre = np.array([[[sa.paged_prefill_ws_bytes(t, n, k, c, **kw) for k in keys] for n in seqs] for t in tokens])
    assert all((np.diff(pre, axis=i) >= 0).all() for i in range(3))


def test_oracle_keys():
    """The definition's attended positions: window, missing pages, positions below zero."""
    table = np.array([[3, -1, 7, 100]], np.int32)
    t, rows = OP.keys_of(table, 0, 40, 16, 8, 0)
    assert t.tolist() == list(range(16)) + list(range(32, 41)) and rows[16] == 7 * 16
    t, _ = OP.keys_of(table, 0, 60, 16, 8, 30)
    assert t.tolist() == list(range(32, 48))
    assert len(OP.keys_of(table, 0, -1, 16, 8, 0)[0]) == 0


@pytest.mark.parametrize("kvh,hd", [(1, 256), (8, 512), (64, 512)])
def test_plans_of_the_largest_batches(lib, kvh, hd):
    """The share of a key split stays within 32 bits, whatever the number of sequences and of keys."""
    for n_seq in (1, 2, 64, 1000, 1024):
        for keys in (1, 1000, 131072, 1 << 20, 1 << 24, 1 << 26, (1 << 30) - 1, 1 << 30):
            for window in (0, 512):
                c = cfg(n_q_heads=8 * kvh, n_kv_heads=kvh, head_dim=hd, window=window)
                need = lib.g4a_decode_ws_bytes(ctypes.byref(c), n_seq, keys)
                assert 0 < need <= (512 + 2 * n_seq * kvh) * 8 * (hd * 4 + 8 + 8) + 1024, (n_seq, keys, window)


@pytest.mark.parametrize("flags", [0, _lib.KV_F32])
@pytest.mark.parametrize("kvh,hd", [(1, 256), (8, 512), (64, 512), (512, 512)])
def test_long_bounds_are_not_refused(lib, kvh, hd, flags):
    """A decode call whose workspace has a size is not refused for its max_key_len: with no workspace, that
    is all that is wrong with it."""
    for n_seq in (1, 2, 64, 100):
        for keys in (1000, 131072, 1 << 20, 1 << 26, 1 << 30):
            c, pg = cfg(n_q_heads=8 * kvh, n_kv_heads=kvh, head_dim=hd, flags=flags), paged(
                n_seq=n_seq, page_size=65536, table_cols=1 << 14, table_stride=1 << 14, max_key_len=keys)
            assert lib.g4a_paged_decode_ws_bytes(ctypes.byref(c), ctypes.byref(pg)) > 0
            far = 1 << 44
            assert decode(lib, c=c, pg=pg, q=far, out=2 * far, ws=None) == W, (n_seq, keys, lib.g4a_last_error())


@pytest.mark.parametrize("groups", [3, 5, 6, 7, 12, 16])
def test_group_sizes_without_a_kernel(lib, groups):
    """Refused before anything is launched, with the sizes that are taken named."""
    c = cfg(n_q_heads=2 * groups, n_kv_heads=2)
    for call in (decode, prefill):
        assert call(lib, c=c) == E and b"1, 2, 4 or 8" in lib.g4a_last_error()
    assert lib.g4a_paged_decode_ws_bytes(ctypes.byref(c), ctypes.byref(paged())) == 0
    assert lib.g4a_paged_prefill_ws_bytes(ctypes.byref(c), ctypes.byref(paged()), 8) == 0


def test_used_configs_are_their_fields():
    """What a call keeps of a config stays out of vars(), copies and pickles of every protocol."""
    @dataclasses.dataclass(frozen=True)
    class Named(sa.AttnConfig):
        name: str = "x"
    for c in (sa.AttnConfig(8, 2, 256, window=100), Named(8, 2, 256, name="y")):
        names = {f.name for f in dataclasses.fields(c)}
        for flags in (0, 3, 3):
            got = ctypes.cast(c.c_ref(flags), ctypes.POINTER(G4ACfg)).contents
            assert (got.n_kv_heads, got.flags) == (2, flags)
        assert c.c_ref(3) is c.c_ref(3)
        assert set(vars(c)) == names and type(c)(**vars(c)) == c and dataclasses.asdict(c) == vars(c)
        with pytest.raises(dataclasses.FrozenInstanceError):
            c.window = 3
        assert copy.copy(c) == c and copy.deepcopy(c) == c and weakref.ref(c)() is c
    c = sa.AttnConfig(8, 2, 256)
    c.c_ref(0)
    for protocol in range(pickle.HIGHEST_PROTOCOL + 1):
        assert pickle.loads(pickle.dumps(c, protocol)) == c
