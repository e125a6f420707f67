"""Host side of the serving operators, without a GPU: the C ABI's struct layouts and refusals (raised before any CUDA
call), workspace sizes, and the checks of the Python entry points that come before device work."""
import ctypes

import pytest
import torch

from first_passage_attention_b200 import FPACache, _lib, verify_draft


def _cache(**kw):
    f = dict(dtype=_lib.DTYPE_F16, storage=_lib.STORE_I8, n_pages=4, H=2, page_size=64, D=64, k=4096, v=4096, k_scale=4096,
             v_scale=4096, phi=4096, psi=4096, phi_min=4096, status=4096)
    f.update(kw)
    return _lib.FpaCache(**f)


def test_struct_sizes_match():
    lib = _lib.load()
    for i, cls in enumerate((_lib.FpaCache, _lib.FpaAppendArgs, _lib.FpaReadArgs, _lib.FpaDecodeArgs, _lib.FpaVerifyArgs), 3):
        assert lib.fpa_struct_size(i) == ctypes.sizeof(cls), cls
    for packer, cls in ((_lib.APPEND_PACKER, _lib.FpaAppendArgs), (_lib.READ_PACKER, _lib.FpaReadArgs),
                        (_lib.DECODE_PACKER, _lib.FpaDecodeArgs), (_lib.VERIFY_PACKER, _lib.FpaVerifyArgs)):
        assert packer.size == ctypes.sizeof(cls)


@pytest.mark.parametrize("change,message", [
    (dict(dtype=5), b"dtype"), (dict(storage=_lib.STORE_F32), b"storage"), (dict(n_pages=0), b"at least one page"),
    (dict(page_size=48), b"page size"), (dict(page_size=16), b"page size"), (dict(D=96), b"head dimension"),
    (dict(phi_min=None), b"null cache pointer"), (dict(k_scale=None), b"scale pointer"), (dict(k=4104), b"16-byte aligned"),
    (dict(H=70000), b"65535")])
def test_cache_descriptions_are_checked(change, message):
    lib = _lib.load()
    c = _cache(**change)
    addr = ctypes.addressof(c)
    for fn, args in ((lib.fpa_cache_append, _lib.FpaAppendArgs(cache=addr, B=1, n=1, max_pages=1)),
                     (lib.fpa_cache_read, _lib.FpaReadArgs(cache=addr, B=1, n=1, max_pages=1)),
                     (lib.fpa_decode, _lib.FpaDecodeArgs(cache=addr, B=1, n=1, max_pages=1))):
        assert fn(ctypes.byref(args), None) in (_lib.ERR_INVALID, _lib.ERR_UNSUPPORTED)
        assert message in lib.fpa_last_error()
    assert lib.fpa_decode_workspace_bytes(ctypes.byref(c), 1, 1, 100) == 0


def test_argument_errors_come_before_any_cuda_call():
    lib = _lib.load()
    c = _cache()
    addr = ctypes.addressof(c)
    A, R, D, V = _lib.FpaAppendArgs, _lib.FpaReadArgs, _lib.FpaDecodeArgs, _lib.FpaVerifyArgs
    dec = dict(cache=addr, B=1, n=1, max_pages=1, q=4096, o=4096, beta=4096, table=4096, lengths=4096)
    ver = dict(dtype=0, B=1, n=1, V=8, p=4096, q=4096, draft=4096, u=4096, noise=4096, accepted=4096, tokens=4096)
    for fn, args, rc, message in [
            (lib.fpa_cache_append, None, _lib.ERR_INVALID, b"null argument"),
            (lib.fpa_cache_append, A(cache=addr, B=0, n=1, max_pages=1), _lib.ERR_INVALID, b"positive"),
            (lib.fpa_cache_append, A(cache=addr, B=1, n=1, max_pages=0), _lib.ERR_INVALID, b"column"),
            (lib.fpa_cache_append, A(cache=addr, B=1, n=1, max_pages=1), _lib.ERR_INVALID, b"null tensor"),
            (lib.fpa_cache_read, R(cache=addr, B=1, n=1, max_pages=1, k=4100, v=4096, phi=4096, psi=4096, table=4096), _lib.ERR_INVALID, b"aligned"),
            (lib.fpa_decode, D(**{**dec, "n": 17}), _lib.ERR_INVALID, b"between 1 and 16"),
            (lib.fpa_decode, D(**{**dec, "n": 0}), _lib.ERR_INVALID, b"between 1 and 16"),
            (lib.fpa_decode, D(**{**dec, "beta": None}), _lib.ERR_INVALID, b"null tensor"),
            (lib.fpa_decode, D(**{**dec, "B": 70000}), _lib.ERR_UNSUPPORTED, b"65535"),
            (lib.fpa_decode, D(**{**dec, "prefix_len": 65, "prefix_pages": 1, "prefix_table": 4096}), _lib.ERR_INVALID, b"longer than the pages"),
            (lib.fpa_decode, D(**{**dec, "prefix_len": 64, "prefix_pages": 1, "prefix_table": 4096}), _lib.ERR_WORKSPACE, b"workspace"),
            (lib.fpa_verify, V(**{**ver, "dtype": 3}), _lib.ERR_INVALID, b"fp16 or fp32"),
            (lib.fpa_verify, V(**{**ver, "V": 0}), _lib.ERR_INVALID, b"positive"),
            (lib.fpa_verify, V(**{**ver, "noise": None}), _lib.ERR_INVALID, b"null tensor"),
            (lib.fpa_verify, V(**{**ver, "B": 70000}), _lib.ERR_UNSUPPORTED, b"65535")]:
        got = fn(None if args is None else ctypes.byref(args), None)
        assert got == rc and message in lib.fpa_last_error(), (message, got, lib.fpa_last_error())


def test_row_groups_fit_the_grid():
    """float32 rows with D = 128 and 256 go in groups of four: their grids are full at half of the rows and heads."""
    lib = _lib.load()
    dec = dict(max_pages=1, q=4096, o=4096, beta=4096, table=4096, lengths=4096)
    pre = dict(prefix_len=64, prefix_pages=1, prefix_table=4096)  # without a workspace: what passes the check ends there
    f32 = dict(dtype=_lib.DTYPE_F32, storage=_lib.STORE_F32)
    for cache, args, rc in [
            (dict(f32, D=128, H=16384), dict(B=1, n=13, **pre), _lib.ERR_UNSUPPORTED),
            (dict(f32, D=256, H=32767), dict(B=1, n=16, **pre), _lib.ERR_UNSUPPORTED),
            (dict(f32, D=128, H=16383), dict(B=1, n=16, **pre), _lib.ERR_WORKSPACE),
            (dict(f32, D=128, H=21845), dict(B=1, n=12, **pre), _lib.ERR_WORKSPACE),
            (dict(f32, D=64, H=32767), dict(B=1, n=16, **pre), _lib.ERR_WORKSPACE),
            (dict(D=128, H=32767), dict(B=1, n=16, **pre), _lib.ERR_WORKSPACE),
            (dict(f32, D=128, H=2), dict(B=20165, n=13, **pre), _lib.ERR_UNSUPPORTED),
            (dict(f32, D=256, H=2), dict(B=65535, n=4, **pre), _lib.ERR_WORKSPACE),
            (dict(f32, D=256, H=2), dict(B=65535, n=5, **pre), _lib.ERR_UNSUPPORTED),
            (dict(f32, D=64, H=2), dict(B=65535, n=8, **pre), _lib.ERR_WORKSPACE),
            (dict(f32, D=64, H=2), dict(B=65535, n=9, **pre), _lib.ERR_UNSUPPORTED),
            (dict(D=256, H=2), dict(B=65535, n=8, **pre), _lib.ERR_WORKSPACE),
            (dict(D=128, H=2), dict(B=65535, n=16, **pre), _lib.ERR_UNSUPPORTED)]:
        c = _cache(**cache)
        got = lib.fpa_decode(ctypes.byref(_lib.FpaDecodeArgs(cache=ctypes.addressof(c), **dec, **args)), None)
        assert got == rc, (cache, args, got, lib.fpa_last_error())


def test_prefixes_end_where_positions_round_up_within_32_bits():
    lib = _lib.load()
    c = _cache()
    dec = dict(cache=ctypes.addressof(c), B=1, n=1, max_pages=1, q=4096, o=4096, beta=4096, table=4096, lengths=4096,
               prefix_table=4096, prefix_pages=2 ** 25)
    for length, rc in ((2 ** 31 - 256, _lib.ERR_WORKSPACE), (2 ** 31 - 255, _lib.ERR_UNSUPPORTED), (2 ** 31 - 1, _lib.ERR_UNSUPPORTED)):
        assert lib.fpa_decode(ctypes.byref(_lib.FpaDecodeArgs(prefix_len=length, **dec)), None) == rc, length
        assert (lib.fpa_decode_workspace_bytes(ctypes.byref(c), 1, 1, length) > 0) == (rc == _lib.ERR_WORKSPACE)


def test_workspace_grows_with_the_rows_of_a_prefix_only():
    lib = _lib.load()
    c = _cache()
    assert lib.fpa_decode_workspace_bytes(ctypes.byref(c), 8, 4, 0) == 0
    small = lib.fpa_decode_workspace_bytes(ctypes.byref(c), 8, 4, 1)
    assert 0 < small < lib.fpa_decode_workspace_bytes(ctypes.byref(c), 80, 4, 1)
    assert lib.fpa_decode_workspace_bytes(ctypes.byref(c), 8, 17, 64) == 0


def test_python_refusals_without_a_device():
    for kw, message in ((dict(dtype=torch.bfloat16), "dtype"), (dict(storage=torch.float32), "storage"),
                        (dict(page_size=48), "page size"), (dict(head_dim=96), "head dimension"),
                        (dict(n_pages=0), "at least one page"), (dict(device="cpu"), "CUDA device")):
        with pytest.raises(ValueError, match=message):
            FPACache(**{**dict(n_pages=2, n_heads=1, head_dim=64), **kw})
    p, q = torch.zeros(1, 3, 5), torch.zeros(1, 2, 5)
    with pytest.raises(ValueError, match="one CUDA device"):
        verify_draft(p, q, torch.zeros(1, 2, dtype=torch.int64), torch.zeros(1, 2), torch.zeros(1, 5))
