"""ctypes binding of ``libelx_ops.so`` (declared in ``include/elx_ops.h``): the operators of a training step beside the
optimizer step in 32 bits.  As with ``libelx_hip.so`` there is no CPU fallback: a library that is missing or was built from
other sources raises, and so does a refused launch."""
import ctypes
import os

import numpy as np

from . import _abi

ELX_OPS_VERSION = 1
STATE_BLOCK = 256    # elements per block of the 8-bit state (checked against the library)

STATE8_DTYPE = np.dtype([('scales', '<u8'), ('first_block', '<u4'), ('salt', '<u4')])

LIB_PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), 'libelx_ops.so')

EXPORTS = ('elx_ops_version', 'elx_ops_source_sha', 'elx_sizeof_state8', 'elx_state8_block', 'elx_adam8_step_mt',
           'elx_adam8_step_args_mt', 'elx_adam8_step_gated_mt', 'elx_check_state8', 'elx_state8_read', 'elx_state8_write',
           'elx_layer_norm_max_cols', 'elx_layer_norm_bwd_workspace', 'elx_layer_norm_fwd', 'elx_layer_norm_bwd',
           'elx_embedding_fwd', 'elx_embedding_bwd_workspace', 'elx_embedding_bwd')

_CSRC = os.path.join(os.path.dirname(os.path.abspath(__file__)), 'csrc')
_INCLUDE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), 'include')


def source_files():
    """The files a build of the library is made from, in the order their digest is taken."""
    ops = os.path.join(_CSRC, 'ops')
    files = [os.path.join(ops, f) for f in sorted(os.listdir(ops)) if f.endswith(('.hip', '.cpp', '.h'))]
    return files + [os.path.join(_CSRC, f) for f in ('elx_host.cpp', 'elx_host.h')] + \
        [os.path.join(_INCLUDE, f) for f in ('elx_abi.h', 'elx_ops.h')]


def source_sha16() -> str:
    """First 16 hex digits of the SHA-256 over the library's sources as they are now."""
    import hashlib
    h = hashlib.sha256()
    for path in source_files():
        h.update(os.path.basename(path).encode() + b'\0')
        with open(path, 'rb') as f:
            h.update(f.read())
    return h.hexdigest()[:16]


def built_source_sha(lib_path: str) -> str:
    """The digest a built library carries ('' when it has none)."""
    try:
        L = ctypes.CDLL(lib_path)
        L.elx_ops_source_sha.restype = ctypes.c_char_p
        L.elx_ops_source_sha.argtypes = []
        return (L.elx_ops_source_sha() or b'').decode()
    except (OSError, AttributeError):
        return ''


_lib = None


def load() -> ctypes.CDLL:
    """Load the library once; raise loudly when it is missing or does not match this binding."""
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(LIB_PATH):
        raise RuntimeError(f'{LIB_PATH} is missing: the HIP extension has not been built. '
                           f'Run `python -m elixir_amd.build` (needs hipcc); there is no CPU fallback.')
    L = ctypes.CDLL(LIB_PATH)
    u32, u64, vp, cint, flt = ctypes.c_uint32, ctypes.c_uint64, ctypes.c_void_p, ctypes.c_int, ctypes.c_float
    L.elx_ops_source_sha.restype = ctypes.c_char_p
    L.elx_ops_source_sha.argtypes = []
    for name, args in (('elx_layer_norm_bwd_workspace', [u64, u32]), ('elx_embedding_bwd_workspace', [u64, u64, u32])):
        getattr(L, name).restype = u64
        getattr(L, name).argtypes = args
    for name in ('elx_sizeof_state8', 'elx_state8_block', 'elx_layer_norm_max_cols'):
        getattr(L, name).restype = u32
        getattr(L, name).argtypes = []
    for name, args in (('elx_ops_version', []),
                       ('elx_check_state8', [vp, vp, u32]),
                       ('elx_adam8_step_mt', [vp, vp, u32, vp, u32, vp, u32, u64, u32, flt, cint, cint, u32, u32, vp]),
                       ('elx_adam8_step_args_mt', [vp, vp, u32, vp, u32, vp, u32, u64, u32, flt, cint, cint, u32, u32, vp]),
                       ('elx_adam8_step_gated_mt', [vp, vp, u32, vp, u32, vp, u32, u64, u32, cint, cint, u32, u32, vp]),
                       ('elx_state8_read', [vp, vp, vp, u64, u64, vp, vp, cint, vp]),
                       ('elx_state8_write', [vp, u64, cint, vp, vp, vp]),
                       ('elx_layer_norm_fwd', [vp, vp, vp, vp, vp, vp, u64, u32, u64, flt, cint, vp]),
                       ('elx_layer_norm_bwd', [vp, vp, vp, vp, vp, vp, vp, vp, vp, u64, u64, u32, u64, u64, cint, vp]),
                       ('elx_embedding_fwd', [vp, cint, u64, vp, u64, u32, flt, vp, cint, vp]),
                       ('elx_embedding_bwd', [vp, cint, u64, vp, u64, vp, u64, u32, flt, ctypes.c_int64, vp, u64, cint, vp])):
        getattr(L, name).restype = cint
        getattr(L, name).argtypes = args
    if L.elx_ops_version() != ELX_OPS_VERSION:
        raise RuntimeError(f'{LIB_PATH}: version {L.elx_ops_version()} != binding version {ELX_OPS_VERSION}; rebuild')
    built, now = (L.elx_ops_source_sha() or b'').decode(), source_sha16()
    if built != now:
        raise RuntimeError(f'{LIB_PATH} was built from other sources (digest {built or "none"}) than the ones beside it '
                           f'({now}): rebuild with `python -m elixir_amd.build`')
    if L.elx_sizeof_state8() != STATE8_DTYPE.itemsize or L.elx_state8_block() != STATE_BLOCK:
        raise RuntimeError(f'{LIB_PATH}: the records of the 8-bit state are not those of this binding')
    _lib = L
    return L


def _ptr(a: np.ndarray):
    assert a.flags['C_CONTIGUOUS']
    return a.ctypes.data_as(ctypes.c_void_p)


# ---- Adam with an 8-bit state


def check_state8(rows: np.ndarray, state: np.ndarray) -> None:
    """Validate the host copy of the state rows that belong to the update rows."""
    assert rows.dtype == _abi.CHUNK_DTYPE and state.dtype == STATE8_DTYPE and len(rows) == len(state)
    _abi.check('elx_check_state8', load().elx_check_state8(_ptr(rows), _ptr(state), len(rows)))


def adam8_step_mt(d_chunks: int, d_state: int, n_chunks: int, d_segs: int, n_segs: int, d_hypers: int, n_hypers: int,
                  info: '_abi.TableInfo', div_scale: float, grad_dtype: int, lowp_dtype: int, blocks_per_cu: int,
                  stream: int) -> None:
    _abi.check('elx_adam8_step_mt',
               load().elx_adam8_step_mt(d_chunks, d_state, n_chunks, d_segs, n_segs, d_hypers, n_hypers, info.total_tiles,
                                        info.max_tiles, div_scale, grad_dtype, lowp_dtype, info.flags, blocks_per_cu, stream))


def adam8_step_args_mt(d_chunks: int, d_state: int, n_chunks: int, d_segs: int, n_segs: int, hyper_host: np.ndarray,
                       info: '_abi.TableInfo', div_scale: float, grad_dtype: int, lowp_dtype: int, blocks_per_cu: int,
                       stream: int) -> None:
    """Up to ``_abi.MAX_ARG_HYPERS`` hyper records from host memory, in the arguments of the launch."""
    assert hyper_host.dtype == _abi.HYPER_DTYPE
    _abi.check('elx_adam8_step_args_mt',
               load().elx_adam8_step_args_mt(d_chunks, d_state, n_chunks, d_segs, n_segs, _ptr(hyper_host), len(hyper_host),
                                             info.total_tiles, info.max_tiles, div_scale, grad_dtype, lowp_dtype, info.flags,
                                             blocks_per_cu, stream))


def adam8_step_gated_mt(d_chunks: int, d_state: int, n_chunks: int, d_segs: int, n_segs: int, d_hypers: int, n_hypers: int,
                        info: '_abi.TableInfo', grad_dtype: int, lowp_dtype: int, blocks_per_cu: int, stream: int) -> None:
    _abi.check('elx_adam8_step_gated_mt',
               load().elx_adam8_step_gated_mt(d_chunks, d_state, n_chunks, d_segs, n_segs, d_hypers, n_hypers,
                                              info.total_tiles, info.max_tiles, grad_dtype, lowp_dtype, info.flags,
                                              blocks_per_cu, stream))


def state8_read(m_codes: int, v_codes: int, scales: int, begin: int, n: int, m_out: int, v_out: int, out_dtype: int,
                stream: int) -> None:
    _abi.check('elx_state8_read',
               load().elx_state8_read(m_codes or None, v_codes or None, scales, begin, n, m_out or None, v_out or None,
                                      out_dtype, stream))


def state8_write(values: int, n: int, moment: int, codes: int, scales: int, stream: int) -> None:
    _abi.check('elx_state8_write', load().elx_state8_write(values, n, moment, codes, scales, stream))


# ---- layer norm, embedding


def layer_norm_max_cols() -> int:
    return int(load().elx_layer_norm_max_cols())


def layer_norm_bwd_workspace(rows: int, cols: int) -> int:
    return int(load().elx_layer_norm_bwd_workspace(rows, cols))


def layer_norm_fwd(x: int, w: int, b: int, y: int, mean: int, rstd: int, rows: int, cols: int, x_stride: int, eps: float, dtype: int,
                   stream: int) -> None:
    _abi.check('elx_layer_norm_fwd',
               load().elx_layer_norm_fwd(x, w or None, b or None, y, mean or None, rstd or None, rows, cols, x_stride, eps, dtype,
                                         stream))


def layer_norm_bwd(dy: int, x: int, w: int, mean: int, rstd: int, dx: int, dw: int, db: int, workspace: int, workspace_bytes: int,
                   rows: int, cols: int, dy_stride: int, x_stride: int, dtype: int, stream: int) -> None:
    _abi.check('elx_layer_norm_bwd',
               load().elx_layer_norm_bwd(dy, x, w or None, mean, rstd, dx or None, dw or None, db or None, workspace or None,
                                         workspace_bytes, rows, cols, dy_stride, x_stride, dtype, stream))


def embedding_fwd(index: int, index_bytes: int, n: int, table: int, vocab: int, cols: int, scale: float, out: int, dtype: int,
                  stream: int) -> None:
    _abi.check('elx_embedding_fwd',
               load().elx_embedding_fwd(index, index_bytes, n, table, vocab, cols, scale, out, dtype, stream))


def embedding_bwd_workspace(n: int, vocab: int, cols: int) -> int:
    return int(load().elx_embedding_bwd_workspace(n, vocab, cols))


def embedding_bwd(index: int, index_bytes: int, n: int, dy: int, dy_stride: int, dtable: int, vocab: int, cols: int, scale: float,
                  padding: int, workspace: int, workspace_bytes: int, dtype: int, stream: int) -> None:
    _abi.check('elx_embedding_bwd',
               load().elx_embedding_bwd(index, index_bytes, n, dy, dy_stride, dtable, vocab, cols, scale, padding, workspace,
                                        workspace_bytes, dtype, stream))
