"""torch operators over the C ABI (namespace ``hilberta_hip``).

The reference launches its kernels as framework-visible Triton launches (paired_kernel.py:181-204,
sparse_kernel.py:315-339) and gathers with ``index_select`` (flux_adapter.py:209-212, :243).
Here each HIP entry point of include/hilberta_hip.h is a registered operator with a schema and a HIP
implementation (csrc/torch_ops.cpp, libhilberta_torch.so, loaded below), a fake (shape-only)
implementation for tracing and, for pair_rows alone, a CPU one:

  hilberta_hip::paired_fwd(q, k, v, out!, lse!?, kv_indices, kv_flags, kv_counts, global_tokens,
                           key_block_size, scale_log2, all_queries, num_groups) -> ()
  hilberta_hip::sparse_fwd(q, k, v, out!, lse!?, kv_indices, kv_counts, global_tokens,
                           scale_log2, all_queries, num_groups) -> ()
  hilberta_hip::gather_rows(x, dim, index) -> Tensor
  hilberta_hip::pair_rows(kv_indices, kv_counts, total_blocks, key_block_size, paired_width)
                           -> (ids, flags, counts)
  hilberta_hip::int8_rows(x) -> (q, scale)
  hilberta_hip::int8_adaln(x, shift, scale, y?, gate?, x_out!?, eps) -> (q, row_scale)
  hilberta_hip::int8_linear(q, scale, weight, weight_scale, bias?, dtype, gelu) -> Tensor
  hilberta_hip::int8_linear_rows(x, weight, weight_scale, bias?, gelu) -> Tensor  (int8_rows, then int8_linear)
  hilberta_hip::int8_linear_out(q, scale, weight, weight_scale, bias?, out!, gelu) -> ()
  hilberta_hip::int8_qkv_out(text_q?, text_scale?, text_weight?, text_weight_scale?, text_bias?, text_norm_q?,
                             text_norm_k?, q, scale, weight, weight_scale, bias?, norm_q?, norm_k?, cos?, sin?,
                             out!, eps) -> ()
  hilberta_hip::int8_qkv(.. as int8_qkv_out up to sin?, dtype, heads, eps) -> Tensor [3, B, N, heads, 128]
  hilberta_hip::int8_adaln_pair, int8_linear_pair_out: two row sets' arguments (the second's names end in 2)

The attention ops write into caller-provided outputs (declared mutated), as the reference's
launches write into ``out``.  Argument checks with the reference's messages stay in the Python
entry points (paired_attention, sparse_attention) and run before the op; the library repeats the
cheap ones and reports them as ValueError.  The attention and gather ops have no CPU kernel: on
CPU tensors they raise.  pair_rows is plan setup and also runs on CPU tensors, through the
library's host table builder (hb_pair_rows_host, bit-identical to the device kernel).  The 8-bit ops
(flux_int8.py) check their arguments on any device and refuse CPU tensors.  Without the
built library the operators do not exist and every use of one raises.
"""

import torch
from torch import Tensor

from ._lib import LIB_PATH, header_abi_version, load

_NS = "hilberta_hip"
TORCH_LIB_PATH = LIB_PATH.with_name("libhilberta_torch.so")
# key blocks per row hb_pair_rows pairs (include/hilberta_hip.h)
PAIR_MAX_BLOCKS = 16384


def _fake_none(*args):
    return None


def _fake_pair_rows(kv_indices, kv_counts, total_blocks, key_block_size, paired_width):
    prows = (kv_indices.shape[0] + 1) // 2
    ids = kv_indices.new_empty((prows, paired_width))
    return ids, torch.empty_like(ids), kv_indices.new_empty((prows,))


def _fake_gather_rows(x, dim, index):
    shape = list(x.shape)
    shape[dim % x.ndim] = index.shape[0]
    return x.new_empty(shape)


def _fake_int8_rows(x, *args):
    *lead, features = x.shape
    return (x.new_empty((*lead, (features + 63) // 64 * 64), dtype=torch.int8),
            x.new_empty(lead, dtype=torch.float32))


def _fake_int8_adaln_pair(x, shift, scale, y, gate, x_out, x2, *args):
    return (*_fake_int8_rows(x), *_fake_int8_rows(x2))


def _fake_int8_linear(q, scale, weight, weight_scale, bias, dtype, gelu):
    return q.new_empty((*q.shape[:-1], weight.shape[0]), dtype=dtype)


def _fake_int8_linear_rows(x, weight, weight_scale, bias, gelu):
    return x.new_empty((*x.shape[:-1], weight.shape[0]))


def _fake_int8_qkv(text_q, text_scale, text_weight, text_weight_scale, text_bias, text_norm_q, text_norm_k, q, scale,
                   weight, weight_scale, bias, norm_q, norm_k, cos, sin, dtype, heads, eps):
    tokens = q.shape[1] + (0 if text_q is None else text_q.shape[1])
    return q.new_empty((3, q.shape[0], tokens, heads, 128), dtype=dtype)


def _pair_rows_cpu(kv_indices: Tensor, kv_counts: Tensor, total_blocks: int, key_block_size: int,
                   paired_width: int) -> tuple[Tensor, Tensor, Tensor]:
    """pair_rows of CPU tensors by hb_pair_rows_host."""
    from ._tables import pair_rows_device

    return pair_rows_device(kv_indices, kv_counts, total_blocks, key_block_size=key_block_size,
                            paired_width=paired_width)


class _Missing:
    """An operator whose library could not be loaded: calling it raises."""

    def __init__(self, name, reason):
        self.name, self.reason = name, reason

    def __call__(self, *args, **kwargs):
        raise RuntimeError(f"{_NS}::{self.name}: {self.reason}")


def _load():
    """The operators of libhilberta_torch.so, in the order they are bound below."""
    if not TORCH_LIB_PATH.exists():
        raise RuntimeError(f"{TORCH_LIB_PATH} is missing: build the library first "
                           "(python -m hilberta_amd.build); there is no CPU fallback")
    load()  # the C ABI library, its version checked, before the operators bind to it
    torch.ops.load_library(str(TORCH_LIB_PATH))
    version = getattr(getattr(torch.ops, _NS), "_abi_version", None)  # (absent in the oldest ones)
    built, declared = version() if version else 0, header_abi_version()
    if built != declared:
        raise RuntimeError(f"{TORCH_LIB_PATH} was built for {f'ABI {built}' if built else 'an older ABI'} but "
                           f"include/hilberta_hip.h declares ABI {declared}: rebuild the libraries "
                           "(python -m hilberta_amd.build)")
    for name in _NAMES:
        if not hasattr(getattr(torch.ops, _NS), name):
            raise RuntimeError(f"{TORCH_LIB_PATH} lacks {name}: rebuild the libraries (python -m hilberta_amd.build)")
    fakes = dict(paired_fwd=_fake_none, sparse_fwd=_fake_none, pair_rows=_fake_pair_rows,
                 gather_rows=_fake_gather_rows, int8_rows=_fake_int8_rows, int8_adaln=_fake_int8_rows,
                 int8_adaln_pair=_fake_int8_adaln_pair, int8_linear=_fake_int8_linear,
                 int8_linear_rows=_fake_int8_linear_rows, int8_linear_out=_fake_none,
                 int8_linear_pair_out=_fake_none, int8_qkv=_fake_int8_qkv, int8_qkv_out=_fake_none)
    for name, fake in fakes.items():
        torch.library.register_fake(f"{_NS}::{name}", fake)
    torch.library.impl(f"{_NS}::pair_rows", "cpu", _pair_rows_cpu)
    return [getattr(getattr(torch.ops, _NS), name).default for name in _NAMES]


_NAMES = ("paired_fwd", "sparse_fwd", "pair_rows", "gather_rows", "_attention_workspace",
          "_workspace_keys", "_clear_workspaces", "int8_rows", "int8_adaln", "int8_adaln_pair", "int8_linear",
          "int8_linear_rows", "int8_linear_out", "int8_linear_pair_out", "int8_qkv", "int8_qkv_out")
try:
    _bound = _load()
except (RuntimeError, OSError) as e:  # the package still imports, so that it can be (re)built
    _bound = [_Missing(name, str(e)) for name in _NAMES]
(paired_fwd, sparse_fwd, pair_rows, gather_rows, attention_workspace, workspace_keys, clear_workspaces,
 int8_rows, int8_adaln, int8_adaln_pair, int8_linear, int8_linear_rows, int8_linear_out, int8_linear_pair_out,
 int8_qkv, int8_qkv_out) = _bound
