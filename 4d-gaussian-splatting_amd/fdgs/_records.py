"""Argument structures of the entry points over lists of tensors and over tables (fdgs_adamw_step, fdgs_moment8_*,
fdgs_embedding_*): the ctypes side of include/fdgs.h, and the packed records of the per-tensor arrays.

An array of records goes to the library in one piece: `struct` packs all its fields at once, which takes a fraction of
the time of setting them one by one (a step over 200 tensors has 3000 of them)."""
import ctypes as C
import struct

TYPE_F32, TYPE_BF16, TYPE_F16 = 0, 1, 2
MOMENT8_BLOCK = 256

# fdgs_adamw_tensor: seven pointers, numel, grad_row_stride, grad_row_len, step, lr, weight_decay, round_key, reserved
ADAMW_TENSOR = "7Qqqiidd2I"
# fdgs_moment8_tensor: codes, exponents, value, numel, is_signed, round_key
MOMENT8_TENSOR = "3QqiI"


class AdamWTensor(C.Structure):
    _fields_ = [("param", C.c_void_p), ("grad", C.c_void_p), ("exp_avg", C.c_void_p), ("exp_avg_sq", C.c_void_p),
                ("residual", C.c_void_p), ("exp_avg_exponents", C.c_void_p), ("exp_avg_sq_exponents", C.c_void_p),
                ("numel", C.c_int64), ("grad_row_stride", C.c_int64), ("grad_row_len", C.c_int32), ("step", C.c_int32),
                ("lr", C.c_double), ("weight_decay", C.c_double), ("round_key", C.c_uint32), ("reserved", C.c_uint32)]


class AdamWArgs(C.Structure):
    _fields_ = [("num_tensors", C.c_int32), ("param_type", C.c_int32), ("state_bits", C.c_int32),
                ("reserved", C.c_int32), ("beta1", C.c_double), ("beta2", C.c_double), ("eps", C.c_double),
                ("tensors", C.c_char_p)]


class Moment8Tensor(C.Structure):
    _fields_ = [("codes", C.c_void_p), ("exponents", C.c_void_p), ("value", C.c_void_p), ("numel", C.c_int64),
                ("is_signed", C.c_int32), ("round_key", C.c_uint32)]


class Moment8Args(C.Structure):
    _fields_ = [("num_tensors", C.c_int32), ("value_type", C.c_int32), ("nearest", C.c_int32), ("reserved", C.c_int32),
                ("tensors", C.c_char_p)]


EMBEDDING_MAX_TOKENS = 1 << 30          # FDGS_EMBEDDING_MAX_TOKENS


class EmbeddingFwdArgs(C.Structure):
    _fields_ = [("num_tokens", C.c_int64), ("num_rows", C.c_int32), ("dim", C.c_int32), ("type", C.c_int32),
                ("id_bytes", C.c_int32), ("ids", C.c_void_p), ("table", C.c_void_p), ("table_row_stride", C.c_int64),
                ("padding_id", C.c_int64), ("out", C.c_void_p), ("scale", C.c_float)]


class EmbeddingBwdArgs(C.Structure):
    _fields_ = [("num_tokens", C.c_int64), ("num_rows", C.c_int32), ("dim", C.c_int32), ("type", C.c_int32),
                ("id_bytes", C.c_int32), ("ids", C.c_void_p), ("grad_out", C.c_void_p),
                ("grad_out_row_stride", C.c_int64), ("padding_id", C.c_int64), ("grad_table", C.c_void_p),
                ("scale", C.c_float), ("workspace", C.c_void_p), ("workspace_bytes", C.c_size_t)]


_PACKERS = {}


def pack(fmt, count, fields):
    """A host array of `count` records with the format `fmt`, from the flat list of their fields."""
    key = (fmt, count)
    packer = _PACKERS.get(key)
    if packer is None:
        if len(_PACKERS) > 256:         # a program has a handful of list lengths
            _PACKERS.clear()
        packer = _PACKERS[key] = struct.Struct("=" + fmt * count)
    return packer.pack(*fields)
