"""Argument structures of the entry points over lists of tensors and over tables (fdgs_adamw_step, fdgs_moment8_*,
fdgs_embedding_*): the ctypes side of include/fdgs.h.  The package makes these calls from fdgs._host (csrc/host.cpp);
the structures here are for a caller of the C ABI, and for calls that are profiled."""
import ctypes as C

TYPE_F32, TYPE_BF16, TYPE_F16 = 0, 1, 2
MOMENT8_BLOCK = 256


class AdamWTensor(C.Structure):
    _fields_ = [("param", C.c_void_p), ("grad", C.c_void_p), ("exp_avg", C.c_void_p), ("exp_avg_sq", C.c_void_p),
                ("residual", C.c_void_p), ("exp_avg_exponents", C.c_void_p), ("exp_avg_sq_exponents", C.c_void_p),
                ("numel", C.c_int64), ("grad_row_stride", C.c_int64), ("grad_row_len", C.c_int32), ("step", C.c_int32),
                ("lr", C.c_double), ("weight_decay", C.c_double), ("round_key", C.c_uint32), ("reserved", C.c_uint32)]


class AdamWArgs(C.Structure):
    _fields_ = [("num_tensors", C.c_int32), ("param_type", C.c_int32), ("state_bits", C.c_int32),
                ("reserved", C.c_int32), ("beta1", C.c_double), ("beta2", C.c_double), ("eps", C.c_double),
                ("tensors", C.c_char_p), ("workspace", C.c_void_p), ("workspace_bytes", C.c_size_t)]


class Moment8Tensor(C.Structure):
    _fields_ = [("codes", C.c_void_p), ("exponents", C.c_void_p), ("value", C.c_void_p), ("numel", C.c_int64),
                ("is_signed", C.c_int32), ("round_key", C.c_uint32)]


class Moment8Args(C.Structure):
    _fields_ = [("num_tensors", C.c_int32), ("value_type", C.c_int32), ("nearest", C.c_int32), ("reserved", C.c_int32),
                ("tensors", C.c_char_p), ("workspace", C.c_void_p), ("workspace_bytes", C.c_size_t)]


EMBEDDING_MAX_TOKENS = 1 << 30          # FDGS_EMBEDDING_MAX_TOKENS


class EmbeddingFwdArgs(C.Structure):
    _fields_ = [("num_tokens", C.c_int64), ("num_rows", C.c_int32), ("dim", C.c_int32), ("type", C.c_int32),
                ("id_bytes", C.c_int32), ("ids", C.c_void_p), ("table", C.c_void_p), ("table_row_stride", C.c_int64),
                ("padding_id", C.c_int64), ("out", C.c_void_p), ("scale", C.c_float), ("sorted", C.c_void_p),
                ("workspace", C.c_void_p), ("workspace_bytes", C.c_size_t)]


class EmbeddingBwdArgs(C.Structure):
    _fields_ = [("num_tokens", C.c_int64), ("num_rows", C.c_int32), ("dim", C.c_int32), ("type", C.c_int32),
                ("id_bytes", C.c_int32), ("ids", C.c_void_p), ("grad_out", C.c_void_p),
                ("grad_out_row_stride", C.c_int64), ("padding_id", C.c_int64), ("grad_table", C.c_void_p),
                ("scale", C.c_float), ("sorted", C.c_void_p), ("workspace", C.c_void_p), ("workspace_bytes", C.c_size_t)]
