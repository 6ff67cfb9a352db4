"""ctypes bindings of the MI355X decode engine (libchpe.so) and the archive writer
(libchpe_pack.so), both built in this directory by its Makefile.

The engine API mirrors the reference's C ABI (src/chpe_c_api.zig) plus the additions
declared in include/chpe.h.  Nothing here computes on the CPU: a missing or unloadable
libchpe.so raises, it is never replaced by a fallback.
"""
import ctypes
import os
import shutil
from pathlib import Path

import numpy as np

PKG_DIR = Path(__file__).resolve().parent
ENGINE_LIB = PKG_DIR / "libchpe.so"
PACK_LIB = PKG_DIR / "libchpe_pack.so"

ARCH_3B, ARCH_9B, ARCH_72B = 0, 1, 2
# archive kinds of chpe_pack_write (include/chpe_pack.h)
(PACK_3B_FP16_RAW, PACK_3B_BF16_RAW, PACK_3B_W4, PACK_3B_W2, PACK_3B_W4_STD, PACK_72B_W4, PACK_72B_W2,
 PACK_9B_W4) = range(8)

# every symbol include/chpe.h declares, in order
ENGINE_SYMBOLS = [
    "chpe_init", "chpe_forward_tokens", "chpe_get_last_logits", "chpe_get_vocab_size",
    "chpe_get_hidden_dim", "chpe_get_num_layers", "chpe_get_last_elapsed_ns",
    "chpe_get_last_argmax", "chpe_get_last_max_logit", "chpe_get_last_token0_logit",
    "chpe_get_last_hidden_norm", "chpe_free", "chpe_init_ex", "chpe_decode_step",
    "chpe_generate", "chpe_verify", "chpe_prefill", "chpe_block_ready", "chpe_last_error", "chpe_build_id", "chpe_get_max_seq_len", "chpe_get_hidden",
    "chpe_time_steps", "chpe_time_stage", "chpe_time_stage_live", "chpe_stage_bytes", "chpe_step_bytes", "chpe_stage_kernel",
    "chpe_debug_gemv", "chpe_debug_flat_tile_weights", "chpe_debug_gemv_flat", "chpe_debug_gemv_cells", "chpe_debug_gemv_poly", "chpe_debug_gemv_raw", "chpe_debug_embed_row_cell",
    "chpe_debug_attention", "chpe_debug_attention_block", "chpe_attention_noalloc", "chpe_paged_append",
    "chpe_paged_attention", "chpe_paged_attention_workspace", "chpe_paged_evict", "chpe_paged_evict_workspace",
    "chpe_debug_deltanet_conv", "chpe_debug_deltanet_step",
]

_c_float_p = ctypes.POINTER(ctypes.c_float)
_c_u32_p = ctypes.POINTER(ctypes.c_uint32)
_c_u8_p = ctypes.POINTER(ctypes.c_uint8)
_engine_lib = None
_pack_lib = None


_U32_MAX = 0xffffffff  # (ctypes keeps the low 32 bits of what is larger, without a word)


class _KvPages(ctypes.Structure):  # chpe_kv_pages
    _fields_ = [("k", ctypes.c_void_p), ("v", ctypes.c_void_p), ("type", ctypes.c_int),
                *[(n, ctypes.c_uint32) for n in ("kv_heads", "head_dim", "page_size", "n_pages")],
                *[(n, ctypes.c_uint64) for n in ("page_stride", "head_stride", "slot_stride")],
                ("table", ctypes.c_void_p), *[(n, ctypes.c_uint32) for n in ("rows", "pages_per_row", "table_stride")]]


def _fp(a):
    return a.ctypes.data_as(_c_float_p)


def source_hash():
    """The hash libchpe.so carries of the sources it was built from (chpe_build_id): the
    Makefile's LIBSRC list, in its order, through SHA-256, first 16 hex digits."""
    import hashlib
    src = PKG_DIR / "csrc"
    files = sorted(list(src.glob("*.hip")) + list(src.glob("*.hpp")), key=lambda p: f"csrc/{p.name}")
    files += [src / "engine.cpp", src / "c_api.cpp", PKG_DIR.parent / "include" / "chpe.h", PKG_DIR / "Makefile"]
    h = hashlib.sha256()
    for f in files:
        h.update(f.read_bytes())
    return h.hexdigest()[:16]


def load_engine_lib():
    """Load libchpe.so (raises OSError when it is not built, or was built from other sources
    than the ones beside it)."""
    global _engine_lib
    if _engine_lib is None:
        if not ENGINE_LIB.exists():
            raise OSError(f"{ENGINE_LIB} is not built (run `make -C {PKG_DIR}`)")
        lib = ctypes.CDLL(str(ENGINE_LIB))
        lib.chpe_build_id.restype = ctypes.c_char_p
        built, here = lib.chpe_build_id().decode(), source_hash()
        if built != here:
            raise OSError(f"{ENGINE_LIB} was built from other sources (build id {built}, sources {here}): "
                          f"run `make -C {PKG_DIR}`")
        V, S, I, U64, F, D = (ctypes.c_void_p, ctypes.c_size_t, ctypes.c_int, ctypes.c_uint64,
                              ctypes.c_float, ctypes.c_double)
        U32, P = ctypes.c_uint32, ctypes.POINTER(_KvPages)
        sig = {
            "chpe_init": (V, [ctypes.c_char_p]),
            "chpe_forward_tokens": (I, [V, _c_u32_p, S, _c_float_p]),
            "chpe_get_last_logits": (S, [V, _c_float_p, S]),
            "chpe_get_vocab_size": (S, [V]),
            "chpe_get_hidden_dim": (S, [V]),
            "chpe_get_num_layers": (S, [V]),
            "chpe_get_last_elapsed_ns": (U64, [V]),
            "chpe_get_last_argmax": (ctypes.c_uint32, [V]),
            "chpe_get_last_max_logit": (F, [V]),
            "chpe_get_last_token0_logit": (F, [V]),
            "chpe_get_last_hidden_norm": (F, [V]),
            "chpe_free": (None, [V]),
            "chpe_init_ex": (V, [ctypes.c_char_p, I, S, I]),
            "chpe_decode_step": (I, [V, ctypes.c_uint32, S, _c_float_p]),
            "chpe_generate": (I, [V, _c_u32_p, S, S, _c_u32_p]),
            "chpe_prefill": (I, [V, _c_u32_p, S, _c_float_p]),
            "chpe_block_ready": (I, [V]),
            "chpe_verify": (I, [V, _c_u32_p, S, S, _c_u32_p]),
            "chpe_last_error": (ctypes.c_char_p, []),
            "chpe_build_id": (ctypes.c_char_p, []),
            "chpe_get_max_seq_len": (S, [V]),
            "chpe_get_hidden": (I, [V, _c_float_p]),
            "chpe_time_steps": (I, [V, S, _c_float_p]),
            "chpe_time_stage": (I, [V, I, S, S, S, _c_float_p]),
            "chpe_time_stage_live": (I, [V, I, S, _c_float_p]),
            "chpe_stage_bytes": (D, [V, I, S]),
            "chpe_step_bytes": (D, [V, S]),
            "chpe_stage_kernel": (ctypes.c_char_p, [V, I]),
            "chpe_debug_gemv": (I, [V, S, I, _c_float_p, _c_float_p]),
            "chpe_debug_flat_tile_weights": (I, [_c_u8_p, _c_float_p]),
            "chpe_debug_gemv_flat": (I, [I, ctypes.c_uint32, ctypes.c_uint32, _c_u8_p, _c_u8_p, S, _c_float_p,
                                         _c_float_p, F, _c_float_p, _c_u32_p, _c_float_p]),
            "chpe_debug_gemv_cells": (I, [I, ctypes.c_uint32, _c_u8_p, _c_u8_p, S, _c_float_p, _c_float_p, F,
                                          _c_float_p, _c_u32_p, _c_float_p]),
            "chpe_debug_gemv_poly": (I, [I, ctypes.c_uint32, ctypes.c_uint32, _c_u8_p, _c_u8_p, S, _c_float_p,
                                         _c_float_p, F, _c_float_p, _c_u32_p, _c_float_p]),
            "chpe_debug_gemv_raw": (I, [I, ctypes.c_uint32, ctypes.c_uint32, I, _c_u8_p, _c_u8_p, S, _c_float_p,
                                        _c_float_p, F, _c_float_p, _c_u32_p, _c_float_p]),
            "chpe_debug_embed_row_cell": (I, [_c_u8_p, S, ctypes.c_uint32, ctypes.c_uint32, _c_float_p]),
            "chpe_debug_attention": (I, [ctypes.c_uint32, ctypes.c_uint32, ctypes.c_uint32, I, ctypes.c_uint32,
                                         _c_float_p, _c_float_p, _c_float_p, _c_float_p]),
            "chpe_debug_attention_block": (I, [ctypes.c_uint32, ctypes.c_uint32, ctypes.c_uint32, I, ctypes.c_uint32,
                                               ctypes.c_uint32, _c_float_p, _c_float_p, _c_float_p, _c_float_p]),
            "chpe_attention_noalloc": (I, [ctypes.c_uint32, ctypes.c_uint32, ctypes.c_uint32, I, ctypes.c_uint32,
                                           ctypes.c_uint32, V, V, V, V, V]),
            "chpe_paged_append": (I, [P, U32, U32, V, U64, U64, V, U64, V, U64, V, V, F, V, V, U32, U32, I, V, V, V, V, V,
                                      V, U64, V]),
            "chpe_paged_attention": (I, [P, U32, V, U32, V, U64, F, U32, V, U64, V, V, U64, V, S, V]),
            "chpe_paged_attention_workspace": (S, [P, U32, U32, I]),
            "chpe_paged_evict": (I, [P, V, U32, U32, U32, U32, V, V, U64, V, V, V, V, V, S, V]),
            "chpe_paged_evict_workspace": (S, [P, U32]),
            "chpe_debug_deltanet_conv": (I, [ctypes.c_uint32, ctypes.c_uint32, _c_float_p, _c_float_p, _c_float_p,
                                             _c_float_p]),
            "chpe_debug_deltanet_step": (I, [ctypes.c_uint32] * 3 + [_c_float_p] * 9 + [F, _c_float_p, _c_float_p]),
        }
        for name, (res, args) in sig.items():
            fn = getattr(lib, name)
            fn.restype = res
            fn.argtypes = args
        _engine_lib = lib
    return _engine_lib


def load_pack_lib():
    global _pack_lib
    if _pack_lib is None:
        if not PACK_LIB.exists():
            raise OSError(f"{PACK_LIB} is not built (run `make -C {PKG_DIR}`)")
        lib = ctypes.CDLL(str(PACK_LIB))
        lib.chpe_pack_size.restype = ctypes.c_uint64
        lib.chpe_pack_size.argtypes = [ctypes.c_int]
        lib.chpe_pack_write.restype = ctypes.c_int
        lib.chpe_pack_write.argtypes = [ctypes.c_char_p, ctypes.c_int, ctypes.c_uint64, ctypes.c_int]
        lib.chpe_pack_records.restype = ctypes.c_int
        lib.chpe_pack_records.argtypes = [ctypes.c_int, ctypes.c_uint64, ctypes.c_uint64, ctypes.c_uint64,
                                          ctypes.c_int, _c_u8_p]
        lib.chpe_pack_header.restype = ctypes.c_int
        lib.chpe_pack_header.argtypes = [ctypes.c_int, _c_u8_p]
        lib.chpe_pack_normals.restype = None
        lib.chpe_pack_normals.argtypes = [ctypes.c_uint64, ctypes.c_uint64, ctypes.c_uint64,
                                          ctypes.c_uint64, ctypes.c_float, _c_float_p]
        lib.chpe_pack_cell16.restype = ctypes.c_int
        lib.chpe_pack_cell16.argtypes = [_c_float_p, ctypes.c_int, ctypes.c_int, ctypes.c_int,
                                         ctypes.c_int, ctypes.c_uint32, _c_u8_p]
        lib.chpe_pack_flat.restype = ctypes.c_int
        lib.chpe_pack_flat.argtypes = [_c_float_p, ctypes.c_int, ctypes.c_int, ctypes.c_uint32, _c_u8_p]
        _pack_lib = lib
    return _pack_lib


# ------------------------------------------------------------------ archive writer
def archive_size(kind):
    return int(load_pack_lib().chpe_pack_size(kind))


def write_archive(path, kind, seed=0, threads=0):
    rc = load_pack_lib().chpe_pack_write(str(path).encode(), kind, seed, threads)
    if rc != 0:
        raise RuntimeError(f"chpe_pack_write({path}, kind={kind}) failed: {rc}")
    return path


def pack_records(kind, first, count, seed=0, threads=0):
    """Records [first, first + count) of archive `kind`, as they lie in the file, as a
    (count, record_bytes) uint8 array."""
    rb = 16384 if kind in (PACK_3B_FP16_RAW, PACK_3B_BF16_RAW) else (20480 if kind == PACK_3B_W4_STD else 17408)
    out = np.zeros((count, rb), dtype=np.uint8)
    if load_pack_lib().chpe_pack_records(kind, seed, first, count, threads, out.ctypes.data_as(_c_u8_p)) != 0:
        raise ValueError("chpe_pack_records rejected the arguments")
    return out


def pack_header(kind):
    out = np.zeros(4096, dtype=np.uint8)
    if load_pack_lib().chpe_pack_header(kind, out.ctypes.data_as(_c_u8_p)) != 0:
        raise ValueError("chpe_pack_header rejected the kind")
    return out


def normals(seed, tid, first, n, std=0.02):
    out = np.empty(n, dtype=np.float32)
    load_pack_lib().chpe_pack_normals(seed, tid, first, n, std, _fp(out))
    return out


def pack_cell16(w, bits=4, n_outlier_cols=8, layer=0):
    w = np.ascontiguousarray(w, dtype=np.float32)
    cell = np.zeros(17408, dtype=np.uint8)
    rc = load_pack_lib().chpe_pack_cell16(_fp(w), w.shape[0], w.shape[1], bits, n_outlier_cols,
                                          layer, cell.ctypes.data_as(_c_u8_p))
    if rc:
        raise ValueError("chpe_pack_cell16 rejected the shape")
    return cell


def pack_flat(w, bits=4, n_outliers=64, layer=0):
    w = np.ascontiguousarray(w, dtype=np.float32).reshape(32768)
    cell = np.zeros(17408, dtype=np.uint8)
    rc = load_pack_lib().chpe_pack_flat(_fp(w), bits, n_outliers, layer, cell.ctypes.data_as(_c_u8_p))
    if rc:
        raise ValueError("chpe_pack_flat rejected the arguments")
    return cell


# ------------------------------------------------------------------ engine
class EngineError(RuntimeError):
    pass


class Engine:
    """One engine context (chpe_init / chpe_init_ex)."""

    def __init__(self, path, arch=-1, max_seq_len=2048, kv_f16=False, reference_init=False):
        self.lib = load_engine_lib()
        if reference_init:
            self.ctx = self.lib.chpe_init(str(path).encode())
        else:
            self.ctx = self.lib.chpe_init_ex(str(path).encode(), arch, max_seq_len, 1 if kv_f16 else 0)
        if not self.ctx:
            raise EngineError(self.lib.chpe_last_error().decode())
        self.vocab = self.lib.chpe_get_vocab_size(self.ctx)
        self.hidden_dim = self.lib.chpe_get_hidden_dim(self.ctx)
        self.num_layers = self.lib.chpe_get_num_layers(self.ctx)
        self.max_seq_len = self.lib.chpe_get_max_seq_len(self.ctx)

    def close(self):
        if self.ctx:
            self.lib.chpe_free(self.ctx)
            self.ctx = None

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def _check(self, rc, what):
        if rc < 0:
            raise EngineError(f"{what} failed: {rc}")
        return rc

    def forward_tokens(self, tokens, want_logits=False):
        toks = np.ascontiguousarray(tokens, dtype=np.uint32)
        logits = np.empty(self.vocab, dtype=np.float32) if want_logits else None
        rc = self.lib.chpe_forward_tokens(self.ctx, toks.ctypes.data_as(_c_u32_p), toks.size,
                                          _fp(logits) if want_logits else None)
        self._check(rc, "chpe_forward_tokens")
        return (rc, logits) if want_logits else rc

    def decode_step(self, token, pos, want_logits=True):
        logits = np.empty(self.vocab, dtype=np.float32) if want_logits else None
        rc = self.lib.chpe_decode_step(self.ctx, token, pos, _fp(logits) if want_logits else None)
        self._check(rc, "chpe_decode_step")
        return (rc, logits) if want_logits else rc

    def generate(self, prompt, n_gen):
        p = np.ascontiguousarray(prompt, dtype=np.uint32)
        out = np.empty(n_gen, dtype=np.uint32)
        rc = self.lib.chpe_generate(self.ctx, p.ctypes.data_as(_c_u32_p), p.size, n_gen,
                                    out.ctypes.data_as(_c_u32_p))
        self._check(rc, "chpe_generate")
        return out

    def prefill(self, tokens, want_logits=False):
        toks = np.ascontiguousarray(tokens, dtype=np.uint32)
        logits = np.empty(self.vocab, dtype=np.float32) if want_logits else None
        rc = self.lib.chpe_prefill(self.ctx, toks.ctypes.data_as(_c_u32_p), toks.size,
                                   _fp(logits) if want_logits else None)
        self._check(rc, "chpe_prefill")
        return (rc, logits) if want_logits else rc

    def block_ready(self):
        return bool(self.lib.chpe_block_ready(self.ctx))

    def verify(self, drafts, pos):
        d = np.ascontiguousarray(drafts, dtype=np.uint32)
        out = np.empty(d.size, dtype=np.uint32)
        rc = self.lib.chpe_verify(self.ctx, d.ctypes.data_as(_c_u32_p), d.size, pos, out.ctypes.data_as(_c_u32_p))
        self._check(rc, "chpe_verify")
        return out

    def logits(self):
        out = np.empty(self.vocab, dtype=np.float32)
        if self.lib.chpe_get_last_logits(self.ctx, _fp(out), self.vocab) != self.vocab:
            raise EngineError("chpe_get_last_logits failed")
        return out

    def hidden(self):
        out = np.empty(self.hidden_dim, dtype=np.float32)
        self._check(self.lib.chpe_get_hidden(self.ctx, _fp(out)), "chpe_get_hidden")
        return out

    def last(self):
        L = self.lib
        return dict(argmax=L.chpe_get_last_argmax(self.ctx), max_logit=L.chpe_get_last_max_logit(self.ctx),
                    token0_logit=L.chpe_get_last_token0_logit(self.ctx),
                    hidden_norm=L.chpe_get_last_hidden_norm(self.ctx),
                    elapsed_ns=L.chpe_get_last_elapsed_ns(self.ctx))

    def debug_gemv(self, layer, which, x, rows):
        x = np.ascontiguousarray(x, dtype=np.float32)
        y = np.empty(rows, dtype=np.float32)
        self._check(self.lib.chpe_debug_gemv(self.ctx, layer, which, _fp(x), _fp(y)), "chpe_debug_gemv")
        return y

    def time_steps(self, n):
        ms = ctypes.c_float()
        self._check(self.lib.chpe_time_steps(self.ctx, n, ctypes.byref(ms)), "chpe_time_steps")
        return ms.value

    def time_stage(self, stage, layer0, layer1, iters):
        ms = ctypes.c_float()
        self._check(self.lib.chpe_time_stage(self.ctx, stage, layer0, layer1, iters, ctypes.byref(ms)),
                    "chpe_time_stage")
        return ms.value

    def time_stage_live(self, stage, n_steps):
        ms = ctypes.c_float()
        self._check(self.lib.chpe_time_stage_live(self.ctx, stage, n_steps, ctypes.byref(ms)),
                    "chpe_time_stage_live")
        return ms.value

    def stage_bytes(self, stage, layer):
        return self.lib.chpe_stage_bytes(self.ctx, stage, layer)

    def step_bytes(self, pos):
        return self.lib.chpe_step_bytes(self.ctx, pos)

    def stage_kernel(self, stage):
        """The kernel that runs `stage`, demangled when c++filt is available."""
        name = self.lib.chpe_stage_kernel(self.ctx, stage).decode()
        try:
            import subprocess
            out = subprocess.run(["c++filt", name], capture_output=True, text=True, timeout=10)
            return out.stdout.strip() or name
        except (OSError, subprocess.SubprocessError):
            return name


class KvPages:
    """A paged key/value cache in torch tensors and its operators (chpe_paged_*, include/chpe.h): k, v
    [n_pages, kv_heads, page_size, head_dim] (f32, fp16 or bf16; any strides but the last dimension's, the
    same for both), table [rows, pages_per_row] int32.  The tensors stay the caller's: the table's and the
    pages' contents may change between calls.  Calls enqueue on torch's current stream of the tensors'
    device."""

    def __init__(self, k, v, table):
        import torch
        self._torch, self.lib = torch, load_engine_lib()
        types = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
        if k.dim() != 4 or k.shape != v.shape or k.dtype not in types or v.dtype != k.dtype:
            raise ValueError("k and v: [n_pages, kv_heads, page_size, head_dim], both f32, fp16 or bf16")
        if k.stride() != v.stride() or k.stride(3) != 1:
            raise ValueError("k and v: the same strides, the last dimension's 1")
        if table.dim() != 2 or table.dtype != torch.int32 or (table.numel() and table.stride(1) != 1):
            raise ValueError("table: [rows, pages_per_row] int32, the last stride 1")
        if table.shape[0] > 1 and table.stride(0) < table.shape[1]:
            raise ValueError("table: rows that do not lie in each other")
        if max(*k.shape, *table.shape, table.stride(0)) > _U32_MAX:
            raise ValueError("k, v and table: sizes within 32 bits")
        if not k.is_cuda or v.device != k.device or table.device != k.device:
            raise ValueError("k, v and table: on one GPU")
        self.k, self.v, self.table, self.device = k, v, table, k.device
        self.rows, self.kv_heads, self.page_size, self.head_dim = table.shape[0], k.shape[1], k.shape[2], k.shape[3]
        self.capacity = table.shape[1] * self.page_size
        self._c = ctypes.byref(_KvPages(
            k.data_ptr(), v.data_ptr(), types[k.dtype], k.shape[1], k.shape[3], k.shape[2], k.shape[0], k.stride(0), k.stride(1),
            k.stride(2), table.data_ptr(), table.shape[0], table.shape[1],
            table.stride(0) if table.shape[0] > 1 else table.shape[1]))
        self._f32, self._i32, self._index = torch.float32, torch.int32, k.device.index
        # (torch.cuda.current_stream builds an object for every call; a step of one token is a few us)
        self._stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
            lambda i: torch.cuda.current_stream(i).cuda_stream)

    def _call(self, name, *args):
        cuda = self._torch.cuda
        if cuda.current_device() != self._index:
            with cuda.device(self._index):
                return self._call(name, *args)
        rc = getattr(self.lib, name)(self._c, *args, self._stream(self._index))
        if rc:
            raise EngineError(f"{name} failed: {rc}")

    def _take(self, t, name, dtype, shape):
        """The address of a contiguous tensor of this type and shape on the cache's device."""
        if t.dtype is not dtype or t.shape != shape or t.get_device() != self._index or not t.is_contiguous():
            raise ValueError(f"{name}: a contiguous {dtype} tensor of shape {tuple(shape)} on {self.device}")
        return t.data_ptr()

    def _slots(self, t, name, dtype, least):
        """The address of a contiguous [rows, kv_heads, n >= least] tensor."""
        if t.dim() != 3 or t.shape[2] < least:
            raise ValueError(f"{name}: [rows, kv_heads, at least {least}]")
        return self._take(t, name, dtype, (self.rows, self.kv_heads, t.shape[2]))

    def _heads(self, t, name, tokens, heads):
        """Address and first two strides of a [tokens, heads, head_dim] f32 tensor whose last stride is 1."""
        if t.dtype is not self._f32 or t.shape != (tokens, heads, self.head_dim) or t.get_device() != self._index:
            raise ValueError(f"{name}: [{tokens}, {heads}, {self.head_dim}] f32 on {self.device}")
        st, sh, sd = t.stride()
        if heads <= 1:
            sh = self.head_dim
        if tokens <= 1:
            st = heads * sh
        if sd != 1 and t.numel():
            raise ValueError(f"{name}: the last stride 1")
        return t.data_ptr(), st, sh

    def append(self, k, v, rows, slots, positions, q=None, q_norm=None, k_norm=None, eps=1e-6, rope=None,
               interleaved=False, q_out=None, slot_pos=None, slot_weight=None):
        """chpe_paged_append: k, v [tokens, kv_heads, head_dim] f32 at slot slots[t] of row rows[t], rotated by
        positions[t] (int32); rope = (cos, sin), each [n, rot_dim / 2].  q [tokens, heads, head_dim] f32 (its
        first two strides free) gives the rotated queries, which are returned (q_out, or a new tensor)."""
        take, f32, i32, t, hd = self._take, self._f32, self._i32, k.shape[0], self.head_dim
        kp, ks, kh = self._heads(k, "k", t, self.kv_heads)
        vp, vs, vh = self._heads(v, "v", t, self.kv_heads)
        if kh != hd or vh != hd:
            raise ValueError("k and v: contiguous within a token")
        heads = qp = qs = qh = qo = 0
        if q is not None:
            heads = q.shape[1] if q.dim() == 3 else 0
            qp, qs, qh = self._heads(q, "q", t, heads)
            if q_out is None:
                q_out = self._torch.empty(q.shape, dtype=f32, device=self.device)
            qo = take(q_out, "q_out", f32, q.shape)
        gq = None if q_norm is None else take(q_norm, "q_norm", f32, (hd,))
        gk = None if k_norm is None else take(k_norm, "k_norm", f32, (hd,))
        cos = sin = None
        n = half = 0
        if rope is not None:
            shape = rope[0].shape
            n, half = shape
            cos, sin = take(rope[0], "rope's cosines", f32, shape), take(rope[1], "rope's sines", f32, shape)
        if max(t, n) > _U32_MAX:
            raise ValueError("tokens and rope's rows: within 32 bits")
        track, sp, sw = 0, None, None
        if slot_pos is not None:
            sp, track = self._slots(slot_pos, "slot_pos", i32, 1), slot_pos.shape[2]
        if slot_weight is not None:
            sw = self._slots(slot_weight, "slot_weight", f32, track or 1)
            if track and slot_weight.shape[2] != track:
                raise ValueError("slot_pos and slot_weight: the same shape")
            track = slot_weight.shape[2]
        self._call("chpe_paged_append", t, heads, qp, qs, qh, kp, ks, vp, vs, gq, gk, eps, cos, sin, 2 * half, n,
                   1 if interleaved else 0, take(rows, "rows", i32, (t,)), take(slots, "slots", i32, (t,)),
                   take(positions, "positions", i32, (t,)), qo, sp, sw, track)
        return q_out

    def attention_workspace(self, heads, max_len, weights=False):
        """Bytes that attention() needs for these sizes."""
        if min(heads, max_len) < 0 or max(heads, max_len) > _U32_MAX:
            raise ValueError("heads and max_len: from 0 to 2^32 - 1")
        n = self.lib.chpe_paged_attention_workspace(self._c, heads, max_len, int(weights))
        if n == 0 and self.rows:
            raise ValueError("chpe_paged_attention_workspace rejected the arguments")
        return n

    def attention(self, q, lens, max_len, scale=None, window=0, out=None, weight_in=None, weight_out=None,
                  workspace=None):
        """chpe_paged_attention: q [rows, heads, head_dim] f32 over the first lens[r] <= max_len slots of row r.
        weight_out [rows, kv_heads, >= max_len] receives weight_in (or 0) plus what each slot was given."""
        f32 = self._f32
        if q.dim() != 3:
            raise ValueError("q: [rows, heads, head_dim]")
        if min(max_len, window) < 0 or max(max_len, window) > _U32_MAX:
            raise ValueError("max_len and window: from 0 to 2^32 - 1")
        heads, width = q.shape[1], q.shape[1] * self.head_dim
        qp = self._take(q, "q", f32, (self.rows, heads, self.head_dim))
        if out is None:
            out = self._torch.empty(q.shape, dtype=f32, device=self.device)
        op = self._take(out, "out", f32, q.shape)
        wi = wo = None
        stride = 0
        if weight_out is not None:
            wo, stride = self._slots(weight_out, "weight_out", f32, max_len), weight_out.shape[2]
        if weight_in is not None:
            if weight_out is None:
                raise ValueError("weight_in without weight_out")
            wi = self._take(weight_in, "weight_in", f32, weight_out.shape)
        if workspace is None:
            workspace = self._torch.empty(self.attention_workspace(heads, max_len, wo is not None),
                                          dtype=self._torch.uint8, device=self.device)
        lp = self._take(lens, "lens", self._i32, (self.rows,))
        ws = self._take(workspace, "workspace", self._torch.uint8, (workspace.numel(),))
        self._call("chpe_paged_attention", heads, lp, max_len, qp, width,
                   1.0 / self.head_dim ** 0.5 if scale is None else scale, window, op, width, wi, wo, stride, ws,
                   workspace.numel())
        return out

    def evict_workspace(self, max_len):
        """Bytes that evict() needs."""
        if max_len < 0 or max_len > _U32_MAX:
            raise ValueError("max_len: from 0 to 2^32 - 1")
        n = self.lib.chpe_paged_evict_workspace(self._c, max_len)
        if n == 0 and self.rows:
            raise ValueError("chpe_paged_evict_workspace rejected the arguments")
        return n

    def evict(self, lens, max_len, budget, slot_weight, slot_pos, recent=0, sinks=0, lens_out=None, weight_out=None,
              pos_out=None, slot_src=None, workspace=None):
        """chpe_paged_evict: every row and kv head down to `budget` slots.  lens_out, weight_out and pos_out
        default to the inputs themselves; returns lens_out."""
        f32, i32 = self._f32, self._i32
        if min(max_len, budget, recent, sinks) < 0 or max(max_len, budget, recent, sinks) > _U32_MAX:
            raise ValueError("max_len, budget, recent and sinks: from 0 to 2^32 - 1")
        lens_out, weight_out, pos_out = (i if o is None else o for o, i in
                                         ((lens_out, lens), (weight_out, slot_weight), (pos_out, slot_pos)))
        w = self._slots(slot_weight, "slot_weight", f32, max_len)
        shape = slot_weight.shape
        args = [self._take(slot_pos, "slot_pos", i32, shape), shape[2], self._take(lens_out, "lens_out", i32, (self.rows,)),
                self._take(weight_out, "weight_out", f32, shape), self._take(pos_out, "pos_out", i32, shape),
                None if slot_src is None else self._take(slot_src, "slot_src", i32, shape)]
        if workspace is None:
            workspace = self._torch.empty(self.evict_workspace(max_len), dtype=self._torch.uint8, device=self.device)
        ws = self._take(workspace, "workspace", self._torch.uint8, (workspace.numel(),))
        self._call("chpe_paged_evict", self._take(lens, "lens", i32, (self.rows,)), max_len, budget, recent, sinks, w,
                   *args, ws, workspace.numel())
        return lens_out


def gpu_flat_tile_weights(cell):
    cell = np.ascontiguousarray(cell, dtype=np.uint8)
    out = np.empty(32768, dtype=np.float32)
    rc = load_engine_lib().chpe_debug_flat_tile_weights(cell.ctypes.data_as(_c_u8_p), _fp(out))
    if rc:
        raise EngineError(f"chpe_debug_flat_tile_weights failed: {rc}")
    return out


GEMV_MODES = {"store": 0, "accum": 1, "swiglu": 2, "logits": 3}


def gpu_gemv_flat(mode, rows, cols, tiles, x, tiles_up=None, gamma=None, eps=1e-6, y=None):
    """One flat-tile GEMV through the decode step's kernels (chpe_debug_gemv_flat).  `tiles`
    (and `tiles_up` for "swiglu") are consecutive 17408-byte cells; returns y, or for "logits"
    (y, argmax, hidden_norm)."""
    m = GEMV_MODES[mode]
    tiles = np.ascontiguousarray(tiles, dtype=np.uint8).reshape(-1)
    n_tiles = tiles.size // 17408
    up = None if tiles_up is None else np.ascontiguousarray(tiles_up, dtype=np.uint8).reshape(-1)
    x = np.ascontiguousarray(x, dtype=np.float32)
    g = None if gamma is None else np.ascontiguousarray(gamma, dtype=np.float32)
    out = np.zeros(rows, np.float32) if y is None else np.array(y, dtype=np.float32)
    am, hn = ctypes.c_uint32(0), ctypes.c_float(0.0)
    rc = load_engine_lib().chpe_debug_gemv_flat(
        m, rows, cols, tiles.ctypes.data_as(_c_u8_p), None if up is None else up.ctypes.data_as(_c_u8_p),
        n_tiles, _fp(x), None if g is None else _fp(g), eps, _fp(out), ctypes.byref(am), ctypes.byref(hn))
    if rc:
        raise EngineError(f"chpe_debug_gemv_flat failed: {rc} {load_engine_lib().chpe_last_error().decode()}")
    return (out, am.value, hn.value) if mode == "logits" else out


def gpu_gemv_cells(mode, rows, cells, x, cells_up=None, gamma=None, eps=1e-6, y=None):
    """One 16-row-cell GEMV at 2048 columns through the decode step's kernels
    (chpe_debug_gemv_cells); returns y, or for "logits" (y, argmax, hidden_norm)."""
    m = GEMV_MODES[mode]
    cells = np.ascontiguousarray(cells, dtype=np.uint8).reshape(-1)
    up = None if cells_up is None else np.ascontiguousarray(cells_up, dtype=np.uint8).reshape(-1)
    x = np.ascontiguousarray(x, dtype=np.float32)
    g = None if gamma is None else np.ascontiguousarray(gamma, dtype=np.float32)
    out = np.zeros(rows, np.float32) if y is None else np.array(y, dtype=np.float32)
    am, hn = ctypes.c_uint32(0), ctypes.c_float(0.0)
    rc = load_engine_lib().chpe_debug_gemv_cells(
        m, rows, cells.ctypes.data_as(_c_u8_p), None if up is None else up.ctypes.data_as(_c_u8_p),
        cells.size // 17408, _fp(x), None if g is None else _fp(g), eps, _fp(out), ctypes.byref(am), ctypes.byref(hn))
    if rc:
        raise EngineError(f"chpe_debug_gemv_cells failed: {rc} {load_engine_lib().chpe_last_error().decode()}")
    return (out, am.value, hn.value) if mode == "logits" else out


def gpu_gemv_poly(mode, rows, cols, cells, x, cells_up=None, gamma=None, eps=1e-6, y=None):
    """One GEMV over polymorphic 16-row cells of any width through the engine's polymorphic
    path (chpe_debug_gemv_poly); returns y, or for "logits" (y, argmax, hidden_norm)."""
    m = GEMV_MODES[mode]
    cells = np.ascontiguousarray(cells, dtype=np.uint8).reshape(-1)
    up = None if cells_up is None else np.ascontiguousarray(cells_up, dtype=np.uint8).reshape(-1)
    x = np.ascontiguousarray(x, dtype=np.float32)
    g = None if gamma is None else np.ascontiguousarray(gamma, dtype=np.float32)
    out = np.zeros(rows, np.float32) if y is None else np.array(y, dtype=np.float32)
    am, hn = ctypes.c_uint32(0), ctypes.c_float(0.0)
    rc = load_engine_lib().chpe_debug_gemv_poly(
        m, rows, cols, cells.ctypes.data_as(_c_u8_p), None if up is None else up.ctypes.data_as(_c_u8_p),
        cells.size // 17408, _fp(x), None if g is None else _fp(g), eps, _fp(out), ctypes.byref(am), ctypes.byref(hn))
    if rc:
        raise EngineError(f"chpe_debug_gemv_poly failed: {rc} {load_engine_lib().chpe_last_error().decode()}")
    return (out, am.value, hn.value) if mode == "logits" else out


RAW_KINDS = {"fp16": 0, "bf16": 1, "int8": 2}


def gpu_gemv_raw(mode, rows, cols, kind, tiles, x, tiles_up=None, gamma=None, eps=1e-6, y=None):
    """One GEMV over raw 16384-byte tiles (one row-major matrix) through the engine's raw
    kernels (chpe_debug_gemv_raw); returns y, or for "logits" (y, argmax, hidden_norm)."""
    m = GEMV_MODES[mode]
    t = np.ascontiguousarray(tiles, dtype=np.uint8).reshape(-1)
    up = None if tiles_up is None else np.ascontiguousarray(tiles_up, dtype=np.uint8).reshape(-1)
    x = np.ascontiguousarray(x, dtype=np.float32)
    g = None if gamma is None else np.ascontiguousarray(gamma, dtype=np.float32)
    out = np.zeros(rows, np.float32) if y is None else np.array(y, dtype=np.float32)
    am, hn = ctypes.c_uint32(0), ctypes.c_float(0.0)
    rc = load_engine_lib().chpe_debug_gemv_raw(
        m, rows, cols, RAW_KINDS[kind], t.ctypes.data_as(_c_u8_p), None if up is None else up.ctypes.data_as(_c_u8_p),
        t.size // 16384, _fp(x), None if g is None else _fp(g), eps, _fp(out), ctypes.byref(am), ctypes.byref(hn))
    if rc:
        raise EngineError(f"chpe_debug_gemv_raw failed: {rc} {load_engine_lib().chpe_last_error().decode()}")
    return (out, am.value, hn.value) if mode == "logits" else out


def gpu_embed_row_cell(region, row, D, init=None):
    region = np.ascontiguousarray(region, dtype=np.uint8)
    out = np.array(init, dtype=np.float32) if init is not None else np.zeros(D, dtype=np.float32)
    rc = load_engine_lib().chpe_debug_embed_row_cell(region.ctypes.data_as(_c_u8_p), region.size, row, D, _fp(out))
    if rc < 0:
        raise EngineError(f"chpe_debug_embed_row_cell failed: {rc}")
    return rc, out


def gpu_attention(q, k_rows, v_rows, pos, heads, kv_heads, head_dim, kv_f16):
    """The decode step's attention kernels on caller rows (k_rows / v_rows: [pos+1][kv*hd] f32)."""
    q = np.ascontiguousarray(q, dtype=np.float32)
    k = np.ascontiguousarray(k_rows, dtype=np.float32)
    v = np.ascontiguousarray(v_rows, dtype=np.float32)
    if q.size != heads * head_dim or k.size != (pos + 1) * kv_heads * head_dim or v.size != k.size:
        raise ValueError("attention operand sizes do not match the shape")
    out = np.empty(heads * head_dim, dtype=np.float32)
    rc = load_engine_lib().chpe_debug_attention(head_dim, heads, kv_heads, int(kv_f16), pos, _fp(q), _fp(k),
                                                _fp(v), _fp(out))
    if rc:
        raise EngineError(f"chpe_debug_attention failed: {rc}")
    return out


def gpu_attention_block(q, k_rows, v_rows, pos, heads, kv_heads, head_dim, kv_f16):
    """The block step's attention kernels on caller rows: q [nq][heads*hd] at positions pos ..
    pos+nq-1, k_rows / v_rows [pos+nq][kv*hd] f32; returns [nq][heads*hd]."""
    q = np.ascontiguousarray(q, dtype=np.float32)
    k = np.ascontiguousarray(k_rows, dtype=np.float32)
    v = np.ascontiguousarray(v_rows, dtype=np.float32)
    nq = q.shape[0]
    if q.ndim != 2 or q.shape[1] != heads * head_dim or k.size != (pos + nq) * kv_heads * head_dim or v.size != k.size:
        raise ValueError("attention operand sizes do not match the shape")
    out = np.empty_like(q)
    rc = load_engine_lib().chpe_debug_attention_block(head_dim, heads, kv_heads, int(kv_f16), pos, nq, _fp(q),
                                                      _fp(k), _fp(v), _fp(out))
    if rc:
        raise EngineError(f"chpe_debug_attention_block failed: {rc}")
    return out


def _f32c(a):
    return np.ascontiguousarray(a, dtype=np.float32)


def gpu_deltanet_conv(x, w, state):
    """k_dn_conv on caller data; returns (out, new_state)."""
    x, w, st = _f32c(x), _f32c(w), _f32c(state).copy()
    ch, taps = w.shape
    out = np.empty(ch, dtype=np.float32)
    rc = load_engine_lib().chpe_debug_deltanet_conv(ch, taps, _fp(x), _fp(w), _fp(st), _fp(out))
    if rc:
        raise EngineError(f"chpe_debug_deltanet_conv failed: {rc}")
    return out, st


def gpu_deltanet_step(q, k, v, a, b, A_log, dt_bias, state, z=None, norm_w=None, eps=1e-6):
    """k_dn_step on caller data; returns (out, new_state)."""
    q, k, v, a, b, A_log, dt_bias = (_f32c(t) for t in (q, k, v, a, b, A_log, dt_bias))
    st = _f32c(state).copy()
    nk, hd = q.shape
    nv = v.shape[0]
    out = np.empty((nv, hd), dtype=np.float32)
    zz = _f32c(z) if z is not None else None
    ww = _f32c(norm_w) if norm_w is not None else None
    rc = load_engine_lib().chpe_debug_deltanet_step(nv, nk, hd, _fp(q), _fp(k), _fp(v), _fp(a), _fp(b), _fp(A_log),
                                                    _fp(dt_bias), _fp(zz) if zz is not None else None,
                                                    _fp(ww) if ww is not None else None, eps, _fp(st), _fp(out))
    if rc:
        raise EngineError(f"chpe_debug_deltanet_step failed: {rc}")
    return out, st


def build(jobs=8):
    """Compile libchpe.so, libchpe_pack.so and the CLIs in place (make)."""
    import subprocess
    subprocess.run(["make", "-C", str(PKG_DIR), f"-j{jobs}"], check=True)


def default_archive_dir():
    d = Path(os.environ.get("CHPE_ARCHIVE_DIR", "/tmp/chpe_archives"))
    d.mkdir(parents=True, exist_ok=True)
    return d


ARCHIVE_NAMES = {
    PACK_3B_FP16_RAW: "qwen2.5-3b-fp16raw", PACK_3B_BF16_RAW: "qwen2.5-3b-bf16raw",
    PACK_3B_W4: "qwen2.5-3b-w4", PACK_3B_W2: "qwen2.5-3b-w2", PACK_3B_W4_STD: "qwen2.5-3b-w4std",
    PACK_72B_W4: "qwen2.5-72b-w4", PACK_72B_W2: "qwen2.5-72b-w2", PACK_9B_W4: "qwen3.5-9b-w4",
}


def _generator_tag():
    import hashlib
    h = hashlib.sha1()
    for f in ("csrc/pack.cpp", "csrc/format.hpp", "csrc/tensor_maps.hpp"):
        h.update((PKG_DIR / f).read_bytes())
    # letters only: chpe_init guesses the architecture from "9b" / "72b" in the path
    return "".join(chr(ord("a") + int(c, 16)) for c in h.hexdigest()[:10])


def ensure_archive(kind, seed=0, directory=None, threads=0):
    """Path of the seeded archive `kind` under `directory` (default $CHPE_ARCHIVE_DIR or
    /tmp/chpe_archives), written on first use and reused while the generator is unchanged."""
    d = Path(directory) if directory else default_archive_dir()
    path = d / f"{ARCHIVE_NAMES[kind]}-s{seed}-{_generator_tag()}.chpe"
    if not path.exists() or path.stat().st_size != archive_size(kind):
        tmp = path.with_suffix(".tmp")
        # the writer fills a memory-mapped file: on a file system without room for it the
        # process would die of SIGBUS mid-write, so the room is checked first
        d.mkdir(parents=True, exist_ok=True)
        tmp.unlink(missing_ok=True)  # (a write that did not finish)
        have = shutil.disk_usage(d).free
        if have < archive_size(kind):
            raise OSError(f"{d}: {have / 1e9:.1f} GB free, {ARCHIVE_NAMES[kind]} needs {archive_size(kind) / 1e9:.1f} GB "
                          "(remove older archives there or set CHPE_ARCHIVE_DIR)")
        write_archive(tmp, kind, seed, threads)
        os.replace(tmp, path)
    return path
