"""forgegpu -- Python binding of the B200 engine's C ABI (include/forgegpu.h).

The classes mirror the reference crate's Rust API (HueCodes/forge-db) so that
code written against it reads the same:

    IVFPQIndex.build(vectors, n_clusters, n_subvectors, metric)   ivf_pq.rs:374
    index.set_nprobe(n); index.search(q, k); index.batch_search(Q, k)
    BruteForceIndex(metric).add(...); .search(q, k); .batch_search(Q, k)
    KMeans(k, max_iters).fit(data)                                   kmeans.rs:33-193
    ProductQuantizer.train(x, m) / .encode(x) / .build_lookup_table_flat(q)

Every call runs on the GPU through libforgegpu.so.  There is no CPU fallback:
if the library is missing or no B200 is visible, calls raise ForgeGpuError.
"""
from __future__ import annotations

import array
import collections
import ctypes as C
import itertools
import os
import threading

import numpy as np

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "libforgegpu.so")

OK = 0
ERRORS = {
    -1: "InvalidParameter", -2: "DimensionMismatch", -3: "EmptyTrainingSet",
    -4: "DimensionNotDivisible", -5: "InsufficientVectors", -6: "Timeout", -7: "Cuda",
    -8: "Nccl", -9: "MemoryLimitExceeded", -10: "EmptyVectorSet", -11: "NotSupported",
    -12: "Io", -13: "SerializationError", -14: "ChecksumMismatch", -15: "InvalidFormat",
    -16: "InsufficientDiskSpace",
}


class IndexType:
    """src/persistence/format.rs:12-23"""
    IvfPq = 1
    Hnsw = 2
    Ivf = 3
    BruteForce = 4


class DistanceMetric:
    """src/distance/mod.rs:16-33"""
    Euclidean = 0
    EuclideanSquared = 1
    Cosine = 2
    DotProduct = 3
    Manhattan = 4


class ForgeGpuError(RuntimeError):
    def __init__(self, code: int, msg: str):
        super().__init__(f"{ERRORS.get(code, code)}: {msg}")
        self.code = code
        self.kind = ERRORS.get(code, str(code))


class Stats(C.Structure):
    _fields_ = [("lists_probed", C.c_uint64), ("codes_scanned", C.c_uint64),
                ("bytes_scanned", C.c_uint64), ("coarse_ms", C.c_double),
                ("scan_ms", C.c_double), ("rescore_ms", C.c_double), ("merge_ms", C.c_double),
                ("total_ms", C.c_double), ("exact_rescans", C.c_uint64),
                ("kernel_ms", C.c_double), ("kernel_scores", C.c_uint64),
                ("extended", C.c_uint64), ("comm_ms", C.c_double * 4)]


class FileInfo(C.Structure):
    _fields_ = [("version", C.c_uint32), ("index_type", C.c_uint32), ("flags", C.c_uint32),
                ("checksum", C.c_uint32), ("n", C.c_uint64), ("dim", C.c_uint64),
                ("nlist", C.c_uint64), ("m", C.c_uint64), ("nprobe", C.c_uint64),
                ("metric", C.c_int32), ("has_rerank", C.c_int32), ("n_rerank", C.c_uint64),
                ("rerank_factor", C.c_uint64)]


class BuilderOpts(C.Structure):
    _fields_ = [("num_clusters", C.c_size_t), ("num_subvectors", C.c_size_t),
                ("metric", C.c_int), ("auto_tune", C.c_int), ("target_memory_mb", C.c_size_t),
                ("target_recall", C.c_float), ("nprobe", C.c_size_t),
                ("rerank_factor", C.c_size_t), ("enable_reranking", C.c_int)]


class TrainOpts(C.Structure):
    _fields_ = [("ivf_sample", C.c_size_t), ("pq_sample", C.c_size_t),
                ("ivf_iters", C.c_size_t), ("pq_iters", C.c_size_t),
                ("ivf_sample_idx", C.c_void_p), ("ivf_init_idx", C.c_void_p),
                ("ivf_kpp_u", C.c_void_p), ("pq_sample_idx", C.c_void_p),
                ("pq_init_idx", C.c_void_p), ("seed", C.c_uint64)]


class LogprobArgs(C.Structure):
    _fields_ = [("dtype", C.c_int), ("queries", C.c_void_p), ("nq", C.c_size_t),
                ("ld_queries", C.c_size_t), ("rows", C.c_void_p), ("n", C.c_size_t),
                ("ld_rows", C.c_size_t), ("dim", C.c_size_t), ("scale", C.c_float),
                ("targets", C.c_void_p), ("allowed", C.c_void_p), ("ld_allowed", C.c_size_t),
                ("k", C.c_size_t), ("logprob", C.c_void_p), ("lse", C.c_void_p),
                ("entropy", C.c_void_p), ("top_ids", C.c_void_p), ("top_logprobs", C.c_void_p),
                ("workspace", C.c_void_p), ("workspace_bytes", C.c_size_t),
                ("stream", C.c_void_p)]


class LogprobGradArgs(C.Structure):
    _fields_ = [("dtype", C.c_int), ("queries", C.c_void_p), ("nq", C.c_size_t),
                ("ld_queries", C.c_size_t), ("rows", C.c_void_p), ("n", C.c_size_t),
                ("ld_rows", C.c_size_t), ("dim", C.c_size_t), ("scale", C.c_float),
                ("targets", C.c_void_p), ("allowed", C.c_void_p), ("ld_allowed", C.c_size_t),
                ("lse", C.c_void_p), ("entropy", C.c_void_p), ("d_logprob", C.c_void_p),
                ("d_lse", C.c_void_p), ("d_entropy", C.c_void_p), ("d_queries", C.c_void_p),
                ("ld_d_queries", C.c_size_t), ("d_rows", C.c_void_p), ("ld_d_rows", C.c_size_t),
                ("workspace", C.c_void_p), ("workspace_bytes", C.c_size_t),
                ("stream", C.c_void_p)]


_TEACHER = [("teacher_ids", C.c_void_p), ("teacher_logits", C.c_void_p), ("k", C.c_size_t),
            ("ld_ids", C.c_size_t), ("ld_logits", C.c_size_t), ("teacher_scale", C.c_float),
            ("rest", C.c_int), ("allowed", C.c_void_p), ("ld_allowed", C.c_size_t)]


class DistillArgs(C.Structure):
    _fields_ = LogprobArgs._fields_[:9] + _TEACHER + [
        ("loss", C.c_void_p), ("lse", C.c_void_p), ("logprobs", C.c_void_p),
        ("rest_logprob", C.c_void_p), ("workspace", C.c_void_p), ("workspace_bytes", C.c_size_t),
        ("stream", C.c_void_p)]


class DistillGradArgs(C.Structure):
    _fields_ = LogprobArgs._fields_[:9] + _TEACHER + [
        ("lse", C.c_void_p), ("logprobs", C.c_void_p), ("rest_logprob", C.c_void_p),
        ("d_loss", C.c_void_p), ("d_queries", C.c_void_p), ("ld_d_queries", C.c_size_t),
        ("d_rows", C.c_void_p), ("ld_d_rows", C.c_size_t), ("workspace", C.c_void_p),
        ("workspace_bytes", C.c_size_t), ("stream", C.c_void_p)]


class BeamArgs(C.Structure):
    _fields_ = [("dtype", C.c_int), ("scores", C.c_void_p), ("groups", C.c_size_t),
                ("beams", C.c_size_t), ("n", C.c_size_t), ("ld_group", C.c_size_t),
                ("ld_beam", C.c_size_t), ("scale", C.c_float), ("normalise", C.c_int),
                ("ids", C.c_void_p), ("ld_ids", C.c_size_t), ("allowed", C.c_void_p),
                ("ld_allowed", C.c_size_t), ("beam_scores", C.c_void_p), ("ended", C.c_void_p),
                ("end_id", C.c_int64), ("width", C.c_size_t), ("out_scores", C.c_void_p),
                ("out_parents", C.c_void_p), ("out_ids", C.c_void_p), ("out_ended", C.c_void_p),
                ("workspace", C.c_void_p), ("workspace_bytes", C.c_size_t),
                ("stream", C.c_void_p)]


class ReorderOpts(C.Structure):
    _fields_ = [("parents", C.c_void_p), ("groups", C.c_size_t), ("beams", C.c_size_t),
                ("width", C.c_size_t), ("clear", C.c_int), ("stream", C.c_void_p)]


class AdamwTensor(C.Structure):
    _fields_ = [("param", C.c_void_p), ("grad", C.c_void_p), ("m", C.c_void_p),
                ("v", C.c_void_p), ("m_scale", C.c_void_p), ("v_scale", C.c_void_p),
                ("n", C.c_size_t)]


class AdamwOpts(C.Structure):
    _fields_ = [("param_dtype", C.c_int), ("grad_dtype", C.c_int), ("state_bits", C.c_int),
                ("seed", C.c_uint32), ("lr", C.c_double), ("beta1", C.c_double),
                ("beta2", C.c_double), ("eps", C.c_double), ("weight_decay", C.c_double),
                ("grad_scale", C.c_double), ("step", C.c_int64), ("d_lr", C.c_void_p),
                ("d_step", C.c_void_p), ("d_grad_scale", C.c_void_p), ("stream", C.c_void_p)]


_vp = C.c_void_p
_sz = C.c_size_t
_SIGS = {
    "fdb_logprobs_workspace": (C.c_int, [_vp, C.POINTER(LogprobArgs), C.POINTER(_sz)]),
    "fdb_logprobs": (C.c_int, [_vp, C.POINTER(LogprobArgs)]),
    "fdb_logprobs_backward_workspace": (C.c_int, [_vp, C.POINTER(LogprobGradArgs),
                                                  C.POINTER(_sz)]),
    "fdb_logprobs_backward": (C.c_int, [_vp, C.POINTER(LogprobGradArgs)]),
    "fdb_logprobs_status": (C.c_int, [_vp, _vp, _vp]),
    "fdb_distill_workspace": (C.c_int, [_vp, C.POINTER(DistillArgs), C.POINTER(_sz)]),
    "fdb_distill": (C.c_int, [_vp, C.POINTER(DistillArgs)]),
    "fdb_distill_backward_workspace": (C.c_int, [_vp, C.POINTER(DistillGradArgs),
                                                 C.POINTER(_sz)]),
    "fdb_distill_backward": (C.c_int, [_vp, C.POINTER(DistillGradArgs)]),
    "fdb_beam_select_workspace": (C.c_int, [_vp, C.POINTER(BeamArgs), C.POINTER(_sz)]),
    "fdb_beam_select": (C.c_int, [_vp, C.POINTER(BeamArgs)]),
    "fdb_beam_reorder": (C.c_int, [_vp, _vp, _sz, C.POINTER(ReorderOpts)]),
    "fdb_bf_logprobs": (C.c_int, [_vp, _vp, _sz, C.c_float, _vp, _sz, _vp, _vp, _vp, _vp, _vp]),
    "fdb_adamw_step": (C.c_int, [_vp, _vp, _sz, C.POINTER(AdamwOpts)]),
    "fdb_adamw_state_values": (C.c_int, [_vp, _vp, _vp, _vp, _vp, _sz, _vp, _vp, _vp]),
    "fdb_last_error": (C.c_char_p, []),
    "fdb_version": (C.c_int, []),
    "fdb_ctx_create": (C.c_int, [C.c_int, C.POINTER(_vp)]),
    "fdb_ctx_free": (C.c_int, [_vp]),
    "fdb_ctx_stream": (C.c_int, [_vp, C.POINTER(_vp)]),
    "fdb_nccl_unique_id": (C.c_int, [_vp]),
    "fdb_ctx_init_comm": (C.c_int, [_vp, C.c_int, C.c_int, _vp]),
    "fdb_ctx_init_comm_timeout": (C.c_int, [_vp, C.c_int, C.c_int, _vp, C.c_double]),
    "fdb_ctx_set_wait_limit": (C.c_int, [_vp, C.c_double]),
    "fdb_ctx_test_stall_scans": (C.c_int, [_vp, C.c_int]),
    "fdb_host_alloc": (C.c_int, [_sz, C.POINTER(_vp)]),
    "fdb_host_free": (C.c_int, [_vp]),
    "fdb_sample_indices": (C.c_int, [C.c_uint64, _sz, _sz, _vp]),
    "fdb_uniform_draws": (C.c_int, [C.c_uint64, _sz, _vp]),
    "fdb_pairwise_distance": (C.c_int, [_vp, C.c_int, _vp, _vp, _sz, _sz, _vp]),
    "fdb_kmeans_fit": (C.c_int, [_vp, _vp, _sz, _sz, _sz, _sz, _vp, _vp, C.c_uint64, _vp, _vp,
                                 C.POINTER(C.c_int)]),
    "fdb_assign": (C.c_int, [_vp, _vp, _sz, _vp, _sz, _sz, _vp]),
    "fdb_find_nearest_centroids": (C.c_int, [_vp, _vp, _sz, _sz, _vp, _sz, _vp]),
    "fdb_find_nearest_centroids_noalloc": (C.c_int, [_vp, _vp, _sz, _sz, _vp, _sz, _sz, _vp]),
    "fdb_pq_train": (C.c_int, [_vp, _vp, _sz, _sz, _sz, _sz, _vp, C.c_uint64, _vp, _vp]),
    "fdb_pq_encode": (C.c_int, [_vp, _vp, _sz, _sz, _vp, _sz, _vp]),
    "fdb_pq_lookup_tables": (C.c_int, [_vp, _vp, _sz, _sz, _vp, _sz, _vp]),
    "fdb_ivfpq_build": (C.c_int, [_vp, _vp, _vp, _sz, _sz, _sz, _sz, C.c_int,
                                  C.POINTER(TrainOpts), C.POINTER(_vp)]),
    "fdb_ivfpq_from_trained": (C.c_int, [_vp, _vp, _vp, _sz, _sz, _sz, _vp, _vp, _vp, C.c_int,
                                         C.POINTER(_vp)]),
    "fdb_ivfpq_export": (C.c_int, [_vp, _vp, _vp, _vp, _vp, _vp]),
    "fdb_ivfpq_shard": (C.c_int, [_vp, C.c_int, C.c_int]),
    "fdb_ivfpq_shard_plan": (C.c_int, [_vp, _sz, C.c_int, _vp]),
    "fdb_ivfpq_set_nprobe": (C.c_int, [_vp, _sz]),
    "fdb_ivfpq_set_scan_mode": (C.c_int, [_vp, C.c_int]),
    "fdb_ivfpq_set_graphs": (C.c_int, [_vp, C.c_int]),
    "fdb_ivfpq_set_pass1_quota": (C.c_int, [_vp, _sz, C.c_uint64]),
    "fdb_ivfpq_set_stage_timers": (C.c_int, [_vp, C.c_int]),
    "fdb_ivfpq_get_pass1_quota": (C.c_int, [_vp, _sz, C.POINTER(C.c_int64)]),
    "fdb_ivfpq_nprobe": (_sz, [_vp]),
    "fdb_ivfpq_len": (_sz, [_vp]),
    "fdb_ivfpq_n_partitions": (_sz, [_vp]),
    "fdb_ivfpq_dim": (_sz, [_vp]),
    "fdb_ivfpq_n_subvectors": (_sz, [_vp]),
    "fdb_ivfpq_search": (C.c_int, [_vp, _vp, _sz, _vp, _vp, C.POINTER(_sz)]),
    "fdb_ivfpq_batch_search": (C.c_int, [_vp, _vp, _sz, _sz, _vp, _vp, _vp, C.POINTER(Stats)]),
    "fdb_ivfpq_batch_search_device": (C.c_int, [_vp, _vp, _sz, _sz, _vp, _vp, _vp,
                                                C.POINTER(Stats)]),
    "fdb_ivfpq_search_with_timeout": (C.c_int, [_vp, _vp, _sz, C.c_double, _vp, _vp,
                                                C.POINTER(_sz), C.POINTER(C.c_double)]),
    "fdb_ivfpq_batch_search_with_timeout": (C.c_int, [_vp, _vp, _sz, _sz, C.c_double, _vp, _vp,
                                                      _vp, C.POINTER(C.c_double)]),
    "fdb_ivfpq_free": (C.c_int, [_vp]),
    "fdb_bf_create": (C.c_int, [_vp, C.c_int, _vp, _vp, _sz, _sz, C.POINTER(_vp)]),
    "fdb_bf_add": (C.c_int, [_vp, _vp, _vp, _sz, _sz]),
    "fdb_bf_shard": (C.c_int, [_vp, C.c_int, C.c_int]),
    "fdb_bf_set_scan_mode": (C.c_int, [_vp, C.c_int]),
    "fdb_bf_len": (_sz, [_vp]),
    "fdb_bf_dimension": (_sz, [_vp]),
    "fdb_bf_search": (C.c_int, [_vp, _vp, _sz, _vp, _vp, C.POINTER(_sz)]),
    "fdb_bf_batch_search": (C.c_int, [_vp, _vp, _sz, _sz, _vp, _vp, _vp, C.POINTER(Stats)]),
    "fdb_bf_batch_search_device": (C.c_int, [_vp, _vp, _sz, _sz, _vp, _vp, _vp,
                                             C.POINTER(Stats)]),
    "fdb_bf_free": (C.c_int, [_vp]),
    "fdb_bf_remove": (C.c_int, [_vp, C.c_uint64, C.POINTER(C.c_int)]),
    "fdb_ivfpq_enable_reranking": (C.c_int, [_vp, _vp, _vp, _sz, _sz, _sz]),
    "fdb_ivfpq_search_filtered": (C.c_int, [_vp, _vp, _sz, _vp, _sz, _vp, _vp, C.POINTER(_sz)]),
    "fdb_ivfpq_batch_search_filtered": (C.c_int, [_vp, _vp, _sz, _sz, _vp, _sz, _vp, _vp, _vp]),
    "fdb_ivfpq_batch_search_filtered_device": (C.c_int, [_vp, _vp, _sz, _sz, _vp, _sz, _vp, _vp,
                                                         _vp, C.POINTER(Stats)]),
    "fdb_ivfpq_insert_batch": (C.c_int, [_vp, _vp, _vp, _sz, _sz]),
    "fdb_ivfpq_delete": (C.c_int, [_vp, C.c_uint64, C.POINTER(C.c_int)]),
    "fdb_ivfpq_num_tombstones": (_sz, [_vp]),
    "fdb_ivfpq_len_with_tombstones": (_sz, [_vp]),
    "fdb_ivfpq_fragmentation_ratio": (C.c_float, [_vp]),
    "fdb_ivfpq_compact": (C.c_int, [_vp]),
    "fdb_ivfpq_rebuild": (C.c_int, [_vp, C.POINTER(TrainOpts)]),
    "fdb_ivfpq_save": (C.c_int, [_vp, C.c_char_p]),
    "fdb_ivfpq_load": (C.c_int, [_vp, C.c_char_p, C.POINTER(_vp)]),
    "fdb_bf_save": (C.c_int, [_vp, C.c_char_p]),
    "fdb_bf_load": (C.c_int, [_vp, C.c_char_p, C.POINTER(_vp)]),
    "fdb_file_inspect": (C.c_int, [C.c_char_p, C.POINTER(FileInfo)]),
    "fdb_crc32": (C.c_uint32, [_vp, _sz]),
    "fdb_builder_defaults": (None, [C.POINTER(BuilderOpts)]),
    "fdb_builder_plan": (C.c_int, [C.POINTER(BuilderOpts), _sz, _sz, C.POINTER(_sz),
                                   C.POINTER(_sz), C.POINTER(_sz), C.POINTER(_sz)]),
    "fdb_builder_build": (C.c_int, [_vp, C.POINTER(BuilderOpts), _vp, _vp, _sz, _sz,
                                    C.POINTER(TrainOpts), C.POINTER(_vp)]),
}

_lib = None
_lock = threading.Lock()


def lib():
    """Load libforgegpu.so (raises if it was not built)."""
    global _lib
    with _lock:
        if _lib is None:
            if not os.path.exists(LIB_PATH):
                raise ForgeGpuError(-11, f"{LIB_PATH} is missing: build it with "
                                         "`python forge-db_b200/build.py`")
            L = C.CDLL(LIB_PATH)
            for name, (res, args) in _SIGS.items():
                fn = getattr(L, name)
                fn.restype = res
                fn.argtypes = args
            _lib = L
    return _lib


def exported_symbols():
    return list(_SIGS)


def _check(rc: int):
    if rc != OK:
        raise ForgeGpuError(rc, lib().fdb_last_error().decode(errors="replace"))


def _p(a):
    return None if a is None else C.c_void_p(a.ctypes.data)


def _f32(a):
    return np.ascontiguousarray(a, dtype=np.float32)


# ---------------------------------------------------------------------------
# context
# ---------------------------------------------------------------------------
class Context:
    """One device, one stream (and, for sharded indexes, one communicator)."""

    def __init__(self, device: int = 0):
        h = C.c_void_p()
        _check(lib().fdb_ctx_create(device, C.byref(h)))
        self.h = h
        self.device = device

    def stream(self) -> int:
        s = C.c_void_p()
        _check(lib().fdb_ctx_stream(self.h, C.byref(s)))
        return s.value or 0

    def init_comm(self, rank: int, world: int, nccl_id: bytes, timeout_s: float = 300.0):
        """The NCCL communicator of a sharded index; FDB_ERR_TIMEOUT (and no
        communicator) if not every rank joins within timeout_s."""
        buf = C.create_string_buffer(bytes(nccl_id), 128)
        _check(lib().fdb_ctx_init_comm_timeout(self.h, rank, world, buf, float(timeout_s)))

    def set_wait_limit(self, seconds: float):
        """Limit of each bounded wait inside the tensor-core kernels."""
        _check(lib().fdb_ctx_set_wait_limit(self.h, float(seconds)))

    def test_stall_scans(self, count: int):
        """Test hook: the next `count` list-scan launches issue no work, so
        their bounded waits run out (the call returns FDB_ERR_TIMEOUT)."""
        _check(lib().fdb_ctx_test_stall_scans(self.h, int(count)))

    def close(self):
        if self.h:
            _check(lib().fdb_ctx_free(self.h))
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def nccl_unique_id() -> bytes:
    buf = C.create_string_buffer(128)
    _check(lib().fdb_nccl_unique_id(buf))
    return buf.raw


_default_ctx = None


def default_context() -> Context:
    global _default_ctx
    if _default_ctx is None:
        _default_ctx = Context(0)
    return _default_ctx


def sample_indices(seed: int, n: int, take: int) -> np.ndarray:
    out = np.empty(take, np.uint32)
    _check(lib().fdb_sample_indices(seed, n, take, _p(out)))
    return out


def uniform_draws(seed: int, count: int) -> np.ndarray:
    out = np.empty(count, np.float32)
    _check(lib().fdb_uniform_draws(seed, count, _p(out)))
    return out


def crc32(data: bytes) -> int:
    """crc32fast::hash, the .fdb header's checksum (host only)."""
    buf = C.create_string_buffer(bytes(data), max(len(data), 1))
    return lib().fdb_crc32(buf, len(data))


def inspect_file(path) -> FileInfo:
    """Header and payload shape of a .fdb file (host only; checks what load does)."""
    info = FileInfo()
    _check(lib().fdb_file_inspect(os.fsencode(path), C.byref(info)))
    return info


def shard_plan(sizes, world: int) -> np.ndarray:
    sizes = np.ascontiguousarray(sizes, np.uint64)
    owner = np.empty(sizes.size, np.int32)
    _check(lib().fdb_ivfpq_shard_plan(_p(sizes), sizes.size, world, _p(owner)))
    return owner


def pairwise_distance(metric: int, a, b, ctx: Context | None = None) -> np.ndarray:
    ctx = ctx or default_context()
    a, b = _f32(a), _f32(b)
    out = np.empty(a.shape[0], np.float32)
    _check(lib().fdb_pairwise_distance(ctx.h, metric, _p(a), _p(b), a.shape[0], a.shape[1],
                                       _p(out)))
    return out


def assign(x, centroids, ctx: Context | None = None) -> np.ndarray:
    ctx = ctx or default_context()
    x, c = _f32(x), _f32(centroids)
    out = np.empty(x.shape[0], np.uint32)
    _check(lib().fdb_assign(ctx.h, _p(x), x.shape[0], _p(c), c.shape[0], x.shape[1], _p(out)))
    return out


# ---------------------------------------------------------------------------
# KMeans / ProductQuantizer
# ---------------------------------------------------------------------------
class KMeans:
    """KMeans::new(k, max_iters) (src/kmeans.rs:33-39)."""

    def __init__(self, k: int, max_iters: int, ctx: Context | None = None):
        self.k, self.max_iters = k, max_iters
        self.ctx = ctx or default_context()
        self.centroids = None
        self.iters = 0
        self.assignments = None

    def fit(self, data, init_idx=None, kpp_u=None, seed: int = 0):
        """fit / fit_raw (kmeans.rs:45-193); draws injected or from `seed`."""
        x = _f32(data)
        n, dim = x.shape
        cents = np.empty((self.k, dim), np.float32)
        assign_out = np.empty(n, np.uint32)
        it = C.c_int(0)
        ii = None if init_idx is None else np.ascontiguousarray(init_idx, np.uint32)
        uu = None if kpp_u is None else _f32(kpp_u)
        _check(lib().fdb_kmeans_fit(self.ctx.h, _p(x), n, dim, self.k, self.max_iters, _p(ii),
                                    _p(uu), seed, _p(cents), _p(assign_out), C.byref(it)))
        self.centroids, self.iters, self.assignments = cents, it.value, assign_out
        return self

    fit_raw = fit

    def find_nearest_centroids(self, query, k: int) -> np.ndarray:
        q = _f32(query)
        out = np.empty(min(k, self.k), np.uint32)
        _check(lib().fdb_find_nearest_centroids(self.ctx.h, _p(self.centroids), self.k,
                                                q.size, _p(q), k, _p(out)))
        return out


class ProductQuantizer:
    """ProductQuantizer (src/pq.rs:33-245)."""

    def __init__(self, codebooks, ctx: Context | None = None):
        self.codebooks = _f32(codebooks)
        self.n_subvectors, _, self.subvector_dim = self.codebooks.shape
        self.dim = self.n_subvectors * self.subvector_dim
        self.ctx = ctx or default_context()
        self.iters = None

    @classmethod
    def try_train(cls, vectors, n_subvectors: int, init_idx=None, seed: int = 0, iters: int = 25,
                  ctx: Context | None = None):
        ctx = ctx or default_context()
        x = _f32(vectors)
        n, dim = (x.shape if x.ndim == 2 else (0, 0))
        cb = np.empty((n_subvectors, 256, dim // max(n_subvectors, 1) if n_subvectors else 0),
                      np.float32)
        its = np.empty(max(n_subvectors, 1), np.int32)
        ii = None if init_idx is None else np.ascontiguousarray(init_idx, np.uint32)
        _check(lib().fdb_pq_train(ctx.h, _p(x) if n else None, n, dim, n_subvectors, iters,
                                  _p(ii), seed, _p(cb), _p(its)))
        pq = cls(cb, ctx)
        pq.iters = its
        return pq

    train = try_train

    def encode(self, vectors) -> np.ndarray:
        x = _f32(vectors)
        if x.ndim == 1:
            x = x[None]
        out = np.empty((x.shape[0], self.n_subvectors), np.uint8)
        _check(lib().fdb_pq_encode(self.ctx.h, _p(self.codebooks), self.n_subvectors, x.shape[1],
                                   _p(x), x.shape[0], _p(out)))
        return out

    def build_lookup_table_flat(self, queries) -> np.ndarray:
        q = _f32(queries)
        single = q.ndim == 1
        if single:
            q = q[None]
        out = np.empty((q.shape[0], self.n_subvectors * 256), np.float32)
        _check(lib().fdb_pq_lookup_tables(self.ctx.h, _p(self.codebooks), self.n_subvectors,
                                          q.shape[1], _p(q), q.shape[0], _p(out)))
        return out[0] if single else out


# ---------------------------------------------------------------------------
# indexes
# ---------------------------------------------------------------------------
def _train_opts(seed=0, ivf_sample=0, pq_sample=0, ivf_iters=0, pq_iters=0, ivf_sample_idx=None,
                ivf_init_idx=None, ivf_kpp_u=None, pq_sample_idx=None, pq_init_idx=None):
    keep = []

    def arr(a, dt):
        if a is None:
            return None
        a = np.ascontiguousarray(a, dt)
        keep.append(a)
        return a.ctypes.data

    o = TrainOpts(ivf_sample, pq_sample, ivf_iters, pq_iters,
                  arr(ivf_sample_idx, np.uint32), arr(ivf_init_idx, np.uint32),
                  arr(ivf_kpp_u, np.float32), arr(pq_sample_idx, np.uint32),
                  arr(pq_init_idx, np.uint32), seed)
    if ivf_sample_idx is not None:
        o.ivf_sample = len(ivf_sample_idx)
    if pq_sample_idx is not None:
        o.pq_sample = len(pq_sample_idx)
    return o, keep


def _results(ids, dists, counts):
    return [list(zip(ids[i, :counts[i]].tolist(), dists[i, :counts[i]].tolist()))
            for i in range(ids.shape[0])]


class IVFPQIndex:
    """IVFPQIndex (src/index/ivf_pq.rs:343-1084) on one B200."""

    def __init__(self, handle, ctx: Context):
        self.h = handle
        self.ctx = ctx

    @classmethod
    def build(cls, vectors, n_clusters: int, n_subvectors: int,
              metric: int = DistanceMetric.Euclidean, ids=None, ctx: Context | None = None,
              seed: int = 0, ivf_sample=0, pq_sample=0, ivf_iters=0, pq_iters=0,
              ivf_sample_idx=None, ivf_init_idx=None, ivf_kpp_u=None, pq_sample_idx=None,
              pq_init_idx=None):
        ctx = ctx or default_context()
        x = _f32(vectors)
        n, dim = x.shape
        o, keep = _train_opts(seed, ivf_sample, pq_sample, ivf_iters, pq_iters, ivf_sample_idx,
                              ivf_init_idx, ivf_kpp_u, pq_sample_idx, pq_init_idx)
        idv = None if ids is None else np.ascontiguousarray(ids, np.uint64)
        h = C.c_void_p()
        _check(lib().fdb_ivfpq_build(ctx.h, _p(x), _p(idv), n, dim, n_clusters, n_subvectors,
                                     metric, C.byref(o), C.byref(h)))
        return cls(h, ctx)

    @classmethod
    def from_trained(cls, centroids, codebooks, offsets, ids, codes,
                     metric: int = DistanceMetric.Euclidean, ctx: Context | None = None):
        ctx = ctx or default_context()
        cents = _f32(centroids)
        cb = _f32(codebooks)
        offs = np.ascontiguousarray(offsets, np.uint64)
        idv = np.ascontiguousarray(ids, np.uint64)
        codes = np.ascontiguousarray(codes, np.uint8)
        nlist, dim = cents.shape
        m = cb.shape[0]
        h = C.c_void_p()
        _check(lib().fdb_ivfpq_from_trained(ctx.h, _p(cents), _p(cb), nlist, m, dim, _p(offs),
                                            _p(idv), _p(codes), metric, C.byref(h)))
        return cls(h, ctx)

    def export(self):
        nlist, dim = self.n_partitions(), self.dim()
        offs = np.empty(nlist + 1, np.uint64)
        _check(lib().fdb_ivfpq_export(self.h, None, None, _p(offs), None, None))
        n = int(offs[-1])
        cents = np.empty((nlist, dim), np.float32)
        m = self.n_subvectors()
        cb = np.empty((m, 256, dim // m), np.float32)
        ids = np.empty(n, np.uint64)
        codes = np.empty((n, m), np.uint8)
        _check(lib().fdb_ivfpq_export(self.h, _p(cents), _p(cb), None, _p(ids), _p(codes)))
        return cents, cb, offs, ids, codes

    def shard(self, rank: int, world: int):
        _check(lib().fdb_ivfpq_shard(self.h, rank, world))

    SCAN_AUTO, SCAN_EXACT, SCAN_TABLES, SCAN_TENSOR = 0, 1, 2, 3

    def set_nprobe(self, nprobe: int):
        _check(lib().fdb_ivfpq_set_nprobe(self.h, nprobe))

    def set_scan_mode(self, mode: int):
        _check(lib().fdb_ivfpq_set_scan_mode(self.h, mode))

    def set_pass1_quota(self, nprobe: int, div: int):
        """The tensor path's pass-1 sampling quota (1/div of the probed codes,
        0: every probe's first tile) for batches with `nprobe` probes."""
        _check(lib().fdb_ivfpq_set_pass1_quota(self.h, int(nprobe), int(div)))

    def pass1_quota(self, nprobe: int):
        """The pass-1 quota in use for `nprobe` probes, None before the first
        large tensor-path batch calibrates it."""
        v = C.c_int64()
        _check(lib().fdb_ivfpq_get_pass1_quota(self.h, int(nprobe), C.byref(v)))
        return None if v.value < 0 else v.value

    def set_stage_timers(self, enable: bool):
        """Fill fdb_stats' stage times (on by default); off, statistics keep
        the counters and the list scan's pass-2 time only."""
        _check(lib().fdb_ivfpq_set_stage_timers(self.h, 1 if enable else 0))

    def set_graphs(self, enable: bool):
        """Replay repeated same-shape batch searches as CUDA graphs."""
        _check(lib().fdb_ivfpq_set_graphs(self.h, int(bool(enable))))

    def nprobe(self) -> int:
        return lib().fdb_ivfpq_nprobe(self.h)

    def len(self) -> int:
        return lib().fdb_ivfpq_len(self.h)

    __len__ = len

    def n_partitions(self) -> int:
        return lib().fdb_ivfpq_n_partitions(self.h)

    def dim(self) -> int:
        return lib().fdb_ivfpq_dim(self.h)

    def n_subvectors(self) -> int:
        return lib().fdb_ivfpq_n_subvectors(self.h)

    def search(self, query, k: int):
        q = _f32(query)
        ids = np.empty(max(k, 1), np.uint64)
        d = np.empty(max(k, 1), np.float32)
        n = C.c_size_t(0)
        _check(lib().fdb_ivfpq_search(self.h, _p(q), k, _p(ids), _p(d), C.byref(n)))
        return list(zip(ids[:n.value].tolist(), d[:n.value].tolist()))

    def batch_search_arrays(self, queries, k: int, stats: bool = False):
        Q = _f32(queries)
        nq = Q.shape[0] if Q.ndim == 2 else 0
        ids = np.empty((nq, k), np.uint64)
        d = np.empty((nq, k), np.float32)
        cnt = np.empty(nq, np.uint32)
        st = Stats()
        _check(lib().fdb_ivfpq_batch_search(self.h, _p(Q) if nq else None, nq, k, _p(ids), _p(d),
                                            _p(cnt), C.byref(st) if stats else None))
        return (ids, d, cnt, st) if stats else (ids, d, cnt)

    def batch_search(self, queries, k: int):
        ids, d, cnt = self.batch_search_arrays(queries, k)
        return _results(ids, d, cnt)

    batch_search_parallel = batch_search

    def search_with_timeout(self, query, k: int, timeout_s: float):
        """search_with_timeout (ivf_pq.rs:1369-1455): (results, elapsed
        seconds), or ForgeGpuError kind "Timeout" past the deadline."""
        q = _f32(query)
        ids = np.empty(max(k, 1), np.uint64)
        d = np.empty(max(k, 1), np.float32)
        n = C.c_size_t(0)
        el = C.c_double(0.0)
        _check(lib().fdb_ivfpq_search_with_timeout(self.h, _p(q), k, float(timeout_s), _p(ids),
                                                   _p(d), C.byref(n), C.byref(el)))
        return list(zip(ids[:n.value].tolist(), d[:n.value].tolist())), el.value

    def batch_search_with_timeout_arrays(self, queries, k: int, timeout_s: float):
        """batch_search under one deadline: (ids, dists, counts, elapsed)."""
        Q = _f32(queries)
        nq = Q.shape[0]
        ids = np.empty((nq, k), np.uint64)
        d = np.empty((nq, k), np.float32)
        cnt = np.empty(nq, np.uint32)
        el = C.c_double(0.0)
        _check(lib().fdb_ivfpq_batch_search_with_timeout(self.h, _p(Q), nq, k, float(timeout_s),
                                                         _p(ids), _p(d), _p(cnt),
                                                         C.byref(el)))
        return ids, d, cnt, el.value

    # --- re-ranking, filters, updates (ivf_pq.rs:513-831, 1731-1890) ---
    def enable_reranking(self, vectors, ids, rerank_factor: int):
        x = _f32(vectors)
        idv = np.ascontiguousarray(ids, np.uint64)
        n = x.shape[0] if x.ndim == 2 else 0
        _check(lib().fdb_ivfpq_enable_reranking(self.h, _p(x) if n else None,
                                                _p(idv) if n else None, n,
                                                x.shape[1] if n else self.dim(), rerank_factor))

    def search_filtered(self, query, k: int, allowed_ids):
        """search_filtered with the matching ids of the metadata filter."""
        q = _f32(query)
        al = np.ascontiguousarray(allowed_ids, np.uint64)
        ids = np.empty(max(k, 1), np.uint64)
        d = np.empty(max(k, 1), np.float32)
        n = C.c_size_t(0)
        _check(lib().fdb_ivfpq_search_filtered(self.h, _p(q), k, _p(al) if al.size else None,
                                               al.size, _p(ids), _p(d), C.byref(n)))
        return list(zip(ids[:n.value].tolist(), d[:n.value].tolist()))

    def batch_search_filtered_arrays(self, queries, k: int, allowed_ids):
        Q = _f32(queries)
        nq = Q.shape[0]
        al = np.ascontiguousarray(allowed_ids, np.uint64)
        ids = np.empty((nq, k), np.uint64)
        d = np.empty((nq, k), np.float32)
        cnt = np.empty(nq, np.uint32)
        _check(lib().fdb_ivfpq_batch_search_filtered(self.h, _p(Q), nq, k,
                                                     _p(al) if al.size else None, al.size,
                                                     _p(ids), _p(d), _p(cnt)))
        return ids, d, cnt

    def insert_batch(self, vectors, ids):
        x = _f32(vectors)
        if x.ndim == 1:
            x = x[None]
        idv = np.ascontiguousarray(np.atleast_1d(ids), np.uint64)
        _check(lib().fdb_ivfpq_insert_batch(self.h, _p(x), _p(idv), x.shape[0], x.shape[1]))

    def delete(self, id_: int) -> bool:
        out = C.c_int(0)
        _check(lib().fdb_ivfpq_delete(self.h, int(id_), C.byref(out)))
        return bool(out.value)

    def num_tombstones(self) -> int:
        return lib().fdb_ivfpq_num_tombstones(self.h)

    def len_with_tombstones(self) -> int:
        return lib().fdb_ivfpq_len_with_tombstones(self.h)

    def fragmentation_ratio(self) -> float:
        return lib().fdb_ivfpq_fragmentation_ratio(self.h)

    def is_empty(self) -> bool:
        return self.len() == 0

    def compact(self):
        _check(lib().fdb_ivfpq_compact(self.h))

    def rebuild(self, seed: int = 0, **draws):
        o, keep = _train_opts(seed, **draws)
        _check(lib().fdb_ivfpq_rebuild(self.h, C.byref(o)))

    # --- Persistable (src/persistence/mod.rs:34-73) ---
    def save(self, path):
        _check(lib().fdb_ivfpq_save(self.h, os.fsencode(path)))

    @classmethod
    def load(cls, path, ctx: Context | None = None):
        ctx = ctx or default_context()
        h = C.c_void_p()
        _check(lib().fdb_ivfpq_load(ctx.h, os.fsencode(path), C.byref(h)))
        return cls(h, ctx)

    load_mmap = load

    def close(self):
        if self.h:
            _check(lib().fdb_ivfpq_free(self.h))
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class IVFPQIndexBuilder:
    """IVFPQIndexBuilder (src/index/ivf_pq_builder.rs:56-331): fluent setters,
    auto-tuned parameters, build() on the GPU."""

    def __init__(self):
        self.o = BuilderOpts()
        lib().fdb_builder_defaults(C.byref(self.o))
        self._vectors = None
        self._ids = None

    def vectors(self, vectors, ids=None):
        self._vectors = _f32(vectors)
        self._ids = None if ids is None else np.ascontiguousarray(ids, np.uint64)
        return self

    def num_clusters(self, n):
        self.o.num_clusters = n
        return self

    def num_subvectors(self, m):
        self.o.num_subvectors = m
        return self

    def metric(self, metric):
        self.o.metric = metric
        return self

    def auto_tune(self, enable: bool):
        self.o.auto_tune = int(bool(enable))
        return self

    def target_memory_mb(self, mb):
        self.o.target_memory_mb = mb
        return self

    def target_recall(self, recall):
        self.o.target_recall = min(max(float(recall), 0.0), 1.0)
        return self

    def nprobe(self, nprobe):
        self.o.nprobe = nprobe
        return self

    def rerank_factor(self, factor):
        self.o.rerank_factor = max(int(factor), 1)
        return self

    def enable_reranking(self, enable: bool):
        self.o.enable_reranking = int(bool(enable))
        return self

    def plan(self, n: int, dim: int):
        """(num_clusters, num_subvectors, nprobe, estimated MiB) for n x dim."""
        c, m, p, mb = C.c_size_t(), C.c_size_t(), C.c_size_t(), C.c_size_t()
        _check(lib().fdb_builder_plan(C.byref(self.o), n, dim, C.byref(c), C.byref(m),
                                      C.byref(p), C.byref(mb)))
        return c.value, m.value, p.value, mb.value

    def build(self, ctx: Context | None = None, seed: int = 0, **draws) -> IVFPQIndex:
        x = self._vectors
        n = 0 if x is None else (x.shape[0] if x.ndim == 2 else 0)
        dim = 0 if n == 0 else x.shape[1]
        # the argument checks come before any device work (no context needed)
        ctx = ctx or (default_context() if n else None)
        t, keep = _train_opts(seed, **draws)
        h = C.c_void_p()
        _check(lib().fdb_builder_build(ctx.h if ctx else None, C.byref(self.o),
                                       None if x is None else (_p(x) if n else C.c_void_p(1)),
                                       _p(self._ids), n, dim, C.byref(t), C.byref(h)))
        return IVFPQIndex(h, ctx)


class BruteForceIndex:
    """BruteForceIndex (src/index/brute_force.rs:60-225) on one B200."""

    def __init__(self, metric: int = DistanceMetric.Euclidean, ctx: Context | None = None):
        self.ctx = ctx or default_context()
        h = C.c_void_p()
        _check(lib().fdb_bf_create(self.ctx.h, metric, None, None, 0, 0, C.byref(h)))
        self.h = h
        self.metric = metric

    def add(self, vectors, ids=None):
        x = _f32(vectors)
        if x.ndim == 1:
            x = x[None]
        idv = None if ids is None else np.ascontiguousarray(np.atleast_1d(ids), np.uint64)
        _check(lib().fdb_bf_add(self.h, _p(x), _p(idv), x.shape[0], x.shape[1]))
        return self

    def shard(self, rank: int, world: int):
        _check(lib().fdb_bf_shard(self.h, rank, world))

    def set_scan_mode(self, mode: int):
        _check(lib().fdb_bf_set_scan_mode(self.h, mode))

    def len(self) -> int:
        return lib().fdb_bf_len(self.h)

    __len__ = len

    def dimension(self) -> int:
        return lib().fdb_bf_dimension(self.h)

    def search(self, query, k: int):
        q = _f32(query)
        ids = np.empty(max(k, 1), np.uint64)
        d = np.empty(max(k, 1), np.float32)
        n = C.c_size_t(0)
        _check(lib().fdb_bf_search(self.h, _p(q), k, _p(ids), _p(d), C.byref(n)))
        return list(zip(ids[:n.value].tolist(), d[:n.value].tolist()))

    search_parallel = search

    def batch_search_arrays(self, queries, k: int, stats: bool = False):
        Q = _f32(queries)
        nq = Q.shape[0]
        ids = np.empty((nq, k), np.uint64)
        d = np.empty((nq, k), np.float32)
        cnt = np.empty(nq, np.uint32)
        st = Stats()
        _check(lib().fdb_bf_batch_search(self.h, _p(Q), nq, k, _p(ids), _p(d), _p(cnt),
                                         C.byref(st) if stats else None))
        return (ids, d, cnt, st) if stats else (ids, d, cnt)

    def batch_search(self, queries, k: int):
        ids, d, cnt = self.batch_search_arrays(queries, k)
        return _results(ids, d, cnt)

    def log_probs(self, queries, target_ids=None, temperature: float = 1.0, k: int = 0):
        """What the dot products are as probabilities over all vectors,
        p(x | q) proportional to exp(q . x / temperature): a LogProbs of
        arrays, with the log probability of target_ids[i] under query i (0
        for an id the index does not hold), and the k most probable ids."""
        Q = _f32(queries)
        nq = Q.shape[0]
        if Q.ndim != 2 or (self.len() and Q.shape[1] != self.dimension()):
            raise ForgeGpuError(-2, f"queries of shape {Q.shape} on an index of dimension "
                                    f"{self.dimension()}")
        t = None if target_ids is None else np.ascontiguousarray(target_ids, np.uint64)
        if t is not None and t.shape != (nq,):
            raise ForgeGpuError(-2, f"{t.shape} target ids for {nq} queries")
        lp, lse, ent = (np.empty(nq, np.float32) for _ in range(3))
        ids, tlp = np.empty((nq, k), np.uint64), np.empty((nq, k), np.float32)
        _check(lib().fdb_bf_logprobs(self.h, _p(Q), nq, float(temperature), _p(t), k, _p(lp),
                                     _p(lse), _p(ent), _p(ids), _p(tlp)))
        return LogProbs(lp, lse, ent, ids, tlp)

    def remove(self, id_: int) -> bool:
        out = C.c_int(0)
        _check(lib().fdb_bf_remove(self.h, int(id_), C.byref(out)))
        return bool(out.value)

    def is_empty(self) -> bool:
        return self.len() == 0

    def save(self, path):
        _check(lib().fdb_bf_save(self.h, os.fsencode(path)))

    @classmethod
    def load(cls, path, ctx: Context | None = None):
        ctx = ctx or default_context()
        self = cls.__new__(cls)
        self.ctx = ctx
        h = C.c_void_p()
        _check(lib().fdb_bf_load(ctx.h, os.fsencode(path), C.byref(h)))
        self.h = h
        self.metric = inspect_file(path).metric
        return self

    def close(self):
        if self.h:
            _check(lib().fdb_bf_free(self.h))
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


# ---------------------------------------------------------------------------
# device operators on torch tensors: softmax over rows, beams, AdamW
# ---------------------------------------------------------------------------
LogProbs = collections.namedtuple("LogProbs", "logprob lse entropy top_ids top_logprobs")
Distilled = collections.namedtuple("Distilled", "loss lse logprobs rest")
Beams = collections.namedtuple("Beams", "scores parents ids ended")
_device_ctx: dict = {}
_DTYPE: dict = {}


def _torch():
    import torch
    if not _DTYPE:
        _DTYPE.update({torch.float32: 0, torch.float16: 1, torch.bfloat16: 2})
    return torch


def _ctx_of(device) -> Context:
    """The context of a tensor's device (made once per device)."""
    i = device.index
    c = _device_ctx.get(i)
    if c is None:
        c = default_context() if i == 0 else Context(i)
        with _lock:
            c = _device_ctx.setdefault(i, c)
    return c


def _refuse(msg: str):
    raise ForgeGpuError(-1, msg)


def _matrix(t, what: str, like=None):
    """(pointer, rows, row distance) of a 2-d tensor whose rows are contiguous."""
    shape, stride = t.shape, t.stride()
    if len(shape) != 2 or not t.is_cuda or t.dtype not in _DTYPE:
        _refuse(f"{what} must be a 2-d float32, float16 or bfloat16 tensor on a GPU")
    n, d = shape
    s0, s1 = stride
    if (s1 != 1 and d > 1) or (n > 1 and s0 < d):
        _refuse(f"{what} must have contiguous rows")
    if like is not None and (t.dtype != like.dtype or t.device != like.device):
        _refuse(f"{what} must have the queries' type and device")
    return t.data_ptr(), n, s0 if n > 1 and s0 > d else d


def _vector(t, n: int, dtype, device, what: str):
    if t is None:
        return None
    if t.dtype != dtype or t.device != device or t.shape != (n,) or not t.is_contiguous():
        _refuse(f"{what} must be a contiguous {dtype} tensor of {n} values on the queries' device")
    return t.data_ptr()


def _softmax_args(q, x, targets, scale, allowed):
    """The fields that both argument structures start with."""
    torch = _torch()
    qp, nq, ldq = _matrix(q, "queries")
    xp, n, ldx = _matrix(x, "rows", q)
    dim, dev = q.shape[1], q.device
    if x.shape[1] != dim:
        raise ForgeGpuError(-2, f"queries of {dim} and rows of {x.shape[1]} dimensions")
    ap, lda = None, 0
    if allowed is not None:
        words = (n + 31) // 32
        if allowed.dtype != torch.int32 or allowed.device != dev or allowed.dim() not in (1, 2) \
                or allowed.shape[-1] != words or (words > 1 and allowed.stride(-1) != 1):
            _refuse(f"allowed must be int32 words [{words}] or [1 or nq, {words}] on the "
                    "queries' device")
        rows = 1 if allowed.dim() == 1 else allowed.shape[0]
        if rows not in (1, nq):
            _refuse(f"allowed has {rows} filters for {nq} queries")
        ap = allowed.data_ptr()
        if rows > 1:
            lda = allowed.stride(0)
            if lda < words:
                _refuse("allowed must have contiguous rows")
    return (_DTYPE[q.dtype], qp, nq, ldq, xp, n, ldx, dim, scale,
            _vector(targets, nq, torch.int64, dev, "targets"), ap, lda)


_ws_bytes: dict = {}


def _workspace(torch, ctx, fn, a, key, device, given):
    """(tensor, its bytes): the caller's workspace, or a new one of the size that
    the call needs (asked for once per shape)."""
    if given is not None:
        if given.dtype != torch.uint8 or given.device != device or not given.is_contiguous():
            _refuse("the workspace must be a contiguous uint8 tensor on the queries' device")
        return given, given.numel()
    need = _ws_bytes.get(key)
    if need is None:
        size = _sz()
        _check(fn(ctx.h, C.byref(a), C.byref(size)))
        if len(_ws_bytes) > 1024:
            _ws_bytes.clear()
        need = _ws_bytes[key] = size.value
    return torch.empty(need, dtype=torch.uint8, device=device), need


def logprobs(queries, rows, targets=None, *, scale: float = 1.0, allowed=None, k: int = 0,
             workspace=None) -> LogProbs:
    """Log probabilities under softmax(scale * queries @ rows.T), on the current
    stream, without the [nq, n] scores (fdb_logprobs in forgegpu.h).

    targets: int64 [nq], the row whose log probability is wanted (none where
    negative).  allowed: int32 words of a bit per row, one filter or one per
    query.  k: number of alternatives.  workspace: a uint8 tensor to use
    instead of a new one (logprobs_status reads a timeout from it).  The
    results have no autograd history, whatever the inputs require: the gradient
    is logprobs_backward's."""
    torch = _torch()
    head = _softmax_args(queries, rows, targets, scale, allowed)
    dev, nq = queries.device, head[2]
    ctx = _ctx_of(dev)
    L = lib()
    empty, f32 = torch.empty, torch.float32
    lp, lse, ent = (empty(nq, dtype=f32, device=dev), empty(nq, dtype=f32, device=dev),
                    empty(nq, dtype=f32, device=dev))
    ids = empty((nq, k), dtype=torch.int64, device=dev)
    top = empty((nq, k), dtype=f32, device=dev)
    a = LogprobArgs(*head, k, lp.data_ptr(), lse.data_ptr(), ent.data_ptr(), ids.data_ptr(),
                    top.data_ptr())
    # (whether the operands are copied depends on their alignment)
    key = (dev.index, k, head[1] & 15, head[4] & 15) + head[0:1] + head[2:4] + head[5:8]
    ws, a.workspace_bytes = _workspace(torch, ctx, L.fdb_logprobs_workspace, a, key, dev, workspace)
    a.workspace = ws.data_ptr()
    a.stream = torch._C._cuda_getCurrentRawStream(dev.index)
    rc = L.fdb_logprobs(ctx.h, C.byref(a))
    if rc:
        _check(rc)
    return LogProbs(lp, lse, ent, ids, top)


def logprobs_backward(queries, rows, targets, lse, entropy=None, *, d_logprob=None, d_lse=None,
                      d_entropy=None, scale: float = 1.0, allowed=None,
                      need_queries: bool = True, need_rows: bool = True, workspace=None):
    """(d_queries, d_rows) of a loss from its gradients with respect to what
    logprobs returned; lse and entropy are that call's (fdb_logprobs_backward
    in forgegpu.h).  A gradient that is not needed is None."""
    torch = _torch()
    head = _softmax_args(queries, rows, targets, scale, allowed)
    dev, f32 = queries.device, torch.float32
    nq, n, dim = head[2], head[5], head[7]
    ctx = _ctx_of(dev)
    L = lib()
    dq = torch.empty((nq, dim), dtype=queries.dtype, device=dev) if need_queries else None
    dx = torch.empty((n, dim), dtype=queries.dtype, device=dev) if need_rows else None
    a = LogprobGradArgs(*head, _vector(lse, nq, f32, dev, "lse"),
                        _vector(entropy, nq, f32, dev, "entropy"),
                        _vector(d_logprob, nq, f32, dev, "d_logprob"),
                        _vector(d_lse, nq, f32, dev, "d_lse"),
                        _vector(d_entropy, nq, f32, dev, "d_entropy"),
                        None if dq is None else dq.data_ptr(), dim,
                        None if dx is None else dx.data_ptr(), dim)
    key = (dev.index, allowed is not None and head[11]) + head[0:1] + head[2:4] + head[5:8]
    ws, a.workspace_bytes = _workspace(torch, ctx, L.fdb_logprobs_backward_workspace, a, key, dev,
                                       workspace)
    a.workspace = ws.data_ptr()
    a.stream = torch._C._cuda_getCurrentRawStream(dev.index)
    rc = L.fdb_logprobs_backward(ctx.h, C.byref(a))
    if rc:
        _check(rc)
    return dq, dx


def logprobs_status(workspace):
    """Raises Timeout if a kernel wait of the last call with this workspace
    ran out (waits for the current stream)."""
    torch = _torch()
    ctx = _ctx_of(workspace.device)
    _check(lib().fdb_logprobs_status(
        ctx.h, workspace.data_ptr(),
        torch._C._cuda_getCurrentRawStream(workspace.device.index)))


def _lists(t, nq: int, k: int, dtype, device, what: str):
    """(pointer, row distance) of a teacher's [nq, k] lists."""
    if t.dtype != dtype or t.device != device or t.shape != (nq, k) or \
            (k > 1 and t.stride(1) != 1) or (nq > 1 and t.stride(0) < k):
        _refuse(f"{what} must be {dtype} [{nq}, {k}] with contiguous rows on the queries' device")
    return t.data_ptr(), t.stride(0) if nq > 1 else k


def _distill_args(q, x, ids, logits, scale, teacher_scale, rest, allowed):
    """The fields that both argument structures start with."""
    torch = _torch()
    head = _softmax_args(q, x, None, scale, allowed)
    if ids.dim() != 2:
        _refuse("teacher_ids must be [nq, k]")
    nq, k = head[2], ids.shape[1]
    ip, ldi = _lists(ids, nq, k, torch.int64, q.device, "teacher_ids")
    zp, ldz = _lists(logits, nq, k, torch.float32, q.device, "teacher_logits")
    return head[:9] + (ip, zp, k, ldi, ldz, teacher_scale, rest) + head[10:]


def distill(queries, rows, teacher_ids, teacher_logits, *, scale: float = 1.0,
            teacher_scale: float = 1.0, rest: bool = False, allowed=None,
            workspace=None) -> Distilled:
    """The loss of a teacher's best rows under softmax(scale * queries @ rows.T),
    per query, on the current stream (fdb_distill in forgegpu.h).

    teacher_ids: int64 [nq, k], rows (none where negative), teacher_logits:
    float32 [nq, k].  With rest they are log probabilities, and what they leave
    is compared with the student's probability of all other rows; else the
    teacher is softmax(teacher_scale * teacher_logits) over its k rows.
    allowed, workspace: as for logprobs (logprobs_status reads a timeout).
    logprobs is the student's log probability of each entry, rest the log of
    what it leaves to other rows (None without).  The results have no autograd
    history: the gradient is distill_backward's."""
    torch = _torch()
    head = _distill_args(queries, rows, teacher_ids, teacher_logits, scale, teacher_scale,
                         1 if rest else 0, allowed)
    dev, nq, k = queries.device, head[2], head[11]
    ctx = _ctx_of(dev)
    L = lib()
    # (made like what is there: half the time of torch.empty)
    like = torch.empty_like
    loss = teacher_logits.new_empty(nq)
    lse, other = like(loss), like(loss) if rest else None
    lp = like(teacher_logits) if teacher_logits.is_contiguous() else teacher_logits.new_empty((nq, k))
    a = DistillArgs(*head, loss.data_ptr(), lse.data_ptr(), lp.data_ptr(),
                    other.data_ptr() if rest else None)
    key = (dev.index, "distill", k, a.rest, head[1] & 15, head[4] & 15) + head[0:1] + head[2:4] + \
        head[5:8]
    ws, a.workspace_bytes = _workspace(torch, ctx, L.fdb_distill_workspace, a, key, dev, workspace)
    a.workspace = ws.data_ptr()
    a.stream = torch._C._cuda_getCurrentRawStream(dev.index)
    rc = L.fdb_distill(ctx.h, C.byref(a))
    if rc:
        _check(rc)
    return Distilled(loss, lse, lp, other)


def distill_backward(queries, rows, teacher_ids, teacher_logits, lse, logprobs, rest=None, *,
                     d_loss, scale: float = 1.0, teacher_scale: float = 1.0, allowed=None,
                     need_queries: bool = True, need_rows: bool = True, workspace=None):
    """(d_queries, d_rows) of sum(d_loss * loss), given what distill returned for
    the same arguments: lse, logprobs and, if it was called with rest, its rest
    (fdb_distill_backward in forgegpu.h).  A gradient that is not needed is None;
    the teacher's lists have none."""
    torch = _torch()
    head = _distill_args(queries, rows, teacher_ids, teacher_logits, scale, teacher_scale,
                         0 if rest is None else 1, allowed)
    dev, f32 = queries.device, torch.float32
    nq, n, dim, k = head[2], head[5], head[7], head[11]
    if logprobs.dtype != f32 or logprobs.device != dev or logprobs.shape != (nq, k) or \
            not logprobs.is_contiguous():
        _refuse(f"logprobs must be a contiguous {f32} tensor [{nq}, {k}] on the queries' device")
    ctx = _ctx_of(dev)
    L = lib()
    dq = torch.empty((nq, dim), dtype=queries.dtype, device=dev) if need_queries else None
    dx = torch.empty((n, dim), dtype=queries.dtype, device=dev) if need_rows else None
    a = DistillGradArgs(*head, _vector(lse, nq, f32, dev, "lse"), logprobs.data_ptr(),
                        _vector(rest, nq, f32, dev, "rest"),
                        _vector(d_loss, nq, f32, dev, "d_loss"),
                        None if dq is None else dq.data_ptr(), dim,
                        None if dx is None else dx.data_ptr(), dim)
    key = (dev.index, "distill_backward", k, allowed is not None and head[17]) + head[0:1] + \
        head[2:4] + head[5:8]
    ws, a.workspace_bytes = _workspace(torch, ctx, L.fdb_distill_backward_workspace, a, key, dev,
                                       workspace)
    a.workspace = ws.data_ptr()
    a.stream = torch._C._cuda_getCurrentRawStream(dev.index)
    rc = L.fdb_distill_backward(ctx.h, C.byref(a))
    if rc:
        _check(rc)
    return dq, dx


def beam_select(scores, beam_scores, *, width: int | None = None, ids=None, scale: float = 1.0,
                normalise: bool = True, allowed=None, ended=None, end_id: int = -1,
                workspace=None) -> Beams:
    """The `width` best continuations of each search's chains, on the current
    stream (fdb_beam_select in forgegpu.h): scores [groups, beams, n] are the
    columns' logits (with normalise) or log probabilities, beam_scores float32
    [groups, beams] the chains' so far.

    ids: int64 [groups, beams, n], what the columns stand for (none where
    negative).  allowed: int32 words of a bit per column, one filter or
    [groups * beams, words].  ended: bool [groups, beams], chains that stay as
    they are; end_id: the id that ends one.  Results [groups, width]: scores,
    the chains (int64) and ids (int64) they continue with, ended (bool)."""
    torch = _torch()
    dev = scores.device
    if scores.dim() != 3 or dev.type != "cuda" or scores.dtype not in _DTYPE:
        _refuse("scores must be a [groups, beams, n] float32, float16 or bfloat16 tensor on a GPU")
    g, b, n = scores.shape
    s0, s1, s2 = scores.stride()
    if (n > 1 and s2 != 1) or (b > 1 and s1 < n):
        _refuse("scores must have contiguous rows")
    f32 = torch.float32
    if beam_scores.dtype != f32 or beam_scores.device != dev or beam_scores.shape != (g, b) or \
            not beam_scores.is_contiguous():
        _refuse("beam_scores must be a contiguous float32 [groups, beams] tensor on the scores' "
                "device")
    ip = ep = ap = None
    if ids is not None:
        if ids.dtype != torch.int64 or ids.device != dev or ids.shape != (g, b, n) or \
                not ids.is_contiguous():
            _refuse("ids must be a contiguous int64 tensor of the scores' shape and device")
        ip = ids.data_ptr()
    lda = 0
    if allowed is not None:
        words = (n + 31) // 32
        if allowed.dtype != torch.int32 or allowed.device != dev or allowed.dim() not in (1, 2) \
                or allowed.shape[-1] != words or (words > 1 and allowed.stride(-1) != 1):
            _refuse(f"allowed must be int32 words [{words}] or [1 or groups * beams, {words}] on "
                    "the scores' device")
        filters = 1 if allowed.dim() == 1 else allowed.shape[0]
        if filters not in (1, g * b):
            _refuse(f"allowed has {filters} filters for {g * b} chains")
        ap = allowed.data_ptr()
        if filters > 1:
            lda = allowed.stride(0)
            if lda < words:
                _refuse("allowed must have contiguous rows")
    if ended is not None:
        if ended.dtype not in (torch.bool, torch.uint8) or ended.device != dev or \
                ended.shape != (g, b) or not ended.is_contiguous():
            _refuse("ended must be a contiguous bool [groups, beams] tensor on the scores' device")
        ep = ended.data_ptr()
    w = b if width is None else width
    if not 1 <= w <= 128:
        _refuse("width must be in [1, 128]")
    ctx = _ctx_of(dev)
    L = lib()
    # (made like what is there: half the time of torch.empty)
    top = torch.empty_like(beam_scores) if w == b else beam_scores.new_empty((g, w))
    parents = top.new_empty((g, w), dtype=torch.int64)
    out, done = torch.empty_like(parents), top.new_empty((g, w), dtype=torch.bool)
    a = BeamArgs(_DTYPE[scores.dtype], scores.data_ptr(), g, b, n, s0, s1 if b > 1 else n, scale,
                 1 if normalise else 0, ip, n, ap, lda, beam_scores.data_ptr(), ep, end_id, w,
                 top.data_ptr(), parents.data_ptr(), out.data_ptr(), done.data_ptr())
    key = (dev.index, "beam", a.dtype, g, b, n, w, a.normalise, ip is None,
           scores.data_ptr() & 15, s0, s1)
    if _ws_bytes.get(key) != 0 or workspace is not None:  # (small searches need none)
        ws, a.workspace_bytes = _workspace(torch, ctx, L.fdb_beam_select_workspace, a, key, dev,
                                           workspace)
        a.workspace = ws.data_ptr()
    a.stream = torch._C._cuda_getCurrentRawStream(dev.index)
    rc = L.fdb_beam_select(ctx.h, C.byref(a))
    if rc:
        _check(rc)
    return Beams(top, parents, out, done)


def _runs(t, what: str):
    """(row distance, runs of a row, run distance, elements of a run) of a state
    [groups, beams, ...] whose rows are evenly spaced and whose inner dimensions
    are contiguous but for one step."""
    shape, stride = t.shape, t.stride()
    if len(shape) < 2:
        _refuse(f"{what} must be [groups, beams, ...]")
    rows = stride[1] if shape[1] > 1 else stride[0]
    if shape[0] > 1 and shape[1] > 1 and stride[0] != shape[1] * stride[1]:
        _refuse(f"{what} must have evenly spaced rows")
    run, d = 1, len(shape) - 1
    while d > 1 and (shape[d] == 1 or stride[d] == run):
        run *= shape[d]
        d -= 1
    parts, step = 1, 0
    while d > 1 and (shape[d] == 1 or parts == 1 or stride[d] == parts * step):
        if shape[d] > 1:
            if parts == 1:
                step = stride[d]
            parts *= shape[d]
        d -= 1
    if d > 1 or (parts > 1 and step < run):
        _refuse(f"{what} must be contiguous past its second dimension, but for one step")
    return rows, parts, step, run


def beam_reorder(states, parents, out=None):
    """States that follow their chains, on the current stream (fdb_beam_reorder
    in forgegpu.h): row [g, w] of each result is row [g, parents[g, w]] of the
    state [groups, beams, ...].  out: tensors to write to (new ones if None); a
    state itself, where width is beams, is reordered in place.  States and out
    may be parts of wider tensors (the positions in use of a cache); what a
    parent outside [0, beams) would bring is left as it was (zeros in a new
    one).  Returns the results.  To autograd it is an in-place change of out."""
    torch = _torch()
    if parents.dtype != torch.int64 or parents.dim() != 2 or not parents.is_contiguous() or \
            not parents.is_cuda:
        _refuse("parents must be a contiguous int64 [groups, width] tensor on a GPU")
    g, w = parents.shape
    dev = parents.device
    if out is not None and len(out) != len(states):
        _refuse("out must be a list of the states' length")
    if not states:
        return []
    b = states[0].shape[1] if states[0].dim() > 1 else 0
    new = out is None
    if new:
        out = [torch.empty((g, w) + t.shape[2:], dtype=t.dtype, device=dev) for t in states]
    table = array.array("Q")
    for t, o in zip(states, out):
        if t.device != dev or o.device != dev or t.dtype != o.dtype or t.shape[:2] != (g, b) or \
                o.shape != (g, w) + t.shape[2:]:
            _refuse("states must be [groups, beams, ...] and out [groups, width, ...] of their "
                    "types, on the parents' device")
        es = t.element_size()
        if t.is_contiguous() and o.is_contiguous():
            bytes_ = t.numel() // max(1, g * b) * es
            table.extend((t.data_ptr(), o.data_ptr(), bytes_, bytes_, 1, 0, 0, bytes_))
            continue
        rows, parts, step, run = _runs(t, "a state")
        orows, oparts, ostep, orun = _runs(o, "out")
        if (parts, run) != (oparts, orun):  # (one of them is contiguous: in the other's runs)
            if oparts == 1 and orun == parts * run:
                oparts, ostep, orun = parts, run, run
            elif parts == 1 and run == oparts * orun:
                parts, step, run = oparts, orun, orun
            else:
                _refuse("a state and its out must fall into the same runs")
        if t.numel() == 0:
            parts = 0
        table.extend((t.data_ptr(), o.data_ptr(), rows * es, orows * es, parts, step * es,
                      ostep * es, run * es))
    opts = ReorderOpts(parents.data_ptr(), g, b, w, 1 if new else 0,
                       torch._C._cuda_getCurrentRawStream(dev.index))
    _check(lib().fdb_beam_reorder(_ctx_of(dev).h, table.buffer_info()[0], len(out),
                                  C.byref(opts)))
    if not new:
        # (written through pointers: a graph that saved one of them has to notice)
        torch.autograd.graph.increment_version(out)
    return list(out)


def _scalar(t, dtype, like, what: str):
    if t is None:
        return None
    if t.dtype != dtype or t.device != like.device or t.numel() != 1:
        _refuse(f"{what} must be one {dtype} value on the params' device")
    return t.data_ptr()


def adamw_step(params, grads, m, v, *, lr: float, step: int = 1, betas=(0.9, 0.999),
               eps: float = 1e-8, weight_decay: float = 0.01, grad_scale: float = 1.0,
               m_scales=None, v_scales=None, seed: int = 0, d_lr=None, d_step=None,
               d_grad_scale=None):
    """One AdamW step in place over lists of tensors, on the current stream
    (fdb_adamw_step in forgegpu.h).  With m_scales and v_scales the moments
    are 8-bit: m int8, v uint8, a float32 scale per 256 elements each.  To
    autograd it is an in-place change of params."""
    torch = _torch()
    count = len(params)
    eight = m_scales is not None or v_scales is not None
    lists = [params, grads, m, v] + ([m_scales, v_scales] if eight else [])
    if any(x is None or len(x) != count for x in lists):
        _refuse("params, grads and states must be lists of one length")
    if count == 0:
        return
    p0, g0 = params[0], grads[0]
    dev = p0.device
    if dev.type != "cuda" or p0.dtype not in _DTYPE or g0.dtype not in _DTYPE:
        _refuse("params and grads must be float32, float16 or bfloat16 tensors on a GPU")
    types = [p0.dtype, g0.dtype] + ([torch.int8, torch.uint8, torch.float32, torch.float32]
                                    if eight else [torch.float32, torch.float32])
    T = torch.Tensor  # (its methods mapped: a model's tensors are many)
    sizes = list(map(T.numel, params))
    blocks = [(n + 255) // 256 for n in sizes] if eight else None
    cols = []
    for what, (ts, dtype) in enumerate(zip(lists, types)):
        if {t.dtype for t in ts} != {dtype} or set(map(T.get_device, ts)) != {dev.index} \
                or list(map(T.numel, ts)) != (sizes if what < 4 else blocks) \
                or not all(map(T.is_contiguous, ts)):
            _refuse("params, grads and states must be contiguous, of one type each, of the "
                    "params' sizes (scales: one per 256 elements) and device")
        cols.append(list(map(T.data_ptr, ts)))
    if not eight:
        cols += [[0] * count] * 2
    table = array.array("Q", itertools.chain.from_iterable(zip(*cols, sizes)))
    o = AdamwOpts(_DTYPE[p0.dtype], _DTYPE[g0.dtype], 8 if eight else 32, seed & 0xFFFFFFFF, lr,
                  betas[0], betas[1], eps, weight_decay, grad_scale, step,
                  _scalar(d_lr, torch.float32, p0, "d_lr"),
                  _scalar(d_step, torch.int64, p0, "d_step"),
                  _scalar(d_grad_scale, torch.float32, p0, "d_grad_scale"),
                  torch._C._cuda_getCurrentRawStream(dev.index))
    _check(lib().fdb_adamw_step(_ctx_of(dev).h, table.buffer_info()[0], count, C.byref(o)))
    # (written through pointers: a graph that saved a param has to notice)
    torch.autograd.graph.increment_version(params)


def adamw_state_values(m, m_scale, v, v_scale):
    """The float32 values (m, v) that 8-bit moments stand for."""
    torch = _torch()
    n = m.numel()
    for t, dtype, size in ((m, torch.int8, n), (v, torch.uint8, n),
                           (m_scale, torch.float32, (n + 255) // 256),
                           (v_scale, torch.float32, (n + 255) // 256)):
        if t.dtype != dtype or t.device != m.device or t.numel() != size or \
                not t.is_contiguous() or t.device.type != "cuda":
            _refuse("8-bit moments are int8 m and uint8 v of one size with a float32 scale per "
                    "256 elements, contiguous, on one GPU")
    om = torch.empty(m.shape, dtype=torch.float32, device=m.device)
    ov = torch.empty(m.shape, dtype=torch.float32, device=m.device)
    _check(lib().fdb_adamw_state_values(
        _ctx_of(m.device).h, m.data_ptr(), m_scale.data_ptr(), v.data_ptr(), v_scale.data_ptr(), n,
        om.data_ptr(), ov.data_ptr(), torch._C._cuda_getCurrentRawStream(m.device.index)))
    return om, ov
