"""Thin torch-tensor front end of the C ABI: shape checks, pointers, the current HIP stream.

torch is used here for device memory and streams only; every function below enqueues one or
more kernels of ``libathena_hip.so`` on ``torch.cuda.current_stream()``.
"""
import collections
import contextlib
import ctypes
import math
import os

import torch

from . import _lib
from ._lib import (ACT_GELU, ACT_MUL_DGELU, ACT_MUL_DRELU6, ACT_MUL_DUNARY, ACT_NONE, ACT_RELU6, ACT_UNARY, BF16,  # noqa: F401
                   F32)


def dt(t):
    """ATHENA dtype code of a tensor or torch dtype."""
    d = t.dtype if isinstance(t, torch.Tensor) else t
    if d == torch.float32:
        return F32
    if d == torch.bfloat16:
        return BF16
    raise TypeError("athena_amd: unsupported dtype %s" % d)


def _ptr(t):
    if t is None:
        return None
    if not t.is_cuda:
        raise RuntimeError("athena_amd: tensors must live on the GPU (got %s)" % t.device)
    return t.data_ptr()


def _extent(t):
    """Elements addressable from ``t``'s first element to the end of its storage (a column block of
    a wider matrix is passed as a view plus the wide leading dimension)."""
    return t.untyped_storage().nbytes() // t.element_size() - t.storage_offset()


def _stream():
    return torch.cuda.current_stream().cuda_stream


def roundup(x, m):
    return (x + m - 1) // m * m


def _rows2d(t):
    """(rows, cols, ld) of a tensor viewed as a matrix with contiguous last dim."""
    if t.stride(-1) != 1:
        raise RuntimeError("athena_amd: last dimension must be contiguous")
    cols = t.shape[-1]
    rows = t.numel() // cols
    if t.dim() == 1:
        return 1, cols, cols
    ld = t.stride(-2)
    # all leading dims must be collapsible onto one row stride
    exp = ld
    for i in range(t.dim() - 2, -1, -1):
        if t.shape[i] != 1 and t.stride(i) != exp:
            raise RuntimeError("athena_amd: tensor is not a strided matrix: shape %s stride %s" %
                               (tuple(t.shape), t.stride()))
        exp *= t.shape[i]
    return rows, cols, ld


# ------------------------------------------------------------------------------------------ GEMM
_WORKSPACE = {}
WORKSPACE_BYTES = 64 << 20


def splitk_workspace(device):
    """Per-device scratch for split-K partial sums.  Kernels on one stream use it one after the
    other; it is allocated once so that captured HIP graphs keep a stable address."""
    key = torch.device(device).index if torch.device(device).index is not None else torch.cuda.current_device()
    ws = _WORKSPACE.get(key)
    if ws is None:
        ws = torch.empty(WORKSPACE_BYTES, dtype=torch.uint8, device=torch.device("cuda", key))
        _WORKSPACE[key] = ws
    return ws


def _fill_gemm_desc(d, a, b, c, M, N, K, trans_a=False, trans_b=False, lda=None, ldb=None, ldc=None, bias=None,
                    act=ACT_NONE, aux=None, ldaux=0, c_pre=None, accumulate=False, split_k=1, alpha=1.0,
                    drop_p=0.0, rng_state=None, rng_site=0, b_colsum=None):
    """Checks the operands of one product and fills the ``athena_gemm_desc`` ``d``."""
    d.A, d.B, d.C = _ptr(a), _ptr(b), _ptr(c)
    d.C_pre = _ptr(c_pre)
    d.bias = _ptr(bias)
    d.aux = _ptr(aux)
    d.rng_state = _ptr(rng_state)
    d.M, d.N, d.K = M, N, K
    d.trans_a, d.trans_b = int(trans_a), int(trans_b)
    d.lda = lda if lda is not None else (M if trans_a else K)
    d.ldb = ldb if ldb is not None else (K if trans_b else N)
    d.ldc = ldc if ldc is not None else N
    d.ldaux = ldaux
    if a.dtype != b.dtype:
        raise TypeError("athena_amd.gemm: operand dtypes differ (%s, %s)" % (a.dtype, b.dtype))
    d.in_dtype = dt(a)
    d.out_dtype = dt(c)
    d.aux_dtype = dt(aux) if aux is not None else F32
    d.act = act
    d.accumulate = int(accumulate)
    d.split_k = split_k
    d.alpha = alpha
    d.drop_p = drop_p
    d.rng_site = rng_site
    if b_colsum is not None:
        if b_colsum.dtype != torch.float32 or b_colsum.numel() < N:
            raise RuntimeError("athena_amd.gemm: b_colsum must be fp32 [N]")
        d.b_colsum = _ptr(b_colsum)
    if split_k == 0:
        ws = splitk_workspace(a.device)
        d.workspace = ws.data_ptr()
        d.workspace_bytes = ws.numel()
    # bounds: the last row read/written must lie inside the tensors
    a_rows = K if trans_a else M
    b_rows = N if trans_b else K
    if _extent(a) < (a_rows - 1) * d.lda + (M if trans_a else K):
        raise RuntimeError("athena_amd.gemm: A too small for M=%d K=%d lda=%d" % (M, K, d.lda))
    if _extent(b) < (b_rows - 1) * d.ldb + (K if trans_b else N):
        raise RuntimeError("athena_amd.gemm: B too small for N=%d K=%d ldb=%d" % (N, K, d.ldb))
    if _extent(c) < (M - 1) * d.ldc + N:
        raise RuntimeError("athena_amd.gemm: C too small for M=%d N=%d ldc=%d" % (M, N, d.ldc))
    if aux is not None and aux.numel() < (M - 1) * ldaux + N:
        raise RuntimeError("athena_amd.gemm: aux too small")
    if bias is not None and (bias.dtype != torch.float32 or bias.numel() < N):
        raise RuntimeError("athena_amd.gemm: bias must be fp32 [N]")


_SMALL_WS = {}


def small_workspace(device):
    """Per-device 8 MB scratch for the slab reductions of the normalisation kernels (kept apart
    from the split-K workspace so that the two never alias)."""
    key = torch.device(device).index if torch.device(device).index is not None else torch.cuda.current_device()
    ws = _SMALL_WS.get(key)
    if ws is None:
        ws = _SMALL_WS[key] = torch.empty(8 << 20, dtype=torch.uint8, device=torch.device("cuda", key))
    return ws


def gemm(a, b, c, M, N, K, **kw):
    """C[M,N] = epilogue(alpha * op(A) op(B)); see ``athena_gemm`` in include/athena_hip.h."""
    lib = _lib.load()
    d = _lib.GemmDesc()
    _fill_gemm_desc(d, a, b, c, M, N, K, **kw)
    _lib.check(lib.athena_gemm(ctypes.byref(d), _stream()), "athena_gemm")


def gemm_grouped(problems):
    """Independent products in one launch; ``problems`` is a list of (a, b, c, M, N, K, kwargs) as
    for ``gemm``.  See ``athena_gemm_grouped`` in include/athena_hip.h."""
    if not problems:
        return
    lib = _lib.load()
    descs = (_lib.GemmDesc * len(problems))()
    for d, (a, b, c, M, N, K, kw) in zip(descs, problems):
        _fill_gemm_desc(d, a, b, c, M, N, K, **kw)
    _lib.check(lib.athena_gemm_grouped(descs, len(problems), _stream()), "athena_gemm_grouped")


PANEL_MAX_BLOCKS = 20
PANEL_ENABLED = os.environ.get("ATHENA_PANEL_GEMM", "1") != "0"


def panel_gemm(x, rows, blocks):
    """out_c[rows, 256] = x[rows, 256] W_c (+ bias_c) for every (w_tiled, bias or None, out, ldo) of
    ``blocks`` in one launch; ``w_tiled``: the fragment-tiled copy of the [256, 256] block whose rows are the
    block's output columns.  bf16; see ``athena_panel_gemm`` in include/athena_hip.h."""
    n = len(blocks)
    ldx = x.stride(-2) if x.dim() >= 2 else 256
    if x.dtype != torch.bfloat16 or x.stride(-1) != 1 or not 0 < n <= PANEL_MAX_BLOCKS or \
            _extent(x) < (rows - 1) * ldx + 256:
        raise RuntimeError("athena_amd.panel_gemm: bf16 rows of 256 and 1..%d blocks expected" % PANEL_MAX_BLOCKS)
    for w, b, out, ldo in blocks:
        if w.dtype != torch.bfloat16 or w.numel() < 65536 or out.dtype != torch.bfloat16 or \
                _extent(out) < (rows - 1) * ldo + 256 or (b is not None and (b.dtype != torch.float32 or b.numel() < 256)):
            raise RuntimeError("athena_amd.panel_gemm: a block needs 256 x 256 tiled bf16 weights, an fp32 bias of 256 "
                               "or none, and a bf16 output of rows x 256")
    wp = (ctypes.c_void_p * n)(*[w.data_ptr() for w, _, _, _ in blocks])
    bp = (ctypes.c_void_p * n)(*[(b.data_ptr() if b is not None else None) for _, b, _, _ in blocks])
    op = (ctypes.c_void_p * n)(*[o.data_ptr() for _, _, o, _ in blocks])
    ld = (ctypes.c_long * n)(*[int(l) for _, _, _, l in blocks])
    _lib.check(_lib.load().athena_panel_gemm(_ptr(x), ldx, rows, n, wp, bp, op, ld, _stream()), "athena_panel_gemm")


def panel_gemm_k(a, rows, kcols, pieces, out, ldo, bias=None, act=ACT_NONE, accumulate=False):
    """out[rows, 256] (+)= act(sum_c a[:, 256 c : 256 c + 256] W_c + bias); ``pieces``: (tiled weights from the
    piece's start, contraction length of that tiled copy) per 256 columns of ``a``.  bf16; see
    ``athena_panel_gemm_k`` in include/athena_hip.h."""
    n = len(pieces)
    lda = a.stride(-2)
    if a.dtype != torch.bfloat16 or out.dtype != torch.bfloat16 or a.stride(-1) != 1 or not 0 < n <= PANEL_MAX_BLOCKS or \
            _extent(a) < (rows - 1) * lda + kcols or _extent(out) < (rows - 1) * ldo + 256 or \
            (bias is not None and (bias.dtype != torch.float32 or bias.numel() < 256)):
        raise RuntimeError("athena_amd.panel_gemm_k: bf16 operands, 1..%d pieces and an fp32 bias of 256 expected"
                           % PANEL_MAX_BLOCKS)
    for w, ldw in pieces:
        if w.dtype != torch.bfloat16 or _extent(w) < 240 * ldw + 4096:      # the last fragment the launch reads ends there
            raise RuntimeError("athena_amd.panel_gemm_k: tiled bf16 weights expected")
    wp = (ctypes.c_void_p * n)(*[w.data_ptr() for w, _ in pieces])
    ld = (ctypes.c_long * n)(*[int(l) for _, l in pieces])
    _lib.check(_lib.load().athena_panel_gemm_k(_ptr(a), lda, rows, kcols, n, wp, ld, _ptr(bias), act, 1 if accumulate else 0,
                                               _ptr(out), ldo, _stream()), "athena_panel_gemm_k")


class _StepTables:
    """Device memory for the problem tables of a step that is being recorded, filled once.

    A table built while a HIP graph is captured holds addresses of that graph's buffers, so it cannot be
    built ahead of the capture; uploaded by a recorded copy it would be copied again at every replay
    (a copy node costs about as much as a small kernel, and a data-parallel step builds eight tables).
    ``begin`` (before the capture) sets aside a chunk of device memory and a pinned host image of it;
    a table built during the capture is placed in the image and the recorded kernel is given the
    address the table will have; ``end`` (after the capture, before the first replay) copies the image
    over in one piece and returns what the recorded step has to keep alive: the chunk and every cached
    table the capture used.  Outside ``begin`` / ``end`` tables are uploaded where they are built."""
    BYTES = 1 << 20
    enabled = os.environ.get("ATHENA_STEP_TABLES", "1") != "0"
    active = None

    @classmethod
    def begin(cls, device):
        if cls.active is not None:
            return
        # (switched off, a recorded step still keeps the tables it used -- device copy and pinned source of
        # the recorded upload -- alive: the caches below drop their oldest entries)
        cls.active = {"chunk": torch.empty(cls.BYTES, dtype=torch.uint8, device=device) if cls.enabled else None,
                      "host": torch.empty(cls.BYTES, dtype=torch.uint8).pin_memory() if cls.enabled else None,
                      "cursor": 0, "kept": []}

    @classmethod
    def place(cls, raw, device):
        a = cls.active
        if a is None or a["chunk"] is None or not torch.cuda.is_current_stream_capturing() or a["chunk"].device != device:
            return None
        at = (a["cursor"] + 255) // 256 * 256
        if at + len(raw) > cls.BYTES:
            return None
        a["host"][at:at + len(raw)] = torch.frombuffer(bytearray(raw), dtype=torch.uint8)
        a["cursor"] = at + len(raw)
        return a["chunk"][at:at + len(raw)]

    @classmethod
    def keep(cls, obj):
        if cls.active is not None:
            cls.active["kept"].append(obj)

    @classmethod
    def end(cls):
        a, cls.active = cls.active, None
        if a is None:
            return None
        if a["cursor"]:
            a["chunk"][:a["cursor"]].copy_(a["host"][:a["cursor"]])
            torch.cuda.current_stream(a["chunk"].device).synchronize()
        return a["kept"] + [a["chunk"]]      # (not the pinned image: it has been copied)


@contextlib.contextmanager
def step_tables(owner, device):
    """Around the captures of one recorded step: see ``_StepTables``.  ``owner`` keeps the tables."""
    _StepTables.begin(device)
    try:
        yield
    finally:
        owner._tables = _StepTables.end()


class _WgradTables:
    """Device copies of the problem tables of ``gemm_wgrad_table``, by content.

    Under HIP-graph replay a step hands over the same table every time (the buffers of a recorded
    step do not move), so a table is split, planned, pinned and uploaded once; the uploads are
    asynchronous copies from pinned memory, which a graph capture can record.  Eager steps produce a
    new table each time: only the most recent ones are kept.  An entry also owns the workspace of
    the partial products of a table whose contractions were split."""
    KEEP = 48
    cache = {}

    @staticmethod
    def _upload(arr, device):
        placed = _StepTables.place(bytes(arr), device)
        if placed is not None:
            return placed, None
        host = torch.frombuffer(bytearray(bytes(arr)), dtype=torch.uint8).pin_memory()
        dev_t = torch.empty(host.numel(), dtype=torch.uint8, device=device)
        dev_t.copy_(host, non_blocking=True)
        return dev_t, host

    @classmethod
    def get(cls, key, items, device):
        hit = cls.cache.pop(key, None)
        if hit is None:
            lib = _lib.load()
            arr = (_lib.WgradItem * len(items))()
            for it, (a, b, c, bsum, M, N, K, lda, ldb, ldc) in zip(arr, items):
                it.A, it.B, it.C, it.bsum = a, b, c, bsum
                it.M, it.N, it.K, it.lda, it.ldb, it.ldc = M, N, K, lda, ldb, ldc
            # a table with few tiles gets its long contractions cut into parts (sizing call, then the real one)
            need, n_out, n_fold, blocks = ctypes.c_int64(0), ctypes.c_int(0), ctypes.c_int(0), ctypes.c_int(0)
            split = cls.split_enabled
            if split:
                _lib.check(lib.athena_gemm_wgrad_split(arr, len(items), 0, None, 0, ctypes.byref(need), None, 0,
                                                       ctypes.byref(n_out), None, 0, ctypes.byref(n_fold), None),
                           "athena_gemm_wgrad_split")
            work, folds_dev, folds_host = None, None, None
            if split and n_fold.value > 0:
                work = torch.empty(need.value, dtype=torch.float32, device=device)
                out = (_lib.WgradItem * n_out.value)()
                folds = (_lib.WgradFold * n_fold.value)()
                _lib.check(lib.athena_gemm_wgrad_split(arr, len(items), 0, work.data_ptr(), need.value,
                                                       ctypes.byref(need), out, n_out.value, ctypes.byref(n_out), folds,
                                                       n_fold.value, ctypes.byref(n_fold), ctypes.byref(blocks)),
                           "athena_gemm_wgrad_split")
                arr = out
            else:
                folds = None
            total = ctypes.c_int(0)
            _lib.check(lib.athena_gemm_wgrad_plan(arr, len(arr), ctypes.byref(total)), "athena_gemm_wgrad_plan")
            # both tables travel in one copy: the items, then (16-byte aligned) the folds
            blob = bytes(arr)
            fold_at = (len(blob) + 15) // 16 * 16
            if folds is not None:
                blob = blob + bytes(fold_at - len(blob)) + bytes(folds)
            dev_t, host = cls._upload(blob, device)
            hit = (dev_t, host, total.value, len(arr), work, dev_t[fold_at:] if folds is not None else None,
                   None, n_fold.value, blocks.value)
        _StepTables.keep(hit)
        if hit[1] is None:
            return hit                           # lies in a recorded step's own chunk: lives and dies with that step
        cls.cache[key] = hit                     # most recently used last
        # (nothing is dropped while a stream is recording: that would release pinned and device memory in the
        # middle of a capture)
        while len(cls.cache) > cls.KEEP and not torch.cuda.is_current_stream_capturing():
            del cls.cache[next(iter(cls.cache))]
        return hit


_WgradTables.split_enabled = os.environ.get("ATHENA_WGRAD_SPLIT", "1") != "0"


def gemm_wgrad_table(problems):
    """kernel.grad_i = x_i^T dy_i and bias.grad_i = column sums of dy_i for many Dense layers in one
    launch (bf16 operands, fp32 results).  ``problems``: list of
    (x [K, ldx], dy [K, lddy], K, M, N, ldx, lddy, dkernel [M, N] fp32, dbias [N] fp32 or None).
    A table too small to fill the chip has its long contractions cut into parts, summed by a second
    launch in a fixed order.  See ``athena_gemm_wgrad_table`` / ``athena_gemm_wgrad_split`` in
    include/athena_hip.h."""
    if not problems:
        return
    items = []
    for (x, dy, K, M, N, ldx, lddy, dk, db) in problems:
        if x.dtype != torch.bfloat16 or dy.dtype != torch.bfloat16 or dk.dtype != torch.float32:
            raise TypeError("athena_amd.gemm_wgrad_table: bf16 operands and fp32 results expected")
        if _extent(x) < (K - 1) * ldx + M or _extent(dy) < (K - 1) * lddy + N or dk.numel() < M * N or \
                (db is not None and (db.dtype != torch.float32 or db.numel() < N)):
            raise RuntimeError("athena_amd.gemm_wgrad_table: operand too small for K=%d M=%d N=%d" % (K, M, N))
        items.append((_ptr(x), _ptr(dy), _ptr(dk), _ptr(db), M, N, K, ldx, lddy, N))
    key = tuple(items)
    table, _, total, count, _, folds, _, n_fold, blocks = _WgradTables.get(key, items, problems[0][0].device)
    lib = _lib.load()
    _lib.check(lib.athena_gemm_wgrad_table(table.data_ptr(), count, total, _stream()), "athena_gemm_wgrad_table")
    if n_fold:
        _lib.check(lib.athena_gemm_wgrad_fold(folds.data_ptr(), n_fold, blocks, _stream()), "athena_gemm_wgrad_fold")


def colsum(x, M, N, ld, out):
    lib = _lib.load()
    if out.dtype != torch.float32 or out.numel() < N or x.numel() < (M - 1) * ld + N:
        raise RuntimeError("athena_amd.colsum: bad operands")
    _lib.check(lib.athena_colsum(_ptr(x), dt(x), M, N, ld, _ptr(out), _stream()), "athena_colsum")


# ------------------------------------------------------------------------------------------ LayerNorm
def layernorm_wide_ok(a):
    """Can ``add_layernorm_fwd`` take / leave the fp32 copy of the residual stream for this tensor?"""
    return a.dtype == torch.bfloat16 and a.is_contiguous() and a.shape[-1] % 8 == 0 and a.shape[-1] <= 512 and \
        a.data_ptr() % 16 == 0


def add_layernorm_fwd(a, b, gamma, beta, eps, drop_p, rng_state, site, a32=None, want_y32=False):
    """z = a + dropout(b), y = LayerNorm(z); returns (z, y, mean, rstd).  ``a32``: ``a`` once more in fp32
    (taken for the sum in its place); ``want_y32``: a fifth result, y in fp32, for the call that takes
    y as its ``a`` -- see ``athena_add_layernorm_fwd_wide`` in include/athena_hip.h."""
    lib = _lib.load()
    rows, d, ld = _rows2d(a)
    if ld != d or (b is not None and (b.shape != a.shape or not b.is_contiguous())):
        raise RuntimeError("athena_amd.add_layernorm_fwd: operands must be contiguous and equal-shaped")
    z = torch.empty_like(a)
    y = torch.empty_like(a)
    mean = torch.empty(rows, dtype=torch.float32, device=a.device)
    rstd = torch.empty(rows, dtype=torch.float32, device=a.device)
    if a32 is not None or want_y32:
        if a32 is not None and (a32.dtype != torch.float32 or a32.numel() != a.numel() or not a32.is_contiguous()):
            raise RuntimeError("athena_amd.add_layernorm_fwd: a32 must be a contiguous fp32 copy of a")
        y32 = torch.empty(a.shape, dtype=torch.float32, device=a.device) if want_y32 else None
        _lib.check(lib.athena_add_layernorm_fwd_wide(_ptr(a), _ptr(a32), _ptr(b), _ptr(gamma), _ptr(beta), eps, rows, d,
                                                     dt(a), drop_p if b is not None else 0.0, _ptr(rng_state), site,
                                                     _ptr(z), _ptr(y), _ptr(y32), _ptr(mean), _ptr(rstd), _stream()),
                   "athena_add_layernorm_fwd_wide")
        return (z, y, mean, rstd, y32) if want_y32 else (z, y, mean, rstd)
    _lib.check(lib.athena_add_layernorm_fwd(_ptr(a), _ptr(b), _ptr(gamma), _ptr(beta), eps, rows, d, dt(a),
                                            drop_p if b is not None else 0.0, _ptr(rng_state), site, _ptr(z),
                                            _ptr(y), _ptr(mean), _ptr(rstd), _stream()), "athena_add_layernorm_fwd")
    return z, y, mean, rstd


class _LnFolds:
    """Column sums (dgamma, dbeta) of the LayerNorm gradients of one backward pass, folded together.

    Inside a backward pass every ``add_layernorm_bwd`` leaves its per-workgroup partial sums in its
    own piece of an arena, and one launch at the end of the pass (an end-of-backward callback of the
    autograd engine) adds them all up.  The table of pieces handed to that launch repeats from step
    to step, so it is built once per distinct sequence; a new one is uploaded from pinned memory
    with an asynchronous copy, which a HIP-graph capture can record."""
    ARENA_BYTES = 128 << 20
    state = {}

    @classmethod
    def get(cls, device):
        index = device.index if device.index is not None else torch.cuda.current_device()
        st = cls.state.get(index)
        if st is None:
            st = cls.state[index] = {"index": index, "arena": None, "cursor": 0, "items": [], "queued": False,
                                     "tables": {}}
        return st

    @classmethod
    def reserve(cls, device, nslab, d, dgamma, dbeta):
        """Arena piece (tensor view) for one deferred call, or None when folding cannot be deferred
        (not inside a backward pass, or the arena is full)."""
        st = cls.get(device)
        need = nslab * 2 * d
        if st["arena"] is None:
            st["arena"] = torch.empty(cls.ARENA_BYTES // 4, dtype=torch.float32,
                                      device=torch.device("cuda", st["index"]))
        if st["cursor"] + need > st["arena"].numel():
            return None
        if not st["queued"]:
            try:
                torch.autograd.Variable._execution_engine.queue_callback(lambda: cls.flush(st))
            except RuntimeError:
                return None
            st["queued"] = True
        piece = st["arena"][st["cursor"]:st["cursor"] + need]
        st["items"].append((piece.data_ptr(), dgamma.data_ptr(), dbeta.data_ptr(), nslab, d))
        st["cursor"] += (need + 63) // 64 * 64
        return piece

    @classmethod
    def flush(cls, st):
        items, st["items"], st["cursor"], st["queued"] = st["items"], [], 0, False
        if not items:
            return
        key = tuple(items)
        table = st["tables"].get(key)
        if table is None:
            import struct
            raw = b"".join(struct.pack("<QQQii", *it) for it in items)
            device = torch.device("cuda", st["index"])
            devt, host = _StepTables.place(raw, device), None
            if devt is None:
                host = torch.frombuffer(bytearray(raw), dtype=torch.uint8).pin_memory()
                devt = torch.empty(len(raw), dtype=torch.uint8, device=device)
                devt.copy_(host, non_blocking=True)
            table = (devt, host)
            if host is not None:
                # kept for good (a few KB per distinct sequence): a recorded step may replay the upload from
                # ``host`` into ``devt`` at any later time.  A table in a recorded step's own chunk is not
                # remembered here: it lives and dies with that step.
                st["tables"][key] = table
        _StepTables.keep(table)
        lib = _lib.load()
        with torch.cuda.device(st["index"]):
            _lib.check(lib.athena_ln_fold_batched(table[0].data_ptr(), len(items), max(it[4] for it in items),
                                                  _stream()), "athena_ln_fold_batched")


def add_layernorm_bwd(dy, z, mean, rstd, gamma, drop_p, rng_state, site, dgamma, dbeta, need_db=True):
    """Returns (da, db).  db is da itself when there is no dropout.  Inside a backward pass dgamma and
    dbeta are complete when the pass ends (see ``_LnFolds``), otherwise on return."""
    lib = _lib.load()
    rows, d, ld = _rows2d(z)
    if not dy.is_contiguous() or dy.shape != z.shape or ld != d:
        raise RuntimeError("athena_amd.add_layernorm_bwd: operands must be contiguous and equal-shaped")
    da = torch.empty_like(z)
    db = torch.empty_like(z) if (drop_p > 0.0 and need_db) else None
    nslab = lib.athena_add_layernorm_bwd_slabs(rows, d)
    piece = _LnFolds.reserve(z.device, nslab, d, dgamma, dbeta) if nslab > 0 else None
    if piece is not None:
        ws_ptr, ws_bytes, pg, pb = piece.data_ptr(), piece.numel() * 4, None, None
    else:
        ws = small_workspace(z.device)
        ws_ptr, ws_bytes, pg, pb = ws.data_ptr(), ws.numel(), _ptr(dgamma), _ptr(dbeta)
    _lib.check(lib.athena_add_layernorm_bwd(_ptr(dy), _ptr(z), _ptr(mean), _ptr(rstd), _ptr(gamma), rows, d,
                                            dt(z), drop_p if db is not None else 0.0, _ptr(rng_state), site, 0,
                                            _ptr(da), _ptr(db), pg, pb, ws_ptr, ws_bytes, _stream()),
               "athena_add_layernorm_bwd")
    return da, (db if db is not None else da)


# ------------------------------------------------------------------------------------------ fused layer tail
LAYER_TAIL_D = 256


LAYER_TAIL_MAX_DFF = 2048


def layer_tail_ok(x, d_model, proj, ffn0=None, ffn1=None):
    """True when ``layer_tail_fwd`` / ``layer_tail_bwd`` handle the layer: bf16, d_model 256, dff a
    multiple of 256 up to 2048 (no feed-forward part without ``ffn0``), fragment-tiled weight copies."""
    dff = ffn0.out_features if ffn0 is not None else 0
    return x.dtype == torch.bfloat16 and d_model == LAYER_TAIL_D and dff % LAYER_TAIL_D == 0 and \
        dff <= LAYER_TAIL_MAX_DFF and all(m is None or m.tiled is not None for m in (proj, ffn0, ffn1)) and \
        os.environ.get("ATHENA_LAYER_TAIL", "1") != "0"


def layer_tail_fwd(ctx, x, proj, norm1, ffn0, ffn1, norm2, eps, drop_p, rng_state, site_res1, site_ffn, site_res2,
                   next_qkv=None, x32=None, want_y32=False):
    """Output projection + residual + LayerNorm (+ feed-forward block + residual + LayerNorm when
    ``ffn0`` is given) of a post-LN transformer layer in one launch; see ``athena_layer_tail_fwd`` in
    include/athena_hip.h.  ``proj``, ``ffn0``, ``ffn1`` are Dense layers (their fragment-tiled bf16
    copies are read), ``norm1``, ``norm2`` LayerNorms.  ``next_qkv``: the three Dense layers (d x d, tiled)
    whose products with the layer's output the launch leaves as well ("q", "k", "v"); without a
    feed-forward part one Dense layer ("q").  ``x32``: the residual input once more in fp32 [rows, d] (what
    the launch in front left as "y32" when asked with ``want_y32``): the residual stream then passes
    unrounded.  Returns a dict of the tensors written."""
    lib = _lib.load()
    rows, d = x.shape
    dff = ffn0.out_features if ffn0 is not None else 0
    dev = x.device
    new = lambda cols: torch.empty((rows, cols), dtype=torch.bfloat16, device=dev)
    stat = lambda: torch.empty(rows, dtype=torch.float32, device=dev)
    out = {"z1": new(d), "y1": new(d), "mean1": stat(), "rstd1": stat()}
    if dff:
        out.update(hpre=new(dff), h=new(dff), z2=new(d), y2=new(d), mean2=stat(), rstd2=stat())
    if not (ctx.is_contiguous() and x.is_contiguous() and ctx.shape == x.shape and ctx.dtype == x.dtype ==
            torch.bfloat16 and proj.tiled_t is not None and proj.tiled_t.numel() == d * d and
            (not dff or (ffn0.tiled_t is not None and ffn1.tiled_t is not None and ffn0.in_features == d and
                         ffn1.in_features == dff and ffn1.out_features == d))):
        raise RuntimeError("athena_amd.layer_tail_fwd: operands must be contiguous bf16 [rows, d] and the Dense "
                           "layers must carry tiled weight copies")
    dsc = _lib.LayerTailFwd()
    dsc.rows, dsc.d_model, dsc.dff = rows, d, dff
    dsc.ctx, dsc.x = _ptr(ctx), _ptr(x)
    dsc.wo_t, dsc.bo = _ptr(proj.tiled_t), _ptr(proj.bias)
    dsc.gamma1, dsc.beta1 = _ptr(norm1.gamma), _ptr(norm1.beta)
    if dff:
        dsc.w1_t, dsc.b1, dsc.w2_t, dsc.b2 = _ptr(ffn0.tiled_t), _ptr(ffn0.bias), _ptr(ffn1.tiled_t), _ptr(ffn1.bias)
        dsc.gamma2, dsc.beta2 = _ptr(norm2.gamma), _ptr(norm2.beta)
    dsc.eps, dsc.drop_p, dsc.rng_state = eps, drop_p, _ptr(rng_state) if drop_p > 0.0 else None
    dsc.site_res1, dsc.site_ffn, dsc.site_res2 = site_res1, site_ffn, site_res2
    for name, t in out.items():
        setattr(dsc, name, _ptr(t))
    if next_qkv is not None:
        if len(next_qkv) != (3 if dff else 1) or any(m.tiled_t is None or m.in_features != d or m.out_features != d
                                                     for m in next_qkv):
            raise RuntimeError("athena_amd.layer_tail_fwd: next_qkv takes three tiled d x d Dense layers behind a "
                               "feed-forward part, one without")
        for i, (name, m) in enumerate(zip("qkv", next_qkv)):
            out[name] = new(d)
            dsc.next_w_t[i], dsc.next_b[i], dsc.next_out[i] = _ptr(m.tiled_t), _ptr(m.bias), _ptr(out[name])
    if x32 is not None:
        if x32.dtype != torch.float32 or x32.shape != x.shape or not x32.is_contiguous():
            raise RuntimeError("athena_amd.layer_tail_fwd: x32 must be a contiguous fp32 copy of x")
        dsc.x_f32 = _ptr(x32)
    if want_y32:
        out["y32"] = torch.empty((rows, d), dtype=torch.float32, device=dev)
        dsc.y_out_f32 = _ptr(out["y32"])
    _lib.check(lib.athena_layer_tail_fwd(ctypes.byref(dsc), _stream()), "athena_layer_tail_fwd")
    return out


def layer_tail_bwd(dy, saved, proj, norm1, ffn0, ffn1, norm2, drop_p, rng_state, site_res1, site_ffn, site_res2,
                   add=None):
    """Backward pass of ``layer_tail_fwd`` in one launch (``saved`` is what that returned).  Returns
    (df, dh, da, dx, dctx); df and dh are None without a feed-forward part.  The LayerNorm parameter
    gradients are complete when the enclosing backward pass ends (see ``_LnFolds``); outside one the
    call is refused (returns None) and the caller runs the separate kernels.  ``add`` = (dqkv [rows, 3d],
    (wq, wk, wv)) -- without the feed-forward part (dq [rows, d], (wq,)) --: ``dy`` is short of
    dqkv (wq | wk | wv)^T and the launch adds it first."""
    lib = _lib.load()
    rows, d = dy.shape
    dff = ffn0.out_features if ffn0 is not None else 0
    dev = dy.device
    nwg = lib.athena_layer_tail_workgroups(rows)
    slab1 = _LnFolds.reserve(dev, nwg, d, norm1.gamma.grad, norm1.beta.grad)
    if slab1 is None:
        return None
    slab2 = None
    if dff:
        slab2 = _LnFolds.reserve(dev, nwg, d, norm2.gamma.grad, norm2.beta.grad)
        if slab2 is None:
            raise RuntimeError("athena_amd.layer_tail_bwd: LayerNorm fold arena is full")
    if not (dy.is_contiguous() and dy.dtype == torch.bfloat16 and proj.tiled is not None and
            (not dff or (ffn0.tiled is not None and ffn1.tiled is not None))):
        raise RuntimeError("athena_amd.layer_tail_bwd: operands must be contiguous bf16 and the Dense layers must "
                           "carry tiled weight copies")
    new = lambda cols: torch.empty((rows, cols), dtype=torch.bfloat16, device=dev)
    da, dx, dctx = new(d), new(d), new(d)
    df, dh = (new(d), new(dff)) if dff else (None, None)
    dsc = _lib.LayerTailBwd()
    dsc.rows, dsc.d_model, dsc.dff = rows, d, dff
    dsc.dy = _ptr(dy)
    dsc.z1, dsc.mean1, dsc.rstd1, dsc.gamma1 = _ptr(saved["z1"]), _ptr(saved["mean1"]), _ptr(saved["rstd1"]), \
        _ptr(norm1.gamma)
    dsc.wo = _ptr(proj.tiled)
    if dff:
        dsc.z2, dsc.mean2, dsc.rstd2, dsc.gamma2 = _ptr(saved["z2"]), _ptr(saved["mean2"]), _ptr(saved["rstd2"]), \
            _ptr(norm2.gamma)
        dsc.hpre, dsc.w2, dsc.w1 = _ptr(saved["hpre"]), _ptr(ffn1.tiled), _ptr(ffn0.tiled)
        dsc.df, dsc.dh, dsc.slab2 = _ptr(df), _ptr(dh), slab2.data_ptr()
    dsc.drop_p, dsc.rng_state = drop_p, _ptr(rng_state) if drop_p > 0.0 else None
    dsc.site_res1, dsc.site_ffn, dsc.site_res2 = site_res1, site_ffn, site_res2
    dsc.da, dsc.dx, dsc.dctx, dsc.slab1 = _ptr(da), _ptr(dx), _ptr(dctx), slab1.data_ptr()
    if add is not None:
        dqkv, mats = add
        na = 3 if dff else 1
        if not (dqkv.is_contiguous() and dqkv.dtype == torch.bfloat16 and dqkv.shape == (rows, na * d)) or \
                len(mats) != na or any(m.tiled is None or m.in_features != d or m.out_features != d for m in mats):
            raise RuntimeError("athena_amd.layer_tail_bwd: add needs a contiguous bf16 [rows, %d d] gradient and %d "
                               "tiled d x d Dense layers" % (na, na))
        dsc.add_dqkv = _ptr(dqkv)
        for i, m in enumerate(mats):
            dsc.add_w[i] = _ptr(m.tiled)
    _lib.check(lib.athena_layer_tail_bwd(ctypes.byref(dsc), _stream()), "athena_layer_tail_bwd")
    return df, dh, da, dx, dctx


# ------------------------------------------------------------------------------------------ attention
def mha_fwd(q, k, v, ldq, ldk, ldv, key_mask, causal, B, h, Tq, Tk, dk, scale, out, ldo, lse):
    lib = _lib.load()
    _lib.check(lib.athena_mha_fwd(_ptr(q), _ptr(k), _ptr(v), ldq, ldk, ldv, _ptr(key_mask), int(causal), B, h,
                                  Tq, Tk, dk, dt(q), scale, _ptr(out), ldo, _ptr(lse), _stream()), "athena_mha_fwd")


def mha_bwd(q, k, v, ldq, ldk, ldv, key_mask, causal, B, h, Tq, Tk, dk, scale, out, dout, ldo, lse, delta,
            dq, dk_, dv, lddq, lddk, lddv):
    lib = _lib.load()
    _lib.check(lib.athena_mha_bwd(_ptr(q), _ptr(k), _ptr(v), ldq, ldk, ldv, _ptr(key_mask), int(causal), B, h,
                                  Tq, Tk, dk, dt(q), scale, _ptr(out), _ptr(dout), ldo, _ptr(lse), _ptr(delta),
                                  _ptr(dq), _ptr(dk_), _ptr(dv), lddq, lddk, lddv, _stream()), "athena_mha_bwd")


def mha_weights(q, k, ldq, ldk, key_mask, causal, B, h, Tq, Tk, dk, scale):
    """softmax(q k^T * scale + mask) as an fp32 tensor [B, h, Tq, Tk] (the inspection path)."""
    if q.dtype != k.dtype or _extent(q) < (B * Tq - 1) * ldq + h * dk or _extent(k) < (B * Tk - 1) * ldk + h * dk:
        raise RuntimeError("athena_amd.mha_weights: bad operands")
    w = torch.empty((B, h, Tq, Tk), dtype=torch.float32, device=q.device)
    _lib.check(_lib.load().athena_mha_weights(_ptr(q), _ptr(k), ldq, ldk, _ptr(key_mask), int(causal), B, h, Tq, Tk, dk,
                                              dt(q), scale, _ptr(w), _stream()), "athena_mha_weights")
    return w


# ------------------------------------------------------------------------------------------ conv / BN
def same_out(n):
    return (n + 1) // 2


def conv3x3s2_fwd(x, w, w_layout, out, B, H, W, Cin, Cout, colstats):
    lib = _lib.load()
    if x.numel() != B * H * W * Cin or out.numel() != B * same_out(H) * same_out(W) * Cout or \
            w.numel() < 9 * Cin * Cout or x.dtype != w.dtype:
        raise RuntimeError("athena_amd.conv3x3s2_fwd: bad operands")
    if colstats is not None and (colstats.dtype != torch.float64 or colstats.numel() < 2 * Cout):
        raise RuntimeError("athena_amd.conv3x3s2_fwd: colstats must be fp64 [2*Cout]")
    _lib.check(lib.athena_conv3x3s2_fwd(_ptr(x), _ptr(w), w_layout, _ptr(out), B, H, W, Cin, Cout, dt(x),
                                        _ptr(colstats), _stream()), "athena_conv3x3s2_fwd")


def conv3x3s2_dgrad(dout, w_hwio, din, B, H, W, Cin, Cout, relu6_out=None):
    lib = _lib.load()
    if relu6_out is not None and (relu6_out.numel() != din.numel() or relu6_out.dtype != din.dtype):
        raise RuntimeError("athena_amd.conv3x3s2_dgrad: relu6_out must match din")
    if din.numel() != B * H * W * Cin or dout.numel() != B * same_out(H) * same_out(W) * Cout or \
            w_hwio.numel() < 9 * Cin * Cout or dout.dtype != w_hwio.dtype or din.dtype != dout.dtype:
        raise RuntimeError("athena_amd.conv3x3s2_dgrad: bad operands")
    _lib.check(lib.athena_conv3x3s2_dgrad(_ptr(dout), _ptr(w_hwio), _ptr(din), B, H, W, Cin, Cout, dt(dout),
                                          _ptr(relu6_out), _stream()), "athena_conv3x3s2_dgrad")


def conv3x3s2_wgrad(x, dout, dw, B, H, W, Cin, Cout):
    lib = _lib.load()
    if x.numel() != B * H * W * Cin or dout.numel() != B * same_out(H) * same_out(W) * Cout or \
            dw.numel() != 9 * Cin * Cout or dw.dtype != torch.float32 or x.dtype != dout.dtype:
        raise RuntimeError("athena_amd.conv3x3s2_wgrad: bad operands")
    ws = splitk_workspace(x.device)
    _lib.check(lib.athena_conv3x3s2_wgrad(_ptr(x), _ptr(dout), _ptr(dw), B, H, W, Cin, Cout, dt(x), ws.data_ptr(),
                                          ws.numel(), _stream()), "athena_conv3x3s2_wgrad")


CONV1_MOMENTS = 90          # tap sums and tap products the backward pass reads


def conv1_moments_len():
    """Length (fp64 elements) of the ``moments`` buffer of ``conv1_bn_stats``: the 90 moments
    followed by the scratch of the reduction."""
    return int(_lib.load().athena_conv1_moments_len())


def conv1_bn_stats(x, w_hwio, B, H, W, Cout, moments, colstats):
    """Input moments and closed-form pre-activation statistics of the one-channel first layer."""
    lib = _lib.load()
    if x.dtype != torch.float32 or w_hwio.dtype != torch.float32 or x.numel() != B * H * W or \
            w_hwio.numel() != 9 * Cout or moments.dtype != torch.float64 or \
            moments.numel() < conv1_moments_len() or colstats.dtype != torch.float64 or colstats.numel() < 2 * Cout:
        raise RuntimeError("athena_amd.conv1_bn_stats: bad operands")
    _lib.check(lib.athena_conv1_bn_stats(_ptr(x), _ptr(w_hwio), B, H, W, Cout, _ptr(moments), _ptr(colstats),
                                         _stream()), "athena_conv1_bn_stats")


def conv1_bn_relu6_fwd(x, w_hwio, s0, s1, gamma, beta, eps, infer, B, H, W, Cout, out):
    lib = _lib.load()
    if x.dtype != torch.float32 or w_hwio.dtype != torch.float32 or x.numel() != B * H * W or \
            w_hwio.numel() != 9 * Cout or out.numel() != B * same_out(H) * same_out(W) * Cout or \
            s0.numel() < (Cout if infer else 2 * Cout):
        raise RuntimeError("athena_amd.conv1_bn_relu6_fwd: bad operands")
    _lib.check(lib.athena_conv1_bn_relu6_fwd(_ptr(x), _ptr(w_hwio), _ptr(s0), _ptr(s1), _ptr(gamma), _ptr(beta), eps,
                                             int(infer), B, H, W, Cout, dt(out), _ptr(out), _stream()),
               "athena_conv1_bn_relu6_fwd")


def conv1_bn_bwd(x, g, w_hwio, moments, mean_rstd, gamma, B, H, W, Cout, dw, dgamma, dbeta, relu6_out=None, beta=None):
    """``relu6_out``: the gate is applied here; with ``beta`` too it is worked out again instead of read."""
    lib = _lib.load()
    if beta is not None and (beta.dtype != torch.float32 or beta.numel() < Cout):
        raise RuntimeError("athena_amd.conv1_bn_bwd: beta must be fp32 [Cout]")
    if relu6_out is not None and (relu6_out.numel() != g.numel() or relu6_out.dtype != g.dtype):
        raise RuntimeError("athena_amd.conv1_bn_bwd: relu6_out must match g")
    if x.dtype != torch.float32 or x.numel() != B * H * W or g.numel() != B * same_out(H) * same_out(W) * Cout or \
            dw.numel() != 9 * Cout or dw.dtype != torch.float32 or moments.numel() < CONV1_MOMENTS or \
            mean_rstd.numel() < 2 * Cout or dgamma.numel() < Cout or dbeta.numel() < Cout:
        raise RuntimeError("athena_amd.conv1_bn_bwd: bad operands")
    ws = splitk_workspace(x.device)
    _lib.check(lib.athena_conv1_bn_bwd(_ptr(x), _ptr(g), _ptr(relu6_out), _ptr(w_hwio), _ptr(moments), _ptr(mean_rstd), _ptr(gamma), _ptr(beta), B,
                                       H, W, Cout, dt(g), ws.data_ptr(), ws.numel(), _ptr(dw), _ptr(dgamma),
                                       _ptr(dbeta), _stream()), "athena_conv1_bn_bwd")


def conv_small_cin_fwd(x, w_hwio, out, B, H, W, Cin, Cout, colstats):
    lib = _lib.load()
    if x.dtype != torch.float32 or w_hwio.dtype != torch.float32 or x.numel() != B * H * W * Cin or \
            out.numel() != B * same_out(H) * same_out(W) * Cout or w_hwio.numel() != 9 * Cin * Cout:
        raise RuntimeError("athena_amd.conv_small_cin_fwd: bad operands")
    _lib.check(lib.athena_conv3x3s2_small_cin_fwd(_ptr(x), _ptr(w_hwio), _ptr(out), B, H, W, Cin, Cout, dt(out),
                                                  _ptr(colstats), _stream()), "athena_conv3x3s2_small_cin_fwd")


def conv_small_cin_wgrad(x, dout, dw, B, H, W, Cin, Cout):
    lib = _lib.load()
    if x.dtype != torch.float32 or dw.dtype != torch.float32 or x.numel() != B * H * W * Cin or \
            dout.numel() != B * same_out(H) * same_out(W) * Cout or dw.numel() != 9 * Cin * Cout:
        raise RuntimeError("athena_amd.conv_small_cin_wgrad: bad operands")
    _lib.check(lib.athena_conv3x3s2_small_cin_wgrad(_ptr(x), _ptr(dout), _ptr(dw), B, H, W, Cin, Cout, dt(dout),
                                                    _stream()), "athena_conv3x3s2_small_cin_wgrad")


def bn_finalize(colstats, rows, C, eps, momentum, mean_rstd, moving_mean, moving_var):
    lib = _lib.load()
    _lib.check(lib.athena_bn_finalize(_ptr(colstats), rows, C, eps, momentum, _ptr(mean_rstd), _ptr(moving_mean),
                                      _ptr(moving_var), _stream()), "athena_bn_finalize")


def bn_relu6_apply(x, mean_rstd, gamma, beta, rows, C, y):
    lib = _lib.load()
    if x.numel() != rows * C or y.numel() != rows * C or x.dtype != y.dtype:
        raise RuntimeError("athena_amd.bn_relu6_apply: bad operands")
    _lib.check(lib.athena_bn_relu6_apply(_ptr(x), _ptr(mean_rstd), _ptr(gamma), _ptr(beta), rows, C, dt(x),
                                         _ptr(y), _stream()), "athena_bn_relu6_apply")


def bn_relu6_infer(x, moving_mean, moving_var, gamma, beta, eps, rows, C, y):
    lib = _lib.load()
    if x.numel() != rows * C or y.numel() != rows * C or x.dtype != y.dtype:
        raise RuntimeError("athena_amd.bn_relu6_infer: bad operands")
    _lib.check(lib.athena_bn_relu6_infer(_ptr(x), _ptr(moving_mean), _ptr(moving_var), _ptr(gamma), _ptr(beta),
                                         eps, rows, C, dt(x), _ptr(y), _stream()), "athena_bn_relu6_infer")


def bn_relu6_bwd_scratch(rows, C, device):
    """Scratch tensor (uint8) for ``bn_relu6_bwd``: fp64 totals and the per-workgroup partial sums."""
    n = int(_lib.load().athena_bn_relu6_bwd_scratch_bytes(rows, C))
    return torch.empty(n, dtype=torch.uint8, device=device)


def bn_relu6_bwd(dy, x, mean_rstd, gamma, beta, rows, C, scratch, dx, dgamma, dbeta):
    lib = _lib.load()
    if any(t.numel() != rows * C for t in (dy, x, dx)):
        raise RuntimeError("athena_amd.bn_relu6_bwd: bad operands")
    _lib.check(lib.athena_bn_relu6_bwd(_ptr(dy), _ptr(x), _ptr(mean_rstd), _ptr(gamma), _ptr(beta), rows, C, dt(x),
                                       _ptr(scratch), scratch.numel() * scratch.element_size(), _ptr(dx),
                                       _ptr(dgamma), _ptr(dbeta), _stream()),
               "athena_bn_relu6_bwd")


def bn_colstats(x, rows, C, colstats):
    """{sum, sumsq} per column of x [rows, C] into the fp64 ``colstats`` [2C]."""
    if x.numel() != rows * C or colstats.dtype != torch.float64 or colstats.numel() < 2 * C:
        raise RuntimeError("athena_amd.bn_colstats: bad operands")
    _lib.check(_lib.load().athena_bn_colstats(_ptr(x), rows, C, dt(x), _ptr(colstats), _stream()), "athena_bn_colstats")


def bn_apply(x, mean_rstd, gamma, beta, rows, C, y):
    if x.numel() != rows * C or y.numel() != rows * C or x.dtype != y.dtype:
        raise RuntimeError("athena_amd.bn_apply: bad operands")
    _lib.check(_lib.load().athena_bn_apply(_ptr(x), _ptr(mean_rstd), _ptr(gamma), _ptr(beta), rows, C, dt(x), _ptr(y),
                                           _stream()), "athena_bn_apply")


def bn_infer(x, moving_mean, moving_var, gamma, beta, eps, rows, C, y):
    if x.numel() != rows * C or y.numel() != rows * C or x.dtype != y.dtype:
        raise RuntimeError("athena_amd.bn_infer: bad operands")
    _lib.check(_lib.load().athena_bn_infer(_ptr(x), _ptr(moving_mean), _ptr(moving_var), _ptr(gamma), _ptr(beta), eps,
                                           rows, C, dt(x), _ptr(y), _stream()), "athena_bn_infer")


def bn_bwd(dy, x, mean_rstd, gamma, beta, rows, C, scratch, dx, dgamma, dbeta):
    if any(t.numel() != rows * C for t in (dy, x, dx)):
        raise RuntimeError("athena_amd.bn_bwd: bad operands")
    _lib.check(_lib.load().athena_bn_bwd(_ptr(dy), _ptr(x), _ptr(mean_rstd), _ptr(gamma), _ptr(beta), rows, C, dt(x),
                                         _ptr(scratch), scratch.numel() * scratch.element_size(), _ptr(dx),
                                         _ptr(dgamma), _ptr(dbeta), _stream()), "athena_bn_bwd")


# ------------------------------------------------------------------------------------------ Conv2D, any kernel
def conv2d_out_shape(H, W, KH, KW, sh, sw):
    """(Ho, Wo) of a "same"-padded convolution: ceil(H / sh), ceil(W / sw)."""
    ho, wo = ctypes.c_int(0), ctypes.c_int(0)
    _lib.check(_lib.load().athena_conv2d_out_shape(H, W, KH, KW, sh, sw, ctypes.byref(ho), ctypes.byref(wo)),
               "athena_conv2d_out_shape")
    return ho.value, wo.value


def _conv2d_sizes(B, H, W, Cin, Cout, KH, KW, sh, sw):
    Ho, Wo = -(-H // sh), -(-W // sw)
    return B * H * W * Cin, B * Ho * Wo * Cout, KH * KW * Cin * Cout


def conv2d_fwd(x, w_hwio, out, B, H, W, Cin, Cout, KH, KW, sh, sw, colstats=None):
    n_in, n_out, n_w = _conv2d_sizes(B, H, W, Cin, Cout, KH, KW, sh, sw)
    if x.numel() != n_in or out.numel() != n_out or w_hwio.numel() < n_w or x.dtype != w_hwio.dtype or \
            out.dtype != x.dtype:
        raise RuntimeError("athena_amd.conv2d_fwd: bad operands")
    if colstats is not None and (colstats.dtype != torch.float64 or colstats.numel() < 2 * Cout):
        raise RuntimeError("athena_amd.conv2d_fwd: colstats must be fp64 [2*Cout]")
    _lib.check(_lib.load().athena_conv2d_fwd(_ptr(x), _ptr(w_hwio), _ptr(out), B, H, W, Cin, Cout, KH, KW, sh, sw,
                                             dt(x), _ptr(colstats), _stream()), "athena_conv2d_fwd")


def conv2d_dgrad(dout, w_hwio, din, B, H, W, Cin, Cout, KH, KW, sh, sw, relu6_out=None):
    n_in, n_out, n_w = _conv2d_sizes(B, H, W, Cin, Cout, KH, KW, sh, sw)
    if din.numel() != n_in or dout.numel() != n_out or w_hwio.numel() < n_w or dout.dtype != w_hwio.dtype or \
            din.dtype != dout.dtype:
        raise RuntimeError("athena_amd.conv2d_dgrad: bad operands")
    if relu6_out is not None and (relu6_out.numel() != n_in or relu6_out.dtype != din.dtype):
        raise RuntimeError("athena_amd.conv2d_dgrad: relu6_out must match din")
    _lib.check(_lib.load().athena_conv2d_dgrad(_ptr(dout), _ptr(w_hwio), _ptr(din), B, H, W, Cin, Cout, KH, KW, sh, sw,
                                               dt(dout), _ptr(relu6_out), _stream()), "athena_conv2d_dgrad")


def conv2d_wgrad(x, dout, dw, B, H, W, Cin, Cout, KH, KW, sh, sw):
    n_in, n_out, n_w = _conv2d_sizes(B, H, W, Cin, Cout, KH, KW, sh, sw)
    if x.numel() != n_in or dout.numel() != n_out or dw.numel() != n_w or dw.dtype != torch.float32 or \
            x.dtype != dout.dtype:
        raise RuntimeError("athena_amd.conv2d_wgrad: bad operands")
    lib = _lib.load()
    need = int(lib.athena_conv2d_wgrad_workspace_bytes(B, H, W, Cin, Cout, KH, KW, sh, sw, dt(x)))
    ws = splitk_workspace(x.device)
    if ws.numel() * ws.element_size() < need:
        ws = torch.empty(need, dtype=torch.uint8, device=x.device)
    _lib.check(lib.athena_conv2d_wgrad(_ptr(x), _ptr(dout), _ptr(dw), B, H, W, Cin, Cout, KH, KW, sh, sw, dt(x),
                                       ws.data_ptr(), ws.numel() * ws.element_size(), _stream()),
               "athena_conv2d_wgrad")


def im2col(x, col, ldcol, B, H, W, Cin, KH, KW, sh, sw):
    """col [B*Ho*Wo, ldcol] (zero padding columns beyond KH*KW*Cin) from the NHWC tensor ``x``."""
    Ho, Wo = -(-H // sh), -(-W // sw)
    if x.numel() != B * H * W * Cin or col.numel() != B * Ho * Wo * ldcol or ldcol < KH * KW * Cin:
        raise RuntimeError("athena_amd.im2col: bad operands")
    _lib.check(_lib.load().athena_im2col(_ptr(x), dt(x), _ptr(col), dt(col), ldcol, B, H, W, Cin, KH, KW, sh, sw,
                                         _stream()), "athena_im2col")


# ------------------------------------------------------------------------------------------ recurrent layers
RNN_GRU, RNN_LSTM = 0, 1


def rnn_workspace(cell, B, H, device):
    n = int(_lib.load().athena_rnn_workspace_bytes(cell, B, H))
    return torch.empty(n, dtype=torch.uint8, device=device)


def rnn_fwd(cell, xw, u, b_rec, hs_ext, cs_ext, y, gates, rh, B, T, H, ws, u_t=None):
    G = 4 if cell == RNN_LSTM else 3
    if xw.numel() != B * T * G * H or u.numel() < H * G * H or hs_ext.numel() != B * (T + 1) * H or \
            y.numel() != B * T * H or gates.numel() != B * T * G * H or \
            any(t.dtype != xw.dtype for t in (u, hs_ext, y, gates)):
        raise RuntimeError("athena_amd.rnn_fwd: bad operands")
    if cell == RNN_LSTM and (cs_ext is None or cs_ext.dtype != torch.float32 or cs_ext.numel() != B * (T + 1) * H):
        raise RuntimeError("athena_amd.rnn_fwd: cs_ext must be fp32 [B, T+1, H]")
    if cell == RNN_GRU and (rh is None or rh.numel() != B * T * H or rh.dtype != xw.dtype):
        raise RuntimeError("athena_amd.rnn_fwd: rh must be [B, T, H]")
    if b_rec is not None and (b_rec.dtype != torch.float32 or b_rec.numel() != G * H):
        raise RuntimeError("athena_amd.rnn_fwd: b_rec must be fp32 [G*H]")
    if u_t is not None and (u_t.dtype != xw.dtype or u_t.numel() < G * H * H):
        raise RuntimeError("athena_amd.rnn_fwd: u_t must be the transposed recurrent kernel [G*H, H]")
    _lib.check(_lib.load().athena_rnn_fwd(cell, _ptr(xw), _ptr(u), _ptr(u_t), _ptr(b_rec), _ptr(hs_ext), _ptr(cs_ext), _ptr(y),
                                          _ptr(gates), _ptr(rh), B, T, H, dt(xw), ws.data_ptr(),
                                          ws.numel() * ws.element_size(), _stream()), "athena_rnn_fwd")


def rnn_bwd(cell, dy, u, hs_ext, cs_ext, gates, rh, dxw, dhu_ext, B, T, H, ws):
    G = 4 if cell == RNN_LSTM else 3
    if dy.numel() != B * T * H or u.numel() < H * G * H or hs_ext.numel() != B * (T + 1) * H or \
            gates.numel() != B * T * G * H or dxw.numel() != B * T * G * H or dhu_ext.numel() != B * (T + 1) * G * H or \
            any(t.dtype != dy.dtype for t in (u, hs_ext, gates, dxw, dhu_ext)):
        raise RuntimeError("athena_amd.rnn_bwd: bad operands")
    _lib.check(_lib.load().athena_rnn_bwd(cell, _ptr(dy), _ptr(u), _ptr(hs_ext), _ptr(cs_ext), _ptr(gates), _ptr(rh),
                                          _ptr(dxw), _ptr(dhu_ext), B, T, H, dt(dy), ws.data_ptr(),
                                          ws.numel() * ws.element_size(), _stream()), "athena_rnn_bwd")


# ------------------------------------------------------------------------------------------ PE / embedding
def add_pe_dropout(x, pe, B, T, d, xscale, drop_p, rng_state, site, y):
    lib = _lib.load()
    if x.numel() != B * T * d or y.numel() != B * T * d or pe.numel() < T * d or pe.dtype != torch.float32:
        raise RuntimeError("athena_amd.add_pe_dropout: bad operands (T=%d exceeds the positional table?)" % T)
    _lib.check(lib.athena_add_pe_dropout(_ptr(x), _ptr(pe), B, T, d, dt(x), xscale, drop_p, _ptr(rng_state), site,
                                         _ptr(y), _stream()), "athena_add_pe_dropout")


def dropout_bwd(dy, xscale, drop_p, rng_state, site, relu6_out, dx):
    lib = _lib.load()
    if dx.numel() != dy.numel() or (relu6_out is not None and relu6_out.numel() != dy.numel()):
        raise RuntimeError("athena_amd.dropout_bwd: size mismatch")
    _lib.check(lib.athena_dropout_bwd(_ptr(dy), dy.numel(), dt(dy), xscale, drop_p, _ptr(rng_state), site,
                                      _ptr(relu6_out), _ptr(dx), _stream()), "athena_dropout_bwd")


def embed_fwd(table, ids, pe, B, L, d, V, xscale, drop_p, rng_state, site, y):
    lib = _lib.load()
    if table.numel() != V * d or ids.numel() != B * L or ids.dtype != torch.int32 or pe.numel() < L * d:
        raise RuntimeError("athena_amd.embed_fwd: bad operands")
    _lib.check(lib.athena_embed_fwd(_ptr(table), _ptr(ids), _ptr(pe), B, L, d, V, dt(y), xscale, drop_p,
                                    _ptr(rng_state), site, _ptr(y), _stream()), "athena_embed_fwd")


def embed_bwd(dy, ids, B, L, d, V, xscale, drop_p, rng_state, site, dtable):
    """dtable [V, d] = the gradient of the embedding table: every row is written (no zeroing before)."""
    lib = _lib.load()
    if dtable.numel() != V * d or ids.numel() != B * L or dy.numel() != B * L * d:
        raise RuntimeError("athena_amd.embed_bwd: bad operands")
    _lib.check(lib.athena_embed_bwd(_ptr(dy), _ptr(ids), B, L, d, V, dt(dy), xscale, drop_p, _ptr(rng_state),
                                    site, _ptr(dtable), _stream()), "athena_embed_bwd")


# ------------------------------------------------------------------------------------------ losses
def ctc_workspace_bytes(B, T, U):
    return int(_lib.load().athena_ctc_workspace_bytes(B, T, U))


def ctc_loss_fwd(logits, ldl, labels, label_len, logit_len, B, T, V, U, blank, loss, workspace, argmax=None):
    """``argmax`` (optional int32 [B*T]) receives the first arg-max class of every row inside logit_len."""
    lib = _lib.load()
    if argmax is not None and (argmax.dtype != torch.int32 or argmax.numel() < B * T or not argmax.is_contiguous()):
        raise RuntimeError("athena_amd.ctc_loss: argmax must be contiguous int32 [B*T]")
    for t_ in (labels, label_len, logit_len):
        if t_.dtype != torch.int32 or not t_.is_contiguous():
            raise RuntimeError("athena_amd.ctc_loss: labels and lengths must be contiguous int32")
    if labels.numel() != B * U or label_len.numel() != B or logit_len.numel() != B or loss.numel() != B:
        raise RuntimeError("athena_amd.ctc_loss: bad label shapes")
    _lib.check(lib.athena_ctc_loss_fwd(_ptr(logits), dt(logits), ldl, _ptr(labels), _ptr(label_len),
                                       _ptr(logit_len), B, T, V, U, blank, _ptr(loss), _ptr(argmax), _ptr(workspace),
                                       workspace.numel() * workspace.element_size(), _stream()),
               "athena_ctc_loss_fwd")


def ctc_loss_fwd_bwd(logits, ldl, labels, label_len, logit_len, B, T, V, U, blank, loss, workspace, grad_scale,
                     grad, argmax=None):
    """Loss and gradient in one pass over the logits: ``grad`` [B,T,ldl] = grad_scale * (softmax - occupancy)."""
    lib = _lib.load()
    if argmax is not None and (argmax.dtype != torch.int32 or argmax.numel() < B * T or not argmax.is_contiguous()):
        raise RuntimeError("athena_amd.ctc_loss: argmax must be contiguous int32 [B*T]")
    for t_ in (labels, label_len, logit_len):
        if t_.dtype != torch.int32 or not t_.is_contiguous():
            raise RuntimeError("athena_amd.ctc_loss: labels and lengths must be contiguous int32")
    if labels.numel() != B * U or label_len.numel() != B or logit_len.numel() != B or loss.numel() != B:
        raise RuntimeError("athena_amd.ctc_loss: bad label shapes")
    if grad.numel() != B * T * ldl or not grad.is_contiguous():
        raise RuntimeError("athena_amd.ctc_loss: grad must be contiguous [B,T,ldl]")
    _lib.check(lib.athena_ctc_loss_fwd_bwd(_ptr(logits), dt(logits), ldl, _ptr(labels), _ptr(label_len),
                                           _ptr(logit_len), B, T, V, U, blank, _ptr(loss), _ptr(argmax),
                                           float(grad_scale), _ptr(grad), dt(grad), _ptr(workspace),
                                           workspace.numel() * workspace.element_size(), _stream()),
               "athena_ctc_loss_fwd_bwd")


def rescale_unless(x, upstream, expected):
    """x *= upstream / expected on the device, a no-op launch when the two are equal."""
    lib = _lib.load()
    if upstream.dtype != torch.float32 or upstream.numel() != 1 or not x.is_contiguous() or x.numel() % 4:
        raise RuntimeError("athena_amd.rescale_unless: bad operands")
    _lib.check(lib.athena_rescale_unless(_ptr(x), x.numel(), dt(x), _ptr(upstream), float(expected), _stream()),
               "athena_rescale_unless")


def ctc_loss_bwd(logits, ldl, labels, label_len, logit_len, B, T, V, U, blank, grad_scale, host_scale, grad,
                 workspace):
    lib = _lib.load()
    _lib.check(lib.athena_ctc_loss_bwd(_ptr(logits), dt(logits), ldl, _ptr(labels), _ptr(label_len),
                                       _ptr(logit_len), B, T, V, U, blank, _ptr(grad_scale), host_scale,
                                       _ptr(grad), dt(grad), _ptr(workspace),
                                       workspace.numel() * workspace.element_size(), _stream()),
               "athena_ctc_loss_bwd")


def ce_loss_fwd(logits, ldl, targets, rows, V, ls, row_loss, lse):
    lib = _lib.load()
    if targets.dtype != torch.int32 or targets.numel() != rows:
        raise RuntimeError("athena_amd.ce_loss: targets must be int32 [rows]")
    _lib.check(lib.athena_ce_loss_fwd(_ptr(logits), dt(logits), ldl, _ptr(targets), rows, V, ls, _ptr(row_loss),
                                      _ptr(lse), _stream()), "athena_ce_loss_fwd")


def ce_loss_bwd(logits, ldl, targets, rows, V, ls, lse, grad_scale, host_scale, grad):
    lib = _lib.load()
    _lib.check(lib.athena_ce_loss_bwd(_ptr(logits), dt(logits), ldl, _ptr(targets), rows, V, ls, _ptr(lse),
                                      _ptr(grad_scale), host_scale, _ptr(grad), dt(grad), _stream()),
               "athena_ce_loss_bwd")


def mpc_loss_fwd(logits, ldl, target, masked, logit_len, B, Tp, N, row_loss):
    lib = _lib.load()
    for t_ in (logits, target, masked, row_loss):
        if t_.dtype != torch.float32:
            raise TypeError("athena_amd.mpc_loss: fp32 tensors expected")
    if target.numel() < B * Tp * N or masked.numel() < B * Tp * N or _extent(logits) < (B * Tp - 1) * ldl + N or \
            logit_len.dtype != torch.int32 or logit_len.numel() < B or row_loss.numel() < B * Tp:
        raise RuntimeError("athena_amd.mpc_loss_fwd: operand too small for B=%d Tp=%d N=%d" % (B, Tp, N))
    _lib.check(lib.athena_mpc_loss_fwd(_ptr(logits), ldl, _ptr(target), _ptr(masked), _ptr(logit_len), B, Tp, N,
                                       _ptr(row_loss), _stream()), "athena_mpc_loss_fwd")


def mpc_loss_bwd(logits, ldl, target, masked, logit_len, B, Tp, N, grad_scale, host_scale, grad):
    lib = _lib.load()
    if grad.numel() < B * Tp * ldl or grad_scale.dtype != torch.float32:
        raise RuntimeError("athena_amd.mpc_loss_bwd: bad operands")
    _lib.check(lib.athena_mpc_loss_bwd(_ptr(logits), ldl, _ptr(target), _ptr(masked), _ptr(logit_len), B, Tp, N,
                                       _ptr(grad_scale), host_scale, _ptr(grad), dt(grad), _stream()),
               "athena_mpc_loss_bwd")


def group_sum(x, ngroups, group, scale, out):
    lib = _lib.load()
    if x.dtype != torch.float32 or out.dtype != torch.float32 or x.numel() < ngroups * group:
        raise RuntimeError("athena_amd.group_sum: bad operands")
    _lib.check(lib.athena_group_sum(_ptr(x), ngroups, group, scale, _ptr(out), _stream()), "athena_group_sum")


def prepare_labels(labels, label_len, input_len, Tp, sos, eos):
    """(y0, tgt, y_mask, logit_len, x_mask) of a batch in one launch; see ``athena_prepare_labels``."""
    lib = _lib.load()
    B, U = labels.shape
    for t_ in (labels, label_len, input_len):
        if t_.dtype != torch.int32 or not t_.is_contiguous():
            raise RuntimeError("athena_amd.prepare_labels: labels and lengths must be contiguous int32")
    dev = labels.device
    y0 = torch.empty((B, U + 1), dtype=torch.int32, device=dev)
    tgt = torch.empty((B, U + 1), dtype=torch.int32, device=dev)
    y_mask = torch.empty((B, U + 1), dtype=torch.uint8, device=dev)
    logit_len = torch.empty(B, dtype=torch.int32, device=dev)
    x_mask = torch.empty((B, Tp), dtype=torch.uint8, device=dev)
    _lib.check(lib.athena_prepare_labels(_ptr(labels), _ptr(label_len), _ptr(input_len), B, U, Tp, sos, eos, _ptr(y0),
                                         _ptr(tgt), _ptr(y_mask), _ptr(logit_len), _ptr(x_mask), _stream()),
               "athena_prepare_labels")
    return y0, tgt, y_mask, logit_len, x_mask


def argmax_rows(logits, ldl, rows, V, out):
    lib = _lib.load()
    if out.dtype != torch.int32 or out.numel() < rows:
        raise RuntimeError("athena_amd.argmax_rows: out must be int32 [rows]")
    _lib.check(lib.athena_argmax_rows(_ptr(logits), dt(logits), ldl, rows, V, _ptr(out), _stream()),
               "athena_argmax_rows")


def seq_errors(ids, hyp_len, labels, mode, special, counts=None, per_utt=None):
    """Edit-distance scoring of arg-max ids [B, L] against the non-zero labels [B, U] on the device
    (mode 0: greedy CTC collapse with blank ``special`` inside ``hyp_len`` frames; mode 1: cut at eos
    ``special``, zeros dropped).  ``counts`` int64 [2] accumulates (errors, labels)."""
    lib = _lib.load()
    B, L = ids.shape
    U = labels.shape[1]
    for t, name in ((ids, "ids"), (labels, "labels"), (hyp_len, "hyp_len"), (per_utt, "per_utt")):
        if t is not None and (t.dtype != torch.int32 or not t.is_contiguous()):
            raise RuntimeError("athena_amd.seq_errors: %s must be contiguous int32" % name)
    if counts is not None and (counts.dtype != torch.int64 or counts.numel() < 2):
        raise RuntimeError("athena_amd.seq_errors: counts must be int64 [2]")
    if labels.shape[0] != B or (hyp_len is not None and hyp_len.numel() < B) or \
            (per_utt is not None and per_utt.numel() < 2 * B):
        raise RuntimeError("athena_amd.seq_errors: operand shapes do not match the batch of %d" % B)
    _lib.check(lib.athena_seq_errors(_ptr(ids), L, _ptr(hyp_len), _ptr(labels), B, L, U, mode, special, _ptr(per_utt),
                                     _ptr(counts), _stream()), "athena_seq_errors")


# ------------------------------------------------------------------------------------------ optimizer
def clip_adam_step(params, grads, m, v, seg_offsets, nseg, norms, step, cfg, lr_out):
    lib = _lib.load()
    n = params.numel()
    if grads.numel() != n or m.numel() != n or v.numel() != n or seg_offsets.dtype != torch.int64 or \
            step.dtype != torch.int64 or seg_offsets.numel() != nseg + 1 or norms.numel() < nseg:
        raise RuntimeError("athena_amd.clip_adam_step: bad operands")
    _lib.check(lib.athena_clip_adam_step(_ptr(params), _ptr(grads), _ptr(m), _ptr(v), n, _ptr(seg_offsets), nseg,
                                         _ptr(norms), _ptr(step), ctypes.byref(cfg), _ptr(lr_out), _stream()),
               "athena_clip_adam_step")


def refresh_shadows(params, shadow, table, nmat, tile_prefix, total_tiles):
    lib = _lib.load()
    _lib.check(lib.athena_refresh_shadows(_ptr(params), _ptr(shadow), _ptr(table), nmat, _ptr(tile_prefix),
                                          total_tiles, _stream()), "athena_refresh_shadows")


def advance_rng(rng_state):
    _lib.check(_lib.load().athena_advance_rng(_ptr(rng_state), _stream()), "athena_advance_rng")


def cast(src, dst):
    if src.numel() != dst.numel():
        raise RuntimeError("athena_amd.cast: size mismatch")
    _lib.check(_lib.load().athena_cast(_ptr(src), dt(src), _ptr(dst), dt(dst), src.numel(), _stream()),
               "athena_cast")


COPY_MANY_MAX = 8


def copy_many(pairs):
    """``dst.copy_(src)`` for every (src, dst) of ``pairs`` -- contiguous tensors of equal dtype and
    size, each on the device or in pinned host memory -- as one launch per eight pairs."""
    import ctypes
    pairs = [(s, d) for s, d in pairs if s.numel() > 0]
    for s, d in pairs:
        if s.dtype != d.dtype or s.numel() != d.numel() or not s.is_contiguous() or not d.is_contiguous():
            raise RuntimeError("athena_amd.copy_many: tensors of a pair must be contiguous and alike")
        if not (s.is_cuda or s.is_pinned()) or not (d.is_cuda or d.is_pinned()):
            raise RuntimeError("athena_amd.copy_many: device or pinned host tensors only")
    lib = _lib.load()
    for i in range(0, len(pairs), COPY_MANY_MAX):
        part = pairs[i:i + COPY_MANY_MAX]
        n = len(part)
        src = (ctypes.c_void_p * n)(*[s.data_ptr() for s, _ in part])
        dst = (ctypes.c_void_p * n)(*[d.data_ptr() for _, d in part])
        nbytes = (ctypes.c_long * n)(*[s.numel() * s.element_size() for s, _ in part])
        _lib.check(lib.athena_copy_many(src, dst, nbytes, n, _stream()), "athena_copy_many")


# ------------------------------------------------------------------------------------------ bf16 gradient hand-over
# autograd casts a gradient to the dtype of the tensor it belongs to, so a loss kernel cannot hand a
# bf16 gradient for fp32 logits back through it.  Inside a solver step (``bf16_grad_handover``), when
# the producer of the logits (a vocabulary projection running in bf16) announces that it consumes
# bf16, the loss writes its gradient in bf16 into a padded buffer of its own, registers it here and
# gives autograd a one-element fp32 stand-in expanded to the logits' shape; the projection's
# backward pass takes the real buffer back out.  The stand-in is NOT the gradient of the logits, so
# the hand-over is off wherever user code may look at that gradient (plain ``loss.backward()`` /
# ``torch.autograd.grad`` outside the solver keep the fp32 gradient tensor).
_BF16_GRADS = {}
_HANDOVER_DEPTH = 0


class bf16_grad_handover:
    """Context of a solver's training step: the loss functions may hand bf16 gradients to the vocabulary
    projections (nothing else looks at the gradient of the logits), and the backward pass starts from
    ``total_loss.backward()``, i.e. from a gradient of exactly 1 at the total loss."""

    def __enter__(self):
        global _HANDOVER_DEPTH
        _HANDOVER_DEPTH += 1
        return self

    def __exit__(self, exc_type, exc, tb):
        global _HANDOVER_DEPTH
        _HANDOVER_DEPTH -= 1
        return False


def root_gradient_is_one():
    """True inside a solver step, where the factor a loss term receives in the backward pass is the
    weight the model gave it in the total loss and nothing else."""
    return _HANDOVER_DEPTH > 0


def bf16_grad_wanted(logits):
    return _HANDOVER_DEPTH > 0 and bool(getattr(logits, "_athena_accepts_bf16_grad", False))


_STANDIN_POOL = {}      # device -> [zeros(64), next index]


def bf16_grad_standin(shape, g16):
    # a second consumer of the logits sees zeros, not noise.  The stand-ins are elements of one
    # zero-filled buffer per device that lives for good (no fill launch per step, and no other tensor
    # can ever have a stand-in's address); an element is not handed out again while its entry exists
    pool = _STANDIN_POOL.get(g16.device)
    if pool is None:
        pool = _STANDIN_POOL[g16.device] = [torch.zeros(64, dtype=torch.float32, device=g16.device), 0]
    for _ in range(64):
        s = pool[0][pool[1]:pool[1] + 1]
        pool[1] = (pool[1] + 1) % 64
        if s.data_ptr() not in _BF16_GRADS:
            break
    else:
        s = torch.zeros(1, dtype=torch.float32, device=g16.device)
    _BF16_GRADS[s.data_ptr()] = (s, g16)
    return s.expand(shape)


def take_bf16_grad(dy):
    """The registered bf16 buffer behind a stand-in; None for an ordinary gradient."""
    if dy.dim() == 0 or any(st != 0 for st in dy.stride()):
        return None
    entry = _BF16_GRADS.pop(dy.data_ptr(), None)
    return None if entry is None else entry[1]


def weighted_sum(terms, weights, out):
    """out[0] = sum_i weights[i] * terms[i][0] (fp32 scalars on the device, host weights), one launch."""
    n = len(terms)
    if n != len(weights) or not 0 < n <= 8 or out.dtype != torch.float32 or out.numel() < 1 or \
            any(t.dtype != torch.float32 or t.numel() != 1 or t.device != out.device for t in terms):
        raise RuntimeError("athena_amd.weighted_sum: 1..8 fp32 scalars on the device of out expected")
    ptrs = (ctypes.c_void_p * n)(*[t.data_ptr() for t in terms])
    w = (ctypes.c_float * n)(*[float(x) for x in weights])
    _lib.check(_lib.load().athena_weighted_sum(ptrs, w, n, _ptr(out), _stream()), "athena_weighted_sum")


_CONST_SCALARS = {}


def const_scalar(device, value):
    """A 0-dim fp32 tensor holding ``value`` that lives for good (one per device and value), or None
    while a stream of this thread is recording and the tensor does not exist yet: memory allocated
    during a recording belongs to the graph and must not outlive it."""
    key = (str(device), float(value))
    t = _CONST_SCALARS.get(key)
    if t is None:
        if torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():
            return None
        t = _CONST_SCALARS[key] = torch.full((), float(value), dtype=torch.float32, device=device)
    return t


def axpby(a, x, b, y):
    if x.numel() != y.numel() or x.dtype != y.dtype:
        raise RuntimeError("athena_amd.axpby: operand mismatch")
    _lib.check(_lib.load().athena_axpby(a, _ptr(x), b, _ptr(y), x.numel(), dt(x), _stream()), "athena_axpby")


# ------------------------------------------------------------------------------------------ decoding: cache, logits
# A decoding step issues these calls many times on little work, so the checks look at every property once and the
# arguments travel in one packed descriptor (see _lib).
KV8_WIDTHS = (32, 64, 128)
KV8_BLOCKS = (16, 32, 64, 128)
_CODES = {torch.float32: F32, torch.bfloat16: BF16}
_I32, _I8, _FP32 = torch.int32, torch.int8, torch.float32


def _refuse(name, what, *args):
    raise RuntimeError("athena_amd.%s: %s" % (name, what % args if args else what))


def _here(name, *tensors):
    """The raw current stream, when every given tensor lives on the current GPU (kernels go to its stream)."""
    here = torch.cuda.current_device()
    for t in tensors:
        if t is not None and t.get_device() != here:
            _refuse(name, "tensors must live on the current GPU, cuda:%d (got %s)", here, t.device)
    return torch._C._cuda_getCurrentRawStream(here)


def _code(name, t):
    c = _CODES.get(t.dtype)
    if c is None:
        raise TypeError("athena_amd.%s: unsupported dtype %s" % (name, t.dtype))
    return c


def _int_vector(name, what, t, n):
    if t.dtype is not _I32 or t.numel() < n or not t.is_contiguous():
        _refuse(name, "%s must be contiguous int32 of %d elements", what, n)


def _tables(name, tables, B):
    """(leading dimension, width) of a table of blocks."""
    shape, stride = tables.shape, tables.stride()
    if tables.dtype is not _I32 or len(shape) != 2 or shape[0] != B or shape[1] < 1 or (stride[1] != 1 and shape[1] > 1):
        _refuse(name, "tables must be int32 [%d, blocks] with rows in one piece", B)
    return stride[0], shape[1]


def kv8_width(head_size):
    """Columns that a head of ``head_size`` takes in the 8-bit cache."""
    for w in KV8_WIDTHS:
        if head_size <= w:
            return w
    raise NotImplementedError("athena_amd: head size %d exceeds the %d columns of the 8-bit cache" % (head_size, KV8_WIDTHS[-1]))


KvPlan = collections.namedtuple("KvPlan", ["cu_rows", "slots", "positions", "lens", "free_count", "status"])


def kv_plan(lens, new_rows, tables, free_blocks, free_count, block_size, rows, in_place=True):
    """Blocks and places of the next ``new_rows[b]`` tokens of every request (``new_rows[b]`` < 0: finished, its
    blocks go back to the stack ``free_blocks[:free_count]``); see ``athena_kv_plan`` in include/athena_hip.h.
    ``rows``: room for new rows.  ``tables`` and ``free_blocks`` are updated; so are ``lens`` and ``free_count``
    unless ``in_place`` is false.  Returns a ``KvPlan``; ``status`` (int32 [4]) is not zero where the plan did not
    fit and nothing was changed."""
    B = lens.numel()
    ldt, width = _tables("kv_plan", tables, B)
    if width > 1 and ldt < width and B > 1:
        _refuse("kv_plan", "tables must not share rows")
    _int_vector("kv_plan", "lens", lens, 1)
    _int_vector("kv_plan", "new_rows", new_rows, B)
    _int_vector("kv_plan", "free_blocks", free_blocks, 1)
    _int_vector("kv_plan", "free_count", free_count, 1)
    if rows < 0:
        _refuse("kv_plan", "room for %d rows", rows)
    if in_place and lens.data_ptr() == new_rows.data_ptr():
        _refuse("kv_plan", "lens are updated and cannot be new_rows too")
    stream = _here("kv_plan", lens, new_rows, tables, free_blocks, free_count)
    # one piece of memory for everything the plan writes afresh; what the caller does not get to see lies at its end
    sizes = [B + 1, rows, rows, 4] + ([] if in_place else [B, 1]) + [3 * B + 3]
    fresh = torch.empty(sum(sizes), dtype=_I32, device=lens.device)
    parts = fresh.split_with_sizes(sizes)
    at = fresh.data_ptr()
    p_slots, p_positions, p_status = at + 4 * (B + 1), at + 4 * (B + 1 + rows), at + 4 * (B + 1 + 2 * rows)
    out, count = (lens, free_count) if in_place else parts[4:6]
    p_lens, p_count = lens.data_ptr(), free_count.data_ptr()
    p_work = p_status + 16 if in_place else p_status + 16 + 4 * (B + 1)
    _lib.check(_lib.load().athena_kv_plan(_lib.KvPlanDesc.pack(
        p_lens, new_rows.data_ptr(), tables.data_ptr(), free_blocks.data_ptr(), p_count, at, p_slots, p_positions,
        p_lens if in_place else p_status + 16, p_count if in_place else p_status + 16 + 4 * B, p_status, p_work,
        ldt if B > 1 else width, width, free_blocks.numel(), B, block_size, rows, 0), stream), "athena_kv_plan")
    return KvPlan(parts[0], parts[1], parts[2], out, count, parts[3])


def _kv8_cache(name, k_codes, v_codes, k_scale, v_scale):
    """(blocks, kv heads, block size, width) of a cache."""
    shape = k_codes.shape
    if k_codes.dtype is not _I8 or v_codes.dtype is not _I8 or len(shape) != 4 or not k_codes.is_contiguous() or \
            not v_codes.is_contiguous():
        _refuse(name, "codes must be contiguous int8 [blocks, heads, tokens, columns] (values: columns, tokens)")
    nb, hk, bs, w = shape
    if v_codes.shape != (nb, hk, w, bs):
        _refuse(name, "v_codes must be [%d, %d, %d, %d]", nb, hk, w, bs)
    if k_scale.dtype is not _FP32 or v_scale.dtype is not _FP32 or k_scale.numel() != nb * hk or v_scale.numel() != nb * hk or \
            not k_scale.is_contiguous() or not v_scale.is_contiguous():
        _refuse(name, "scales must be contiguous fp32 [%d, %d]", nb, hk)
    return nb, hk, bs, w


def _head_rows(name, what, x):
    """(shape, strides) of [rows, heads, columns] with contiguous columns."""
    shape, stride = x.shape, x.stride()
    if len(shape) != 3 or (stride[2] != 1 and shape[2] > 1):
        _refuse(name, "%s must be [rows, heads, columns] with contiguous columns", what)
    return shape, stride


def kv8_append(k, v, slots, k_codes, v_codes, k_scale, v_scale):
    """Keys and values [rows, kv heads, head size] into the 8-bit cache at ``slots`` [rows] (-1 skips a row);
    see ``athena_kv8_append`` in include/athena_hip.h."""
    nb, hk, bs, w = _kv8_cache("kv8_append", k_codes, v_codes, k_scale, v_scale)
    shape, sk = _head_rows("kv8_append", "k", k)
    v_shape, sv = _head_rows("kv8_append", "v", v)
    n, heads, dk = shape
    if v_shape != shape or v.dtype != k.dtype or heads != hk or dk > w or dk < 1:
        _refuse("kv8_append", "k and v must be alike, [rows, %d, up to %d]", hk, w)
    _int_vector("kv8_append", "slots", slots, n)
    code = _code("kv8_append", k)
    stream = _here("kv8_append", k, v, slots, k_codes, v_codes, k_scale, v_scale)
    _lib.check(_lib.load().athena_kv8_append(_lib.Kv8AppendDesc.pack(
        k.data_ptr(), v.data_ptr(), slots.data_ptr(), k_codes.data_ptr(), v_codes.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(),
        sk[0], sk[1], sv[0], sv[1], code, n, nb, hk, bs, dk, w, 0), stream), "athena_kv8_append")


def kv8_attention(q, k_codes, v_codes, k_scale, v_scale, tables, lens, cu_rows=None, max_rows=1, causal=True, scale=None,
                  out=None, lse=None):
    """Attention of the query rows [rows, heads, head size] over the 8-bit cache; see ``athena_kv8_attention`` in
    include/athena_hip.h.  ``cu_rows`` None: row b belongs to sequence b.  ``scale`` None: 1 / sqrt(head size).
    Rows of ``out`` that belong to no sequence are left as they were (not set, without ``out``)."""
    nb, hk, bs, w = _kv8_cache("kv8_attention", k_codes, v_codes, k_scale, v_scale)
    shape, sq = _head_rows("kv8_attention", "q", q)
    n, h, dk = shape
    B = lens.numel()
    ldt, width = _tables("kv8_attention", tables, B)
    if h % hk or h < 1 or dk > w or dk < 1 or max_rows < 1:
        _refuse("kv8_attention", "%d heads of %d over %d kv heads of up to %d, %d rows at most", h, dk, hk, w, max_rows)
    _int_vector("kv8_attention", "lens", lens, 1)
    if cu_rows is None:
        if n != B:
            _refuse("kv8_attention", "%d rows for %d sequences need cu_rows", n, B)
    else:
        _int_vector("kv8_attention", "cu_rows", cu_rows, B + 1)
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
        so = (h * dk, dk)
    else:
        o_shape, so = _head_rows("kv8_attention", "out", out)
        if o_shape != shape or out.dtype != q.dtype:
            _refuse("kv8_attention", "out must be like q")
    if lse is not None and (lse.dtype is not _FP32 or lse.numel() != n * h or not lse.is_contiguous()):
        _refuse("kv8_attention", "lse must be contiguous fp32 [%d, %d]", n, h)
    code = _code("kv8_attention", q)
    stream = _here("kv8_attention", q, k_codes, v_codes, k_scale, v_scale, tables, lens, cu_rows, out, lse)
    lib = _lib.load()
    work = 0
    while True:
        desc = _lib.Kv8AttentionDesc.pack(
            q.data_ptr(), k_codes.data_ptr(), v_codes.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), tables.data_ptr(),
            lens.data_ptr(), cu_rows.data_ptr() if cu_rows is not None else 0, out.data_ptr(),
            lse.data_ptr() if lse is not None else 0, ws.data_ptr() if work else 0, work, sq[0], sq[1], so[0], so[1], ldt, code, nb, bs, w,
            width, B, max_rows, n, h, hk, dk, 1 if causal else 0, scale if scale is not None else 1.0 / math.sqrt(dk), 0.0)
        # (a table of fewer than 1024 places never needs a workspace)
        if work or width * bs < 1024:
            break
        work = lib.athena_kv8_attention_workspace_bytes(desc)
        if not work:
            break
        ws = torch.empty(work, dtype=torch.uint8, device=q.device)
    _lib.check(lib.athena_kv8_attention(desc, stream), "athena_kv8_attention")
    return out


def _row_vector(name, what, t, rows):
    if t is None:
        return 0
    if t.dtype is not _FP32 or t.numel() != rows or not t.is_contiguous():
        _refuse(name, "%s must be contiguous fp32 [%d]", what, rows)
    return t.data_ptr()


def _row_matrix(name, what, t, dtype, rows, cols):
    """Leading dimension of [rows, cols], or 0 for one row [cols] / [1, cols] that serves all."""
    shape, stride = t.shape, t.stride()
    dims = len(shape)
    if t.dtype is not dtype or dims not in (1, 2) or shape[-1] != cols or (stride[-1] != 1 and cols > 1) or \
            (dims == 2 and shape[0] != rows and shape[0] != 1):
        _refuse(name, "%s must be %s [%d, %d] or one such row", what, dtype, rows, cols)
    return stride[0] if dims == 2 and shape[0] == rows else 0


def logits_process(logits, history=None, history_len=None, repetition=None, presence=None, frequency=None, bias=None,
                   bias_ids=None, bias_values=None, allowed=None, out=None):
    """Penalties for repeated tokens, biases and a grammar mask on logits [rows, classes]; see
    ``athena_logits_process`` in include/athena_hip.h.  ``history`` int32 [rows, L] with ``history_len`` int32
    [rows]; ``repetition``, ``presence``, ``frequency`` fp32 [rows]; ``bias`` fp32 [rows or 1, classes];
    ``bias_ids`` / ``bias_values`` int32 / fp32 [rows, n]; ``allowed`` int32 [rows or 1, ceil(classes / 32)], a bit per
    class.  Returns ``out`` (a new tensor unless given; it may be ``logits``)."""
    name = "logits_process"
    shape, stride = logits.shape, logits.stride()
    if len(shape) != 2 or (stride[1] != 1 and shape[1] > 1):
        _refuse(name, "logits must be [rows, classes] with contiguous rows")
    R, V = shape
    L = ldh = ldb = ldi = ldv = lda = nb = 0
    if history is not None:
        L = history.shape[-1]
        ldh = _row_matrix(name, "history", history, _I32, R, L)
        if history.dim() != 2 or history.shape[0] != R:
            _refuse(name, "history must be int32 [%d, tokens]", R)
        if history_len is not None:
            _int_vector(name, "history_len", history_len, R)
    elif history_len is not None or repetition is not None or presence is not None or frequency is not None:
        _refuse(name, "penalties need a history")
    rep, pres, freq = _row_vector(name, "repetition", repetition, R), _row_vector(name, "presence", presence, R), \
        _row_vector(name, "frequency", frequency, R)
    if bias is not None:
        ldb = _row_matrix(name, "bias", bias, _FP32, R, V)
    if (bias_ids is None) != (bias_values is None):
        _refuse(name, "bias_ids and bias_values come together")
    if bias_ids is not None:
        nb = bias_ids.shape[-1]
        ldi = _row_matrix(name, "bias_ids", bias_ids, _I32, R, nb)
        ldv = _row_matrix(name, "bias_values", bias_values, _FP32, R, nb)
    if allowed is not None:
        lda = _row_matrix(name, "allowed", allowed, _I32, R, (V + 31) // 32)
    if out is None:
        out, ldo = torch.empty_like(logits, memory_format=torch.contiguous_format), V
    else:
        so = out.stride()
        if out.shape != shape or out.dtype != logits.dtype or (so[1] != 1 and V > 1):
            _refuse(name, "out must be like logits")
        ldo = so[0] if R > 1 else V
    code = _code(name, logits)
    stream = _here(name, logits, history, history_len, repetition, presence, frequency, bias, bias_ids, bias_values, allowed, out)
    ptr = lambda t: 0 if t is None else t.data_ptr()
    _lib.check(_lib.load().athena_logits_process(_lib.LogitsDesc.pack(
        logits.data_ptr(), out.data_ptr(), ptr(history), ptr(history_len), ptr(bias_ids), ptr(allowed), rep, pres, freq, ptr(bias),
        ptr(bias_values), stride[0] if R > 1 else V, ldo, ldh, ldb, ldi, ldv, lda, code, R, V, L, nb, 0), stream),
        "athena_logits_process")
    return out
