"""Embeddings held in 8 bits and scored there (HIP kernels ``tt_cat_*``).

``EmbeddingCatalogue`` keeps the rows that retrieval scores against (the CEO
embeddings) in e4m3, in blocks of 128 values with a power-of-two scale: a
quarter of the fp32 rows' bytes.  Rows are quantised as they are written and
read back as the values they stand for; the product with a block of queries is
that of the values (exact in bfloat16, the matrix cores' operands).

    cat = EmbeddingCatalogue(n_ceos, 256, device="cuda")
    cat.write(ceo_embeddings)                    # rows 0, 1, ...
    cat.write(changed, rows=where)               # rows[i] takes changed[i]
    s = cat.scores(firm_embeddings)              # [m, n_ceos]
    s.backward(ds)                               # gradient of firm_embeddings

Values: every rounding to e4m3 is to nearest even, off by at most 2^-4 of the
value (2^-10 of the block's scale near zero).  Infinities and NaN are held as
NaN and reach only the scores of their own row.  The queries are rounded the
same way inside ``scores``, whose sums are in 32 bits and rounded once to the
results' type; the gradient passes the queries' rounding through unchanged and
is ``ds @ read()`` with sums in 32 bits.  The catalogue itself gets no
gradient.

On CPU tensors the same values come from torch ops.
"""
from __future__ import annotations

from typing import Optional

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _native as N
from . import block8


def _check_dtype(dtype: torch.dtype, what: str):
    if dtype not in N.DTYPES:
        raise NotImplementedError(f"{what}: float32, bfloat16 or float16, got {dtype}")


# (without a Python frame where torch has it)
_is_tracing = getattr(torch._C, "_is_tracing", torch.jit.is_tracing)


def _check_traced(what: str):
    """The kernels are launched on addresses: a traced graph would hold their empty results."""
    if _is_tracing():
        raise NotImplementedError(f"{what}: HIP kernels cannot be traced")


def _rows_2d(x: torch.Tensor, d: int, what: str) -> torch.Tensor:
    """[m, d] with unit stride in a row and rows that do not overlap."""
    if x.dim() != 2 or x.shape[1] != d:
        raise ValueError(f"{what}: expected [rows, {d}], got {tuple(x.shape)}")
    if (d > 1 and x.stride(1) != 1) or (x.shape[0] > 1 and x.stride(0) < d):
        x = x.contiguous()
    return x


def _scores(q, codes, scales, d, n, out_dtype):
    """q [m, d] against the first n rows, [m, n] in out_dtype."""
    dev = q.device
    if dev.type != "cuda":
        qv = block8.decode(*block8.encode(q), d)
        return (qv @ block8.decode(codes[:n], scales[:n], d).t()).to(out_dtype)
    m, L = q.shape[0], N.lib()
    with N.on_device(dev):
        out = torch.empty(m, n, dtype=out_dtype, device=dev)
        wsb = L.tt_cat_scores_workspace_bytes(m, n, d)
        if wsb < 0:
            N.check(wsb, "tt_cat_scores_workspace_bytes")
        ws = torch.empty(wsb, dtype=torch.uint8, device=dev) if wsb else None
        N.check(L.tt_cat_scores(q.data_ptr(), N.DTYPES[q.dtype], m, q.stride(0), d, codes.data_ptr(),
                                scales.data_ptr(), n, out.data_ptr(), N.DTYPES[out_dtype], N.ptr(ws), wsb,
                                N.stream_ptr(dev)), "tt_cat_scores")
    return out


def _dq(ds, codes, scales, d, n, dtype):
    """ds [m, n] times the first n rows, [m, d] in dtype."""
    dev, m = ds.device, ds.shape[0]
    if dev.type != "cuda":
        return (ds.to(torch.float32) @ block8.decode(codes[:n], scales[:n], d)).to(dtype)
    if (n > 1 and ds.stride(1) != 1) or (m > 1 and ds.stride(0) < n):
        ds = ds.contiguous()
    L = N.lib()
    with N.on_device(dev):
        dq = torch.empty(m, d, dtype=dtype, device=dev)
        wsb = L.tt_cat_dq_workspace_bytes(m, n, d, N.DTYPES[ds.dtype])
        if wsb < 0:
            N.check(wsb, "tt_cat_dq_workspace_bytes")
        ws = torch.empty(wsb, dtype=torch.uint8, device=dev) if wsb else None
        N.check(L.tt_cat_dq(ds.data_ptr(), N.DTYPES[ds.dtype], m, ds.stride(0), n, codes.data_ptr(),
                            scales.data_ptr(), d, dq.data_ptr(), N.DTYPES[dtype], N.ptr(ws), wsb,
                            N.stream_ptr(dev)), "tt_cat_dq")
    return dq


class _ScoresFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, codes, scales, d, n, out_dtype):
        ctx.save_for_backward(codes, scales)
        ctx.meta = (d, n, q.dtype)
        return _scores(q, codes, scales, d, n, out_dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, ds):
        codes, scales = ctx.saved_tensors
        d, n, dtype = ctx.meta
        return _dq(ds, codes, scales, d, n, dtype), None, None, None, None, None


class EmbeddingCatalogue:
    """``capacity`` rows of ``dim`` values in e4m3 blocks of 128.

    ``codes`` uint8 [capacity, kp] (kp = dim rounded up to 128, padding zero)
    and ``scales`` uint8 [capacity, kp / 128] (2^(byte - 127)) are the storage:
    ``torch.save`` them, and rebuild with :meth:`from_storage`.  Rows never
    written are zero.  Calls run on the current stream of the catalogue's
    device; writes from several streams have to be ordered by the caller.
    """

    def __init__(self, capacity: int, dim: int, device=None):
        capacity, dim = int(capacity), int(dim)
        if capacity < 0 or not 1 <= dim <= 1 << 20:
            raise ValueError(f"EmbeddingCatalogue: capacity >= 0 and 1 <= dim <= {1 << 20}, got {capacity}, {dim}")
        dev = torch.device("cpu" if device is None else device)
        nkb = block8.blocks_of(dim)
        self._bind(torch.zeros(capacity, nkb * block8.BLOCK, dtype=torch.uint8, device=dev),
                   torch.full((capacity, nkb), 127, dtype=torch.uint8, device=dev), dim)

    @classmethod
    def from_storage(cls, codes: torch.Tensor, scales: torch.Tensor, dim: int) -> "EmbeddingCatalogue":
        """A catalogue on existing storage (shared, not copied)."""
        dim = int(dim)
        if not 1 <= dim <= 1 << 20:
            raise ValueError(f"EmbeddingCatalogue: 1 <= dim <= {1 << 20}, got {dim}")
        nkb = block8.blocks_of(dim)
        if codes.dtype != torch.uint8 or scales.dtype != torch.uint8 or codes.device != scales.device:
            raise ValueError("from_storage: codes and scales are uint8 tensors on one device")
        if codes.dim() != 2 or tuple(scales.shape) != (codes.shape[0], nkb) or codes.shape[1] != nkb * block8.BLOCK:
            raise ValueError(f"from_storage: codes [rows, {nkb * block8.BLOCK}] and scales [rows, {nkb}] for dim {dim}, "
                             f"got {tuple(codes.shape)} and {tuple(scales.shape)}")
        if not codes.is_contiguous() or not scales.is_contiguous() or codes.data_ptr() % 16:
            raise ValueError("from_storage: contiguous storage, codes on a 16-byte boundary")
        self = cls.__new__(cls)
        self._bind(codes, scales, dim)
        return self

    def _bind(self, codes, scales, dim):
        self.codes, self.scales, self.dim = codes, scales, dim
        self.capacity, self.device = codes.shape[0], codes.device
        # which mention of a row an indexed write keeps; zero between calls
        self._owner = (torch.zeros(self.capacity, dtype=torch.int32, device=codes.device)
                       if codes.device.type == "cuda" else None)

    # -- rows of a call -------------------------------------------------------
    def _check_rows(self, rows, m: int, what: str):
        if rows is None:
            return None
        if rows.dim() != 1 or rows.dtype not in (torch.int64, torch.int32):
            raise ValueError(f"{what}: rows is a 1-d int64 or int32 tensor")
        if rows.device != self.device:
            raise ValueError(f"{what}: rows on {rows.device}, the catalogue on {self.device}")
        if m >= 0 and rows.shape[0] != m:
            raise ValueError(f"{what}: {rows.shape[0]} row numbers for {m} rows")
        if rows.dtype == torch.int64 and rows.is_contiguous():
            return rows
        return rows.to(torch.int64).contiguous()

    def _check_range(self, start: int, m: int, what: str):
        if start < 0 or m < 0 or start + m > self.capacity:
            raise ValueError(f"{what}: rows {start} .. {start + m} of {self.capacity}")

    def write(self, emb: torch.Tensor, rows: Optional[torch.Tensor] = None, start: int = 0) -> None:
        """Quantise ``emb`` [m, dim] into rows ``start ..`` or, with ``rows``
        [m], into those.  Row numbers outside the catalogue are left out (a
        padded batch uses -1); a row named twice takes its last mention."""
        emb = _rows_2d(emb.detach(), self.dim, "write")
        _check_dtype(emb.dtype, "write")
        if emb.device != self.device:
            raise ValueError(f"write: embeddings on {emb.device}, the catalogue on {self.device}")
        m, start = emb.shape[0], int(start)
        rows = self._check_rows(rows, m, "write")
        if rows is None:
            self._check_range(start, m, "write")
        elif start:
            raise ValueError("write: rows or start, not both")
        if self.device.type == "cuda":
            _check_traced("write")
        if m == 0:
            return
        if not self.codes.is_inference():  # a backward that saved the old rows must notice
            torch.autograd.graph.increment_version((self.codes, self.scales))
        if self.device.type != "cuda":
            codes, scales = block8.encode(emb)
            if rows is None:
                self.codes[start:start + m], self.scales[start:start + m] = codes, scales
                return
            last = {int(r): i for i, r in enumerate(rows.tolist()) if 0 <= r < self.capacity}
            if last:
                r, i = torch.tensor(list(last.keys())), torch.tensor(list(last.values()))
                self.codes[r], self.scales[r] = codes[i], scales[i]
            return
        with N.on_device(self.device):
            N.check(N.lib().tt_cat_write(emb.data_ptr(), N.DTYPES[emb.dtype], m, emb.stride(0), self.dim, N.ptr(rows),
                                         start, self.codes.data_ptr(), self.scales.data_ptr(), self.capacity,
                                         N.ptr(self._owner), N.stream_ptr(self.device)), "tt_cat_write")

    def read(self, rows: Optional[torch.Tensor] = None, start: int = 0, count: Optional[int] = None,
             dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """The values rows ``start .. start + count`` (default: to the end) or
        ``rows`` stand for, [m, dim]; row numbers outside the catalogue read
        as zeros.  float32 and bfloat16 hold every value exactly."""
        _check_dtype(dtype, "read")
        rows = self._check_rows(rows, -1, "read")
        start = int(start)
        if rows is not None:
            if start or count is not None:
                raise ValueError("read: rows or a range, not both")
            m = rows.shape[0]
        else:
            m = self.capacity - start if count is None else int(count)
            self._check_range(start, m, "read")
        if self.device.type != "cuda":
            if rows is None:
                return block8.decode(self.codes[start:start + m], self.scales[start:start + m], self.dim).to(dtype)
            ok = (rows >= 0) & (rows < self.capacity)
            out = torch.zeros(m, self.dim)
            out[ok] = block8.decode(self.codes[rows[ok]], self.scales[rows[ok]], self.dim)
            return out.to(dtype)
        _check_traced("read")
        with N.on_device(self.device):
            out = torch.empty(m, self.dim, dtype=dtype, device=self.device)
            N.check(N.lib().tt_cat_read(self.codes.data_ptr(), self.scales.data_ptr(), self.capacity, self.dim,
                                        N.ptr(rows), start, m, out.data_ptr(), N.DTYPES[dtype], self.dim,
                                        N.stream_ptr(self.device)), "tt_cat_read")
        return out

    def scores(self, queries: torch.Tensor, count: Optional[int] = None,
               dtype: Optional[torch.dtype] = None) -> torch.Tensor:
        """Inner products of ``queries`` [..., dim] with the first ``count``
        rows (default: all), [..., count], in ``dtype`` (default: the
        queries').  Differentiable in the queries, once, in reverse mode."""
        dtype = queries.dtype if dtype is None else dtype
        _check_dtype(queries.dtype, "scores")
        _check_dtype(dtype, "scores")
        if queries.device != self.device:
            raise ValueError(f"scores: queries on {queries.device}, the catalogue on {self.device}")
        if queries.dim() < 1 or queries.shape[-1] != self.dim:
            raise ValueError(f"scores: expected [..., {self.dim}], got {tuple(queries.shape)}")
        # (outside every dual level, known without a call, there is no tangent)
        if getattr(forward_ad, "_current_level", 0) >= 0 and forward_ad.unpack_dual(queries).tangent is not None:
            raise NotImplementedError("scores: no forward-mode derivative, use backward")
        if self.device.type == "cuda":
            _check_traced("scores")
        n = self.capacity if count is None else int(count)
        self._check_range(0, n, "scores")
        flat = queries.dim() == 2
        q = _rows_2d(queries if flat else queries.reshape(-1, self.dim), self.dim, "scores")
        if q.requires_grad and torch.is_grad_enabled():
            s = _ScoresFn.apply(q, self.codes, self.scales, self.dim, n, dtype)
        else:
            s = _scores(q, self.codes, self.scales, self.dim, n, dtype)
        return s if flat else s.reshape(*queries.shape[:-1], n)
