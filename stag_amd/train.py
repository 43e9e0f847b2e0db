"""Learning node classifiers on the GPU (include/stag_train.h): the counterpart of the scoring that the walk does.

The reference fits one logistic regression per tree node on the CPU (stag/create_db.py:127-145).  Here the children of a
node -- or all nodes of a level -- share a TABLE of coefficients [n_features, k]: row f belongs to token f (5 * alignment column +
symbol), column c to classifier c, and a step of the fit is

    scores        = row_scores(bits, table, bias, rows=batch)
    loss, grad    = sibling_loss(scores, label, ...)
    row_scores_grad(bits, grad, n_features, rows=batch, out=(table_grad, bias_grad))
    optimizer.step()                                   # AdamW over every table and bias, with an L1 penalty

``bits`` are packed one-hot rows as ``Database.encode_a2m`` / ``stag_encode_a2m_dev`` make them, on the GPU.  ``fit_siblings`` runs
these steps for the children of one node and returns coefficients in the form ``load_db`` gives them, for
``Database.from_dicts``.

All functions take torch tensors on one GPU, enqueue their work on that GPU's current stream and return without waiting;
they take no part in autograd.  With their outputs given (``out=``: fixed buffers, at the price of more checks on the host) or allocated
under capture they can be recorded into a HIP graph.  Inputs whose rows are not contiguous (or lie more than 2^21 values apart) are copied
first; outputs have to be as documented and may share memory with nothing else that the call takes.
"""
import ctypes
import functools
import math

import numpy as np
import torch

from . import _lib

BLOCK, TILE, STEP_WORDS = 256, 1024, 1088            # STAG_ADAMW_BLOCK, STAG_ADAMW_TILE, STAG_ADAMW_STEP_WORDS
_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_TENSOR = np.dtype([("param", "<u8"), ("grad", "<u8"), ("count", "<i8"), ("state_at", "<i8"), ("weight_decay", "<f4"), ("l1", "<f4"),
                    ("param_type", "<i4"), ("grad_type", "<i4")])      # stag_adamw_tensor_t


_Tensor = torch.Tensor
_F32, _I32 = torch.float32, torch.int32
_BITS = (torch.int32, torch.uint32)
_empty = torch.empty_strided
_raw_stream = torch._C._cuda_getCurrentRawStream      # torch.cuda.current_stream(i).cuda_stream without the objects
_current = torch._C._cuda_getDevice
_address, _size = _Tensor.data_ptr, torch._C.StorageBase.nbytes
_MAX_STRIDE = 1 << 21                                # values from one row of a matrix to the next


def _need(cond, msg, *args):
    if not cond:
        raise ValueError(msg % args)


def _is(name, t, dtypes, dim):
    if not isinstance(t, _Tensor):
        raise TypeError("%s must be a torch tensor" % name)
    dtypes = dtypes if isinstance(dtypes, tuple) else (dtypes,)
    if t.dtype not in dtypes:
        raise TypeError("%s is %s: %s is wanted" % (name, t.dtype, " or ".join(str(d) for d in dtypes)))
    _need(t.dim() == dim, "%s has %d dimensions: %d are wanted", name, t.dim(), dim)


def _plain(t, dtype, shape, gpu):
    """Whether t is a contiguous tensor of this type and shape on this GPU: nothing to check or copy."""
    return type(t) is _Tensor and t.dtype is dtype and t.get_device() == gpu and t.is_contiguous() and t.shape == shape


def _one_gpu(**tensors):
    device = None
    for name, t in tensors.items():
        if t is None:
            continue
        _need(t.device.type == "cuda", "%s is on %s: the operators run on the GPU", name, t.device)
        _need(device is None or t.device == device, "%s is on %s, other tensors on %s", name, t.device, device)
        device = t.device
    return device


def _rows(t):
    """t with contiguous rows (copied if they are not), and its row stride."""
    n, k = t.shape
    if (k > 1 and t.stride(1) != 1) or (n > 1 and not k <= t.stride(0) <= _MAX_STRIDE):
        t = t.contiguous()
    return t, (t.stride(0) if n > 1 else k)


def _out_rows(name, t, shape, dtype):
    _is(name, t, dtype, len(shape))
    _need(tuple(t.shape) == tuple(shape), "%s has shape %s: %s is wanted", name, tuple(t.shape), tuple(shape))
    if len(shape) == 1:
        _need(shape[0] <= 1 or t.stride(0) == 1, "%s must be contiguous", name)
        return shape[0]
    _need((shape[1] <= 1 or t.stride(1) == 1) and (shape[0] <= 1 or t.stride(0) >= shape[1]), "%s must have contiguous rows that do not overlap", name)
    _need(shape[0] <= 1 or t.stride(0) <= _MAX_STRIDE, "%s has rows more than %d values apart", name, _MAX_STRIDE)
    return t.stride(0) if shape[0] > 1 else shape[1]


def _share(a, b):
    """Whether two tensors of contiguous rows share memory."""
    if a.numel() == 0 or b.numel() == 0:
        return False
    place = []
    for t in (a, b):
        size, rows = t.element_size(), t.shape[0] if t.dim() == 2 else 1
        step = t.stride(0) * size if rows > 1 else 0
        width = t.shape[-1] * size
        place.append((t.data_ptr(), step, width, (rows - 1) * step + width))
    (at, step_a, width_a, all_a), (bt, step_b, width_b, all_b) = place
    if at + all_a <= bt or bt + all_b <= at:
        return False
    step = step_a or step_b
    if not step or (step_a and step_b and step_a != step_b):
        return True
    apart = (at - bt) % step                           # columns of one buffer
    return apart < width_b or apart + width_a > step


def _apart(outputs, inputs):
    """Refuses outputs that share memory with one another or an input."""
    named = list(outputs.items())
    for j, (name, t) in enumerate(named):
        for other, u in named[j + 1:] + list(inputs.items()):
            if u is not None and t is not None and _share(t, u):
                raise ValueError("%s and %s share memory" % (name, other))


def _packed(bits, n_features):
    """bits, its row stride in words."""
    _need(bits.shape[1] * 32 >= n_features, "bits has %d words a row: too few for %d features", bits.shape[1], n_features)
    n, w = bits.shape
    if (w > 1 and bits.stride(1) != 1) or (n > 1 and bits.stride(0) < w):
        bits = bits.contiguous()
    stride = bits.stride(0) if n > 1 else -(-w // 4) * 4
    _need(w % 4 == 0 and stride % 4 == 0 and bits.data_ptr() % 16 == 0, "rows of bits must be whole, aligned 16-byte units (as stag_encode_a2m writes them)")
    return bits, stride


def _ptr(t):
    return None if t is None else t.data_ptr()


@functools.lru_cache(maxsize=65536)
def _workspace(name, m, *sizes):
    _need(max(sizes) < 2**31, "sizes of 2^31 and more: %s", sizes)          # the C ABI has 32 bits for all but m
    nbytes = getattr(_lib.train_lib(), name)(m, *sizes)
    if nbytes < 0:
        _lib.check_train(int(nbytes))
    return nbytes


def _check_scores(bits, table, bias, rows, out):
    _is("bits", bits, _BITS, 2)
    _is("table", table, tuple(_TYPES), 2)
    n_features, k = table.shape
    _need(n_features >= 1 and k >= 1, "table is empty: %s", tuple(table.shape))
    if bias is not None:
        _is("bias", bias, torch.float32, 1)
        _need(bias.shape[0] == k, "bias has %d values, the table %d columns", bias.shape[0], k)
        bias = bias.contiguous()
    if rows is not None:
        _is("rows", rows, torch.int32, 1)
        rows = rows.contiguous()
    m = bits.shape[0] if rows is None else rows.shape[0]
    score_stride = k if out is None else _out_rows("out", out, (m, k), torch.float32)
    _one_gpu(bits=bits, table=table, bias=bias, rows=rows, out=out)
    bits, row_stride = _packed(bits, n_features)
    table, table_stride = _rows(table)
    _apart({"out": out}, {"bits": bits, "table": table, "bias": bias, "rows": rows})
    return bits, table, bias, rows, row_stride, table_stride, score_stride


def row_scores(bits, table, bias=None, *, scale=1.0, rows=None, out=None):
    """scores[i, c] = scale * (sum of table[f, c] over the features f of row rows[i] of bits) + bias[c], float32 [m, k]
    (the sum of run_logistic_prediction, stag/classify.py:22-27; an embedding lookup summed over a row's tokens).

    bits: int32 / uint32 [n, words]; table: float32, bfloat16 or float16 [n_features, k]; bias: float32 [k]; rows: int32 [m], any
    order, repeats allowed, an index outside 0..n-1 is padding and scores 0 (default: all rows of bits)."""
    kind = -1
    if type(bits) is _Tensor and type(table) is _Tensor and out is None and bits.is_contiguous() and table.is_contiguous():
        gpu = bits.get_device()
        if gpu >= 0 and table.get_device() == gpu and bits.dim() == 2 and table.dim() == 2 and bits.dtype in _BITS:
            row_stride, (n_features, k) = bits.shape[1], table.shape
            if (row_stride & 3 == 0 and bits.data_ptr() & 15 == 0 and k and 0 < n_features <= row_stride * 32 and (bias is None or _plain(bias, _F32, (k,), gpu))
                    and (rows is None or (type(rows) is _Tensor and rows.dim() == 1 and _plain(rows, _I32, rows.shape, gpu)))):
                kind = 0 if table.dtype is _F32 else _TYPES.get(table.dtype, -1)
                table_stride = score_stride = k
    if kind < 0:
        bits, table, bias, rows, row_stride, table_stride, score_stride = _check_scores(bits, table, bias, rows, out)
        gpu, kind = bits.get_device(), _TYPES[table.dtype]
    if gpu != _current():
        with torch.cuda.device(gpu):
            return row_scores(bits, table, bias, scale=scale, rows=rows, out=out)
    n = bits.shape[0]
    n_features, k = table.shape
    m = n if rows is None else rows.shape[0]
    need = _workspace("stag_row_scores_workspace", m, n_features, k, kind)
    if out is None:
        out = _empty((m, k), (k, 1), dtype=_F32, device=bits.device)
    work = _empty((need,), (1,), dtype=torch.uint8, device=bits.device) if need else None
    rc = _lib.train_lib().stag_row_scores_dev(bits.data_ptr(), n, row_stride, n_features, None if rows is None else rows.data_ptr(), m, table.data_ptr(), kind,
                                              table_stride, None if bias is None else bias.data_ptr(), k, float(scale), out.data_ptr(), score_stride,
                                              work.data_ptr() if need else None, need, _raw_stream(gpu))
    if rc:
        _lib.check_train(rc)
    return out


def _check_grad(bits, grad, n_features, rows, out):
    _is("bits", bits, _BITS, 2)
    _is("grad", grad, tuple(_TYPES), 2)
    m, k = grad.shape
    _need(n_features >= 1 and k >= 1, "no features (%d) or no classifiers (%d)", n_features, k)
    if rows is not None:
        _is("rows", rows, torch.int32, 1)
        rows = rows.contiguous()
    batch = bits.shape[0] if rows is None else rows.shape[0]
    _need(m == batch, "grad has %d rows, the batch %d", m, batch)
    table_grad, bias_grad = out if out is not None else (None, None)
    stride = k
    if out is not None:
        stride = _out_rows("out[0]", table_grad, (n_features, k), torch.float32)
        _out_rows("out[1]", bias_grad, (k,), torch.float32)
    _one_gpu(bits=bits, grad=grad, rows=rows, table_grad=table_grad, bias_grad=bias_grad)
    bits, row_stride = _packed(bits, n_features)
    grad, grad_stride = _rows(grad)
    _apart({"out[0]": table_grad, "out[1]": bias_grad}, {"bits": bits, "grad": grad, "rows": rows})
    return bits, grad, rows, row_stride, grad_stride, stride


def row_scores_grad(bits, grad, n_features, *, scale=1.0, rows=None, out=None):
    """The gradient of row_scores: (table_grad float32 [n_features, k], bias_grad float32 [k]) with
    table_grad[f, c] = scale * (sum of grad[i, c] over the i whose row has feature f), bias_grad[c] = sum of grad[i, c].

    grad: float32, bfloat16 or float16 [m, k].  Padding rows (see row_scores) take part in neither, whatever grad holds for
    them.  out: a pair of tensors to overwrite."""
    n_features, kind = int(n_features), -1
    if type(bits) is _Tensor and type(grad) is _Tensor and bits.is_contiguous() and grad.is_contiguous():
        gpu = bits.get_device()
        if gpu >= 0 and grad.get_device() == gpu and bits.dim() == 2 and grad.dim() == 2 and bits.dtype in _BITS:
            (n, row_stride), (m, k) = bits.shape, grad.shape
            if (row_stride & 3 == 0 and bits.data_ptr() & 15 == 0 and k and m and 0 < n_features <= row_stride * 32 and (n == m if rows is None else _plain(rows, _I32, (m,), gpu))
                    and out is None):
                kind = 0 if grad.dtype is _F32 else _TYPES.get(grad.dtype, -1)
                grad_stride = stride = k
    if kind < 0:
        bits, grad, rows, row_stride, grad_stride, stride = _check_grad(bits, grad, n_features, rows, out)
        gpu, kind = bits.get_device(), _TYPES[grad.dtype]
    if gpu != _current():
        with torch.cuda.device(gpu):
            return row_scores_grad(bits, grad, n_features, scale=scale, rows=rows, out=out)
    m, k = grad.shape
    need = _workspace("stag_row_scores_grad_workspace", m, n_features, k, kind)
    if out is None:
        table_grad = _empty((n_features, k), (k, 1), dtype=_F32, device=bits.device)
        bias_grad = _empty((k,), (1,), dtype=_F32, device=bits.device)
    else:
        table_grad, bias_grad = out
    work = _empty((need,), (1,), dtype=torch.uint8, device=bits.device) if need else None
    rc = _lib.train_lib().stag_row_scores_grad_dev(bits.data_ptr(), bits.shape[0], row_stride, n_features, None if rows is None else rows.data_ptr(), m, grad.data_ptr(),
                                                   kind, grad_stride, k, float(scale), table_grad.data_ptr(), stride, bias_grad.data_ptr(),
                                                   work.data_ptr() if need else None, need, _raw_stream(gpu))
    if rc:
        _lib.check_train(rc)
    return table_grad, bias_grad


def _check_loss(scores, label, siblings, weight, dtype, out):
    _is("scores", scores, torch.float32, 2)
    _is("label", label, torch.int32, 1)
    m, k = scores.shape
    _need(k >= 1, "no classifiers")
    _need(label.shape[0] == m, "label has %d values, scores %d rows", label.shape[0], m)
    label = label.contiguous()
    if siblings is not None:
        _is("siblings", siblings, torch.int32, 2)
        _need(tuple(siblings.shape) == (m, 2), "siblings has shape %s: %s is wanted", tuple(siblings.shape), (m, 2))
        siblings = siblings.contiguous()
    if weight is not None:
        _is("weight", weight, torch.float32, 1)
        _need(weight.shape[0] == m, "weight has %d values, scores %d rows", weight.shape[0], m)
        weight = weight.contiguous()
    if dtype not in _TYPES:
        raise TypeError("grad_dtype is %s: %s is wanted" % (dtype, " or ".join(str(d) for d in _TYPES)))
    loss, grad = out if out is not None else (None, None)
    grad_stride = k
    if out is not None:
        _out_rows("out[0]", loss, (k,), torch.float32)
        grad_stride = _out_rows("out[1]", grad, (m, k), dtype)
    _one_gpu(scores=scores, label=label, siblings=siblings, weight=weight, loss=loss, grad=grad)
    scores, score_stride = _rows(scores)
    _apart({"out[0]": loss, "out[1]": grad}, {"scores": scores, "label": label, "siblings": siblings, "weight": weight})
    return scores, label, siblings, weight, score_stride, grad_stride


def sibling_loss(scores, label, *, siblings=None, weight=None, scale=1.0, grad_dtype=None, out=None):
    """Logistic loss of "this sibling or one of the others" and its gradient: (loss float32 [k], grad [m, k]).

    Row i trains the columns siblings[i, 0] <= c < siblings[i, 1] (int32 [m, 2]; children of a node are neighbours in
    breadth-first numbering; default: all k) with target 1 for c == label[i] (int32 [m]) and 0 for the others; a label
    outside them makes the row a negative example for all.  loss[c] = scale * sum of weight[i] * softplus(+-score);
    grad is d(sum of loss)/d(scores) of type grad_dtype (default float32), 0 where a row does not train, and scores are not
    read there.  weight: float32 [m].  out: a pair of tensors to overwrite."""
    dtype = grad_dtype or (out[1].dtype if out is not None else torch.float32)
    plain = False
    if type(scores) is _Tensor and out is None and scores.dtype is _F32 and scores.is_contiguous() and dtype in _TYPES:
        gpu = scores.get_device()
        if gpu >= 0 and scores.dim() == 2:
            m, k = scores.shape
            plain = (m and k and _plain(label, _I32, (m,), gpu) and (siblings is None or _plain(siblings, _I32, (m, 2), gpu))
                     and (weight is None or _plain(weight, _F32, (m,), gpu)))
            score_stride = grad_stride = k
    if not plain:
        scores, label, siblings, weight, score_stride, grad_stride = _check_loss(scores, label, siblings, weight, dtype, out)
        gpu = scores.get_device()
    if gpu != _current():
        with torch.cuda.device(gpu):
            return sibling_loss(scores, label, siblings=siblings, weight=weight, scale=scale, grad_dtype=dtype, out=out)
    m, k = scores.shape
    need = _workspace("stag_sibling_loss_workspace", m, k)
    if out is None:
        loss = _empty((k,), (1,), dtype=_F32, device=scores.device)
        grad = _empty((m, k), (k, 1), dtype=dtype, device=scores.device)
    else:
        loss, grad = out
    work = _empty((need,), (1,), dtype=torch.uint8, device=scores.device) if need else None
    rc = _lib.train_lib().stag_sibling_loss_dev(scores.data_ptr(), score_stride, m, k, label.data_ptr(), None if siblings is None else siblings.data_ptr(),
                                                None if weight is None else weight.data_ptr(), float(scale), loss.data_ptr(), grad.data_ptr(), _TYPES[dtype], grad_stride,
                                                work.data_ptr() if need else None, need, _raw_stream(gpu))
    if rc:
        _lib.check_train(rc)
    return loss, grad


def _fixed(t):
    """t's memory as a tensor whose storage cannot be resized."""
    return None if t is None else torch.utils.dlpack.from_dlpack(torch.utils.dlpack.to_dlpack(t.view(torch.uint8))).view(t.dtype)


class AdamW:
    """AdamW over a list of tensors, one launch a step, with an optional L1 shrinkage (stag_adamw_dev).

    params, grads: lists of contiguous tensors (float32, bfloat16 or float16) on one GPU, a gradient as large as its parameter.  The
    optimizer holds THESE tensors: it reads the gradients from them and updates the parameters in place, at every step.  They keep
    the memory they had when it was made: after ``.data = ...``, ``set_``, a ``resize_`` that moves one or a module's ``.to(dtype)``, step() raises
    ValueError.  (Of views that share a storage it looks at one; another that is given other memory is not followed: step() goes on with the old.)
    weight_decay, l1: a number, or one for each tensor.  state_bits 32 keeps the moments as floats; 8 keeps e4m3 codes with a
    power-of-two scale for each 256 values (m, m_scale: the first moment; v, v_scale: the ROOT of the second), 2.03 bytes
    a value instead of 8.  m, v and the scales are flat: tensor j's values begin at place state_at[j], a multiple of 256.
    Addresses are taken once, so an AdamW is neither copied nor pickled: make another, and load_state() into it.
    The step count lives on the GPU, so a captured step() counts on when it is replayed (a graph holds none of this memory: the AdamW
    has to live as long); lr and the others are the values that step() was called with (attributes, may be changed between steps)."""

    def __init__(self, params, grads, *, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.0, l1=0.0, state_bits=32):
        params, grads = list(params), list(grads)
        _need(len(params) >= 1, "no parameters")
        _need(len(params) == len(grads), "%d parameters, %d gradients", len(params), len(grads))
        _need(state_bits in (8, 32), "state_bits = %r: 8 or 32 are wanted", state_bits)
        decay = [float(x) for x in (weight_decay if isinstance(weight_decay, (list, tuple)) else [weight_decay] * len(params))]
        l1 = [float(x) for x in (l1 if isinstance(l1, (list, tuple)) else [l1] * len(params))]
        _need(len(decay) == len(params) and len(l1) == len(params), "weight_decay and l1 are one number, or one for each of the %d tensors", len(params))
        for x in set(decay + l1):
            _need(math.isfinite(x) and x >= 0, "weight_decay and l1 are not negative: got %r", x)
        self.lr, self.betas, self.eps, self.state_bits = lr, tuple(betas), eps, state_bits
        b1, b2 = self.betas
        _need(math.isfinite(lr) and lr >= 0, "lr = %r", lr)
        _need(0 < b1 < 1 and 0 < b2 < 1, "betas = %r: not inside (0, 1)", betas)
        _need(math.isfinite(eps) and eps >= 0, "eps = %r", eps)
        both = params + grads
        n = len(params)
        name = lambda j: "params[%d]" % j if j < n else "grads[%d]" % (j - n)      # noqa: E731
        if not all(isinstance(x, _Tensor) for x in both) or not {x.dtype for x in both} <= set(_TYPES):
            j = next(j for j, x in enumerate(both) if not isinstance(x, _Tensor) or x.dtype not in _TYPES)
            raise TypeError("%s must be a float32, bfloat16 or float16 tensor" % name(j))
        for j, x in enumerate(both):
            if not x.is_contiguous():
                raise ValueError("%s is not contiguous" % name(j))
        for j, (x, g) in enumerate(zip(params, grads)):
            if x.shape != g.shape:
                raise ValueError("params[%d] has shape %s, its gradient %s" % (j, tuple(x.shape), tuple(g.shape)))
        gpus = [x.get_device() for x in both]
        if len(set(gpus)) > 1 or gpus[0] < 0:
            _one_gpu(**{name(j): x for j, x in enumerate(both)})
        device = params[0].device
        counts = np.array([x.numel() for x in params], dtype=np.int64)
        at = np.array([x.data_ptr() for x in both], dtype=np.uint64)
        end = at + np.array([x.nbytes for x in both], dtype=np.uint64)
        order = np.flatnonzero(end > at)
        order = order[np.lexsort((order, at[order]))]
        # gradients may share memory with each other, what is written with nothing
        for mine, others in ((order < n, np.ones(len(order), bool)), (order >= n, order < n)):
            reach = np.maximum.accumulate(np.where(others, end[order], 0))[:-1]          # how far those before go
            bad = np.flatnonzero(mine[1:] & (reach > at[order][1:]))
            if len(bad):
                k = int(bad[0]) + 1
                before = max((int(end[q]), int(q)) for q, o in zip(order[:k], others[:k]) if o)[1]
                raise ValueError("%s and %s share memory" % (name(before), name(int(order[k]))))
        self._device, self._params, self._grads = device, tuple(params), tuple(grads)
        table = np.zeros(n, dtype=_TENSOR)
        padded = -(-counts // BLOCK) * BLOCK
        self.state_at = np.concatenate([[0], np.cumsum(padded)[:-1]]).tolist()
        self.state_values = int(padded.sum())
        table["param"], table["grad"] = at[:n], at[n:]
        table["count"], table["state_at"] = counts, self.state_at
        table["weight_decay"], table["l1"] = decay, l1
        table["param_type"] = [_TYPES[p.dtype] for p in params]
        table["grad_type"] = [_TYPES[g.dtype] for g in grads]
        n_tiles = -(-counts // TILE)
        first = np.concatenate([[0], np.cumsum(n_tiles)[:-1]])
        tiles = np.empty((int(n_tiles.sum()), 2), dtype=np.int32)
        tiles[:, 0] = np.repeat(np.arange(len(params)), n_tiles)
        tiles[:, 1] = np.arange(len(tiles)) - np.repeat(first, n_tiles)
        self._n_tiles = len(tiles)
        self._tensors = torch.from_numpy(table.view(np.uint8)).to(device)
        self._tiles = torch.from_numpy(tiles).to(device)
        self._step = torch.zeros(STEP_WORDS, dtype=torch.int32, device=device)
        size = max(self.state_values, BLOCK)
        kind = torch.float32 if state_bits == 32 else torch.float8_e4m3fn
        self._m = torch.zeros(size, dtype=torch.float32, device=device).to(kind)
        self._v = torch.zeros(size, dtype=torch.float32, device=device).to(kind)
        self._m_scale = self._v_scale = None
        if state_bits == 8:
            self._m_scale = torch.ones(size // BLOCK, dtype=torch.float32, device=device)
            self._v_scale = torch.ones(size // BLOCK, dtype=torch.float32, device=device)
        # What the kernel reads and writes stays allocated while its address is held: a storage for each memory, and a tensor whose address shows
        # whether it moved.  The states are given out as tensors that cannot be resized.
        memory = {}
        for x in both:
            storage = x.untyped_storage()
            memory.setdefault(storage._cdata, (x, storage))
        self._watched, self._storages = [list(x) for x in zip(*memory.values())]
        self._addresses, self._sizes = [*map(_address, self._watched)], [*map(_size, self._storages)]
        pointer = lambda x: None if x is None else ctypes.c_void_p(x.data_ptr())      # noqa: E731
        self._where = (pointer(self._tensors), pointer(self._tiles), self._n_tiles, state_bits, pointer(self._m), pointer(self._v), pointer(self._m_scale),
                       pointer(self._v_scale), pointer(self._step))
        self._given_m, self._given_v, self._given_m_scale, self._given_v_scale = (_fixed(x) for x in (self._m, self._v, self._m_scale, self._v_scale))
        self._gpu, self._launch = device.index, _lib.train_lib().stag_adamw_dev

    device, params, grads, m, v, m_scale, v_scale = (
        property(lambda self, name=name: getattr(self, name)) for name in ("_device", "_params", "_grads", "_given_m", "_given_v", "_given_m_scale", "_given_v_scale"))

    def __reduce_ex__(self, protocol):
        raise TypeError("an AdamW holds the addresses of its tensors: make another, and load_state() into it")

    def step(self):
        """One step with the gradients as they stand."""
        gpu = self._gpu
        if gpu != _current():
            with torch.cuda.device(gpu):
                return self.step()
        if [*map(_address, self._watched)] != self._addresses or [*map(_size, self._storages)] != self._sizes:
            self._moved()
        rc = self._launch(*self._where, self.lr, *self.betas, self.eps, _raw_stream(gpu))
        if rc:
            _lib.check_train(rc)

    def _moved(self):
        for x, at, storage, size in zip(self._watched, self._addresses, self._storages, self._sizes):
            if x.data_ptr() != at or _size(storage) != size:
                name = next("%s[%d]" % (kind, j) for kind, held in (("params", self._params), ("grads", self._grads)) for j, y in enumerate(held) if y is x)
                raise ValueError("%s has other memory than when this AdamW was made: make another" % name)

    @property
    def steps(self):
        """Steps done so far (waits for the GPU)."""
        return int(self._step[0].item())

    def load_state(self, steps, m, v, m_scale=None, v_scale=None):
        """Takes up a state as .steps, .m, .v, .m_scale and .v_scale give it."""
        _need(0 <= int(steps) < 2**31 - 1, "steps = %r", steps)
        given = {"m": m, "v": v, "m_scale": m_scale, "v_scale": v_scale}
        for name, t in given.items():
            mine = getattr(self, "_" + name)
            _need((t is None) == (mine is None), "%s: %s", name, "missing" if t is None else "states of 32 bits have none")
            if mine is not None:
                _is(name, t, mine.dtype, 1)
                _need(t.shape == mine.shape, "%s has %d values: %d are wanted", name, t.shape[0], mine.shape[0])
        for name, t in given.items():
            if t is not None:
                getattr(self, "_" + name).copy_(t)
        self._step[0] = int(steps)


def fit_siblings(bits, label, k, n_features, *, steps=200, batch=None, lr=0.05, l1=0.0, weight_decay=0.0, weight=None, table_dtype=torch.float32,
                 state_bits=32, seed=0, device=None):
    """Fits the classifiers of k siblings (the children of one node, stag/create_db.py:127-145) and returns float64 [k, 1 + n_features]:
    intercept and coefficients as load_db gives them (stag/databases.py:96-104), one row a sibling.

    bits: packed rows uint32 [n, words] (NumPy, as Database.encode_a2m returns them) or a tensor; label: the sibling of each row,
    another value = a negative example for all.  l1 penalises coefficients (not the intercept) by l1 * |w| beside the mean loss
    of a row.  batch: rows a step (default all), drawn anew each pass by `seed`."""
    if isinstance(bits, np.ndarray):
        if bits.dtype not in (np.uint32, np.int32):
            raise TypeError("bits is %s: uint32 words are wanted" % bits.dtype)
        bits = torch.from_numpy(np.ascontiguousarray(bits).view(np.int32)).to(device or "cuda")
    _is("bits", bits, _BITS, 2)
    device = bits.device
    n, k, n_features = bits.shape[0], int(k), int(n_features)
    _need(n >= 1, "no rows")
    _need(k >= 1 and n_features >= 1, "no features (%d) or no classifiers (%d)", n_features, k)
    _need(batch is None or int(batch) >= 1, "batch = %r", batch)
    label = torch.as_tensor(label)
    _need(tuple(label.shape) == (n,), "label has shape %s: %s is wanted", tuple(label.shape), (n,))
    if label.is_floating_point() or label.is_complex():
        raise TypeError("label is %s: whole numbers are wanted" % label.dtype)
    label = label.to(device=device, dtype=torch.int64)
    label = torch.where((label >= 0) & (label < k), label, -1).to(torch.int32)       # before 64 bits become 32
    if weight is not None:
        weight = torch.as_tensor(weight).to(device=device, dtype=torch.float32)
        _need(tuple(weight.shape) == (n,), "weight has shape %s: %s is wanted", tuple(weight.shape), (n,))
    batch = n if batch is None else min(int(batch), n)
    table = torch.zeros((n_features, k), dtype=table_dtype, device=device)
    bias = torch.zeros(k, device=device)
    table_grad, bias_grad = torch.empty((n_features, k), device=device), torch.empty(k, device=device)
    optimizer = AdamW([table, bias], [table_grad, bias_grad], lr=lr, weight_decay=[weight_decay, 0.0], l1=[l1, 0.0], state_bits=state_bits)
    draw = torch.Generator(device="cpu").manual_seed(int(seed))
    order, at, rows = None, 0, None
    for _ in range(int(steps)):
        if batch < n:
            if order is None or at + batch > n:
                order, at = torch.randperm(n, generator=draw).to(device=device, dtype=torch.int32), 0
            rows, at = order[at:at + batch], at + batch
        here = None if rows is None else rows.long()
        scores = row_scores(bits, table, bias, rows=rows)
        _, grad = sibling_loss(scores, label if here is None else label[here], weight=weight if here is None or weight is None else weight[here],
                               scale=1.0 / batch)
        row_scores_grad(bits, grad, n_features, rows=rows, out=(table_grad, bias_grad))
        optimizer.step()
    return torch.cat([bias[:, None], table.float().t()], 1).double().cpu().numpy()
