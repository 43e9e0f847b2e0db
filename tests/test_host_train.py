"""CPU-only checks of the training operators: libstag_train.so exports what include/stag_train.h declares, and both levels
refuse what they cannot do before anything reaches a GPU."""
import copy
import ctypes
import os
import pickle
import re

import numpy as np
import pytest
import torch

from stag_amd import _lib, train

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = 4096          # a pointer that is aligned to everything and never followed


def test_library_exports_every_declared_symbol():
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "stag_train.h")).read(), flags=re.S)
    names = set(re.findall(r"\b(stag_[a-z0-9_]+)\s*\(", text))
    L = ctypes.CDLL(_lib.TRAIN_LIB_PATH)
    for name in names:
        assert hasattr(L, name), name
    assert names == set(_lib.TRAIN_EXPORTS), names ^ set(_lib.TRAIN_EXPORTS)


def test_descriptors_have_the_layout_of_the_header():
    assert train._TENSOR.itemsize == 48
    assert [train._TENSOR.fields[f][1] for f in ("param", "grad", "count", "state_at", "weight_decay", "l1", "param_type", "grad_type")] == \
        [0, 8, 16, 24, 32, 36, 40, 44]


def test_workspaces_of_every_size():
    L = _lib.train_lib()
    for m in (0, 1, 63, 64, 65, 1000, 100000, 2**31 - 1):
        for f in (1, 31, 7500, 157500, 1 << 27):
            for k in (1, 13, 64, 1000, 1 << 20):
                for kind in range(3):
                    assert L.stag_row_scores_workspace(m, f, k, kind) >= 0
                    assert L.stag_row_scores_grad_workspace(m, f, k, kind) >= 0
            assert L.stag_sibling_loss_workspace(m, k) >= 0


SCORES = dict(bits=P, n=10, row_stride=4, n_features=100, rows=None, m=10, table=P, type=0, table_stride=3, bias=None, k=3, scale=1.0, scores=P,
              score_stride=3, work=P, work_bytes=1 << 40, stream=None)


@pytest.mark.parametrize("change, message", [
    (dict(type=3), "unknown type"), (dict(n_features=0), "n_features"), (dict(k=0), "k = 0"), (dict(k=1 << 21), "k = "), (dict(m=-1), "m = -1"),
    (dict(m=11), "without d_rows"), (dict(row_stride=3), "row_stride"), (dict(row_stride=0), "row_stride"), (dict(n_features=129), "row_stride"),
    (dict(bits=None), "d_bits"), (dict(bits=P + 4), "d_bits"), (dict(table=None), "d_table"), (dict(table=P + 2), "d_table"),
    (dict(table_stride=2), "d_table's stride"), (dict(scores=None), "d_scores"), (dict(score_stride=2), "d_scores's stride"), (dict(bias=P + 1), "d_bias"),
    (dict(rows=P + 2), "d_rows"), (dict(n=-1, rows=P), "n = -1"), (dict(m=1 << 31, rows=P), "m = "),
    (dict(m=(1 << 31) - 1, rows=P), "2147483647 rows of 3 columns are too many"),
])
def test_scores_refusals(change, message):
    rc = _lib.train_lib().stag_row_scores_dev(*{**SCORES, **change}.values())
    assert rc == -1 and message in _lib.train_lib().stag_train_last_error().decode()


GRAD = dict(bits=P, n=10, row_stride=4, n_features=100, rows=None, m=10, grad=P, type=0, grad_stride=3, k=3, scale=1.0, table_grad=P,
            table_grad_stride=3, bias_grad=P, work=P, work_bytes=1 << 40, stream=None)


@pytest.mark.parametrize("change, message", [
    (dict(type=-1), "unknown type"), (dict(n_features=0), "n_features"), (dict(k=0), "k = 0"), (dict(m=11), "without d_rows"),
    (dict(grad=None), "d_grad"), (dict(grad=P + 2), "d_grad"), (dict(grad_stride=2), "d_grad's stride"), (dict(table_grad=P + 2), "d_table_grad"),
    (dict(table_grad_stride=2), "d_table_grad's stride"), (dict(bias_grad=P + 2), "d_bias_grad"), (dict(bits=P + 8), "d_bits"),
])
def test_grad_refusals(change, message):
    rc = _lib.train_lib().stag_row_scores_grad_dev(*{**GRAD, **change}.values())
    assert rc == -1 and message in _lib.train_lib().stag_train_last_error().decode()


LOSS = dict(scores=P, score_stride=3, m=10, k=3, label=P, siblings=None, weight=None, scale=1.0, loss=P, grad=P, type=0, grad_stride=3, work=P,
            work_bytes=1 << 40, stream=None)


@pytest.mark.parametrize("change, message", [
    (dict(type=9), "unknown type"), (dict(k=0), "k = 0"), (dict(m=-5), "m = -5"), (dict(scores=None), "d_scores"), (dict(score_stride=2), "stride"),
    (dict(label=None), "d_label"), (dict(siblings=P + 1), "d_siblings"), (dict(weight=P + 2), "d_weight"), (dict(grad=P + 2), "d_grad"),
    (dict(grad_stride=0), "d_grad's stride"), (dict(m=100000, work_bytes=16), "d_work"), (dict(m=100000, work=P + 16), "d_work"),
])
def test_loss_refusals(change, message):
    rc = _lib.train_lib().stag_sibling_loss_dev(*{**LOSS, **change}.values())
    assert rc == -1 and message in _lib.train_lib().stag_train_last_error().decode()


ADAMW = dict(tensors=P, tiles=P, n_tiles=1, bits=32, m=P, v=P, m_scale=None, v_scale=None, step=P, lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, stream=None)


@pytest.mark.parametrize("change, message", [
    (dict(bits=16), "state_bits"), (dict(n_tiles=-1), "n_tiles"), (dict(lr=-1.0), "lr"), (dict(lr=float("nan")), "lr"), (dict(beta1=1.0), "beta1"),
    (dict(beta2=0.0), "beta2"), (dict(eps=-1.0), "eps"), (dict(tensors=None), "d_tensors"), (dict(m=P + 4), "d_m"), (dict(bits=8), "scales"), (dict(step=P + 1), "d_step"),
])
def test_adamw_refusals(change, message):
    rc = _lib.train_lib().stag_adamw_dev(*{**ADAMW, **change}.values())
    assert rc == -1 and message in _lib.train_lib().stag_train_last_error().decode()


# ---------------------------------------------------------------------------------------------------- the Python level
def rows(n=6, words=4):
    return torch.zeros((n, words), dtype=torch.int32)


@pytest.mark.parametrize("call, error, message", [
    (lambda: train.row_scores(rows(), torch.zeros(100, 3)), ValueError, "on cpu"),
    (lambda: train.row_scores(np.zeros((6, 4), np.int32), torch.zeros(100, 3)), TypeError, "bits must be a torch tensor"),
    (lambda: train.row_scores(rows().long(), torch.zeros(100, 3)), TypeError, "bits is torch.int64"),
    (lambda: train.row_scores(rows(), torch.zeros(100, 3).double()), TypeError, "table is torch.float64"),
    (lambda: train.row_scores(rows(), torch.zeros(100)), ValueError, "table has 1 dimensions"),
    (lambda: train.row_scores(rows(), torch.zeros(100, 0)), ValueError, "table is empty"),
    (lambda: train.row_scores(rows(), torch.zeros(100, 3), torch.zeros(2)), ValueError, "bias has 2 values"),
    (lambda: train.row_scores(rows(), torch.zeros(100, 3), rows=torch.zeros(5)), TypeError, "rows is"),
    (lambda: train.row_scores(rows(), torch.zeros(100, 3), out=torch.zeros(5, 3)), ValueError, "out has shape"),
    (lambda: train.row_scores(rows(), torch.zeros(100, 3), out=torch.zeros(3, 6).t()), ValueError, "out must have contiguous rows"),
    (lambda: train.row_scores(rows(), torch.zeros(100, 3), out=torch.zeros(1, 3).expand(6, 3)), ValueError, "do not overlap"),
    (lambda: train.row_scores_grad(rows(), torch.zeros(5, 3), 100), ValueError, "grad has 5 rows"),
    (lambda: train.row_scores_grad(rows(), torch.zeros(6, 3), 0), ValueError, "no features"),
    (lambda: train.row_scores_grad(rows(), torch.zeros(6, 3).int(), 100), TypeError, "grad is torch.int32"),
    (lambda: train.row_scores_grad(rows(), torch.zeros(6, 3), 100, out=(torch.zeros(99, 3), torch.zeros(3))), ValueError, "out[0] has shape"),
    (lambda: train.sibling_loss(torch.zeros(6, 3), torch.zeros(5).int()), ValueError, "label has 5 values"),
    (lambda: train.sibling_loss(torch.zeros(6, 3), torch.zeros(6)), TypeError, "label is"),
    (lambda: train.sibling_loss(torch.zeros(6, 3).half(), torch.zeros(6).int()), TypeError, "scores is"),
    (lambda: train.sibling_loss(torch.zeros(6, 3), torch.zeros(6).int(), siblings=torch.zeros(6, 3).int()), ValueError, "siblings has shape"),
    (lambda: train.sibling_loss(torch.zeros(6, 3), torch.zeros(6).int(), weight=torch.zeros(2)), ValueError, "weight has 2 values"),
    (lambda: train.sibling_loss(torch.zeros(6, 3), torch.zeros(6).int(), grad_dtype=torch.float64), TypeError, "grad_dtype"),
    (lambda: train.AdamW([], []), ValueError, "no parameters"),
    (lambda: train.AdamW([torch.zeros(3)], []), ValueError, "1 parameters, 0 gradients"),
    (lambda: train.AdamW([torch.zeros(3)], [torch.zeros(4)]), ValueError, "its gradient"),
    (lambda: train.AdamW([torch.zeros(3)], [torch.zeros(3)], state_bits=16), ValueError, "state_bits"),
    (lambda: train.AdamW([torch.zeros(3)], [torch.zeros(3)], betas=(0.9, 1.0)), ValueError, "betas"),
    (lambda: train.AdamW([torch.zeros(3)], [torch.zeros(3)], l1=-1.0), ValueError, "not negative"),
    (lambda: train.AdamW([torch.zeros(3)], [torch.zeros(3)], weight_decay=[0.0, 0.0]), ValueError, "one for each"),
    (lambda: train.AdamW([torch.zeros(4, 4).t()], [torch.zeros(4, 4)]), ValueError, "not contiguous"),
    (lambda: train.AdamW([torch.zeros(3).double()], [torch.zeros(3)]), TypeError, "params[0] must be"),
    (lambda: train.AdamW([torch.zeros(3)], [torch.zeros(3)]), ValueError, "on cpu"),
])
def test_python_refusals(call, error, message):
    with pytest.raises(error, match=re.escape(message)):
        call()


def test_too_narrow_and_unaligned_rows():
    with pytest.raises(ValueError, match="too few for 129 features"):
        train._packed(rows(6, 4), 129)
    with pytest.raises(ValueError, match="16-byte units"):
        train._packed(rows(6, 8)[:, 1:7], 100)
    bits, stride = train._packed(rows(6, 8)[:, :4], 100)
    assert stride == 8
    assert train._packed(rows(8, 8).t(), 100)[1] == 8       # copied to contiguous rows


def test_sizes_that_32_bits_would_wrap_are_refused():
    for name, *sizes in (("stag_row_scores_workspace", 1, 2**32 + 5, 3, 0), ("stag_row_scores_workspace", 1, 5, 2**32 + 3, 0),
                         ("stag_row_scores_grad_workspace", 1, 2**32 + 5, 3, 0), ("stag_sibling_loss_workspace", 1, 2**32 + 3)):
        with pytest.raises(ValueError, match="sizes of 2"):
            train._workspace(name, *sizes)
    with pytest.raises(_lib.StagError, match="m = 4294967301"):
        train._workspace("stag_sibling_loss_workspace", 2**32 + 5, 3)


def test_rows_far_apart_are_copied_or_refused():
    """A matrix whose rows lie more than 2^21 values apart: inputs are copied, outputs refused, and so is the stride at the C entry."""
    wide = torch.empty(2, 2**21 + 8)[:, :3]
    assert train._rows(wide)[1] == 3 and train._rows(torch.empty(2, 2**21)[:, :3])[1] == 2**21
    with pytest.raises(ValueError, match="rows more than 2097152 values apart"):
        train._out_rows("out", wide, (2, 3), torch.float32)
    for args, which, name in ((SCORES, "table_stride", "d_table"), (SCORES, "score_stride", "d_scores")):
        assert _lib.train_lib().stag_row_scores_dev(*{**args, which: 2**21 + 1}.values()) == -1
        message = _lib.train_lib().stag_train_last_error().decode()
        assert name in message and "is over 2097152" in message


def test_outputs_that_share_memory():
    """Only tensors that have a byte in common: columns of one buffer beside one another do not."""
    buffer = torch.zeros(6, 20)
    share = train._share
    assert not share(buffer[:, :5], buffer[:, 5:9]) and not share(buffer[:, 5:9], buffer[:, :5]) and not share(buffer[:, 15:], buffer[:, :15])
    assert share(buffer[:, :5], buffer[:, 4:9]) and share(buffer[:, 4:9], buffer[:, :5]) and share(buffer[:, 3:4], buffer)
    assert not share(buffer[:3], buffer[3:]) and share(buffer[:3], buffer[2:])
    assert share(buffer[2, 3:9], buffer[:, 8:10]) and not share(buffer[2, 3:8], buffer[:, 8:10]) and not share(buffer[0], buffer[1])
    assert share(buffer.view(12, 10)[:, :3], buffer[:, 10:13]) and not share(buffer, buffer.clone()) and not share(buffer[:0], buffer)
    assert share(buffer.view(torch.int32), buffer) and share(buffer.flatten(), buffer[:, 2:3])
    with pytest.raises(ValueError, match=re.escape("out[1] and scores share memory")):
        train._apart({"out[0]": torch.zeros(3), "out[1]": buffer}, {"label": None, "scores": buffer})
    with pytest.raises(ValueError, match=re.escape("out[0] and out[1] share memory")):
        train._apart({"out[0]": buffer[0], "out[1]": buffer}, {})


def test_an_optimizer_is_not_copied():
    """It holds addresses: a copy's would be those of the tensors copied from."""
    opt = train.AdamW.__new__(train.AdamW)
    for call in (copy.copy, copy.deepcopy, pickle.dumps):
        with pytest.raises(TypeError, match="load_state"):
            call(opt)
    for name in ("params", "grads", "m", "v", "device"):
        with pytest.raises(AttributeError):
            setattr(opt, name, None)


@pytest.mark.parametrize("change, error, message", [
    (dict(bits=np.zeros((6, 16), np.uint8)), TypeError, "bits is uint8"),
    (dict(bits=torch.zeros(6, dtype=torch.int32)), ValueError, "bits has 1 dimensions"),
    (dict(bits=rows(0)), ValueError, "no rows"),
    (dict(k=0), ValueError, "no classifiers (0)"),
    (dict(n_features=0), ValueError, "no features (0)"),
    (dict(label=np.zeros(6)), TypeError, "label is torch.float64"),
    (dict(label=np.zeros(7, int)), ValueError, "label has shape (7,)"),
    (dict(weight=np.ones(7)), ValueError, "weight has shape (7,)"),
    (dict(batch=0), ValueError, "batch = 0"),
    (dict(), ValueError, "on cpu"),
])
def test_fit_siblings_refusals(change, error, message):
    with pytest.raises(error, match=re.escape(message)):
        train.fit_siblings(**{**dict(bits=rows(), label=np.zeros(6, int), k=2, n_features=100), **change})
