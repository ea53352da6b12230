"""The plain forms the GPU tests compare with, against answers worked out by hand, and the refusals of the entry points
that need no GPU: a refused call never looks behind its handles."""
import ctypes as C
import math

import numpy as np
import pytest

import policy_plain as P
from gym_amd import _lib as L

INF = math.inf


def test_order_and_cuts():
    x = [0.0, math.log(2.0), math.log(2.0), math.log(5.0)]  # probabilities .1 .2 .2 .5
    assert [P.sample_row(x, u)[0] for u in (0.0, 0.05, 0.15, 0.35, 0.55, 0.999)] == [0, 0, 1, 2, 3, 3]
    assert abs(P.sample_row(x, 0.15)[1] - math.log(0.2)) < 1e-15
    assert [P.sample_row(x, u, top_k=2)[0] for u in (0.0, 0.28, 0.29, 0.9)] == [1, 1, 3, 3]   # equal logits: the lower index
    assert [P.sample_row(x, u, top_p=0.6)[0] for u in (0.0, 0.28, 0.29)] == [1, 1, 3]
    assert [P.sample_row(x, u, top_p=0.0)[0] for u in (0.0, 0.9)] == [3, 3]
    assert [P.sample_row(x, u, min_p=0.3)[0] for u in (0.0, 0.3, 0.9)] == [1, 2, 3]
    # top_p is a share of what top_k left: .5 + .2 = .7 is all of it
    assert [P.sample_row(x, u, top_k=2, top_p=0.71)[0] for u in (0.0, 0.9)] == [3, 3]
    assert P.sample_row(x, 0.1, temperature=0)[0] == 3 and P.sample_row([1, 1], 0.9, temperature=0) == (0, 0.0)


def test_masked_rows():
    assert P.sample_row([-INF, -INF], 0.5) == (-1, -INF)
    assert P.sample_row([-INF, 3.0, math.nan], 0.99) == (1, 0.0)
    assert P.sample_row([0.0, INF, -INF, INF], 0.6)[0] == 3
    low = -3.4028234663852886e38
    assert [P.sample_row([low, low], u)[0] for u in (0.2, 0.7)] == [0, 1]
    assert P.sample_row([low, -INF, low / 2], 0.0, temperature=0.5)[0] == 2


def test_embed_grad():
    t, size, count = P.embed_grad([[1.0, 2.0], [3.0, -4.0], [5.0, 6.0], [7.0, 7.0]], [1, 1, 3, 0], 3, 2.0)
    assert t.tolist() == [[14, 14], [8, -4], [0, 0]] and size.tolist() == [[14, 14], [8, 12], [0, 0]]
    assert count.tolist() == [1, 2, 0]


# --------------------------------------------------------------------- refusals ---
HANDLE = C.create_string_buffer(4096)  # stands for a context: nothing reads it before the arguments have passed
BUF = C.create_string_buffer(4096)
AT = (C.addressof(BUF) + 255) & ~255


def _sample(**kw):
    s = L.GxSample(C.sizeof(L.GxSample), 0, L.F32, 4, 8, 4, 1, AT, AT, None, None, None, None, 1.0, 0, 1.0, 0.0, AT, AT, None, 0)
    for k, v in kw.items():
        setattr(s, k, v)
    return s


@pytest.mark.parametrize("change,code,word", [
    (dict(struct_size=8), L.GX_ERR_INVALID, "struct_size"),
    (dict(op_flags=2), L.GX_ERR_INVALID, "op_flags"),
    (dict(logits_dtype=L.F64), L.GX_ERR_UNSUPPORTED, "dtype"),
    (dict(n_actions=0), L.GX_ERR_INVALID, "n_actions"),
    (dict(n_actions=(1 << 24) + 1), L.GX_ERR_INVALID, "n_actions"),
    (dict(rows=(1 << 40) + 1), L.GX_ERR_INVALID, "rows"),
    (dict(row_stride=-4), L.GX_ERR_INVALID, "stride"),
    (dict(col_stride=-1), L.GX_ERR_INVALID, "stride"),
    (dict(row_stride=1 << 58), L.GX_ERR_INVALID, "2^60"),
    (dict(col_stride=1 << 62), L.GX_ERR_INVALID, "2^60"),
    (dict(temperature_all=-0.5), L.GX_ERR_INVALID, "temperature"),
    (dict(temperature_all=math.nan), L.GX_ERR_INVALID, "temperature"),
    (dict(top_k_all=-1), L.GX_ERR_INVALID, "top_k"),
    (dict(top_p_all=1.5), L.GX_ERR_INVALID, "top_p"),
    (dict(top_p_all=math.nan), L.GX_ERR_INVALID, "top_p"),
    (dict(min_p_all=-0.1), L.GX_ERR_INVALID, "min_p"),
    (dict(logits=None), L.GX_ERR_INVALID, "logits"),
    (dict(actions=None), L.GX_ERR_INVALID, "actions"),
    (dict(u=None), L.GX_ERR_INVALID, "random numbers"),
    (dict(logits=AT + 2), L.GX_ERR_INVALID, "aligned"),
    (dict(actions=AT + 2), L.GX_ERR_INVALID, "aligned"),
    (dict(top_p=AT + 1), L.GX_ERR_INVALID, "aligned"),
])
def test_sample_refusals(change, code, word):
    lib = L.load()
    assert lib.gx_sample_logits(HANDLE, C.byref(_sample(**change)), None) == code
    assert word in lib.gx_last_error().decode()


def _embed(**kw):
    e = L.GxEmbed(C.sizeof(L.GxEmbed), 0, L.F32, L.F32, L.I32, 0, 8, 16, 4, 4, 4, AT, AT, AT, None, 0, 1.0, 0)
    for k, v in kw.items():
        setattr(e, k, v)
    return e


@pytest.mark.parametrize("change,code,word", [
    (dict(struct_size=8), L.GX_ERR_INVALID, "struct_size"),
    (dict(op_flags=4), L.GX_ERR_INVALID, "op_flags"),
    (dict(table_dtype=L.I32), L.GX_ERR_UNSUPPORTED, "dtype"),
    (dict(rows_dtype=L.F64), L.GX_ERR_UNSUPPORTED, "dtype"),
    (dict(ids_dtype=L.U8), L.GX_ERR_UNSUPPORTED, "ids"),
    (dict(tokens=1 << 31), L.GX_ERR_INVALID, "tokens"),
    (dict(n_states=0), L.GX_ERR_INVALID, "n_states"),
    (dict(n_states=1 << 31), L.GX_ERR_INVALID, "n_states"),
    (dict(dim=0), L.GX_ERR_INVALID, "dim"),
    (dict(dim=(1 << 24) + 1), L.GX_ERR_INVALID, "dim"),
    (dict(table_stride=3), L.GX_ERR_INVALID, "overlap"),
    (dict(rows_stride=3), L.GX_ERR_INVALID, "overlap"),
    (dict(rows_stride=1 << 60), L.GX_ERR_INVALID, "2^60"),
    (dict(table=None), L.GX_ERR_INVALID, "table"),
    (dict(rows=None), L.GX_ERR_INVALID, "rows"),
    (dict(ids=None), L.GX_ERR_INVALID, "ids"),
    (dict(table=AT + 2), L.GX_ERR_INVALID, "aligned"),
    (dict(ids_dtype=L.I64, ids=AT + 4), L.GX_ERR_INVALID, "aligned"),
    (dict(scale=math.inf), L.GX_ERR_INVALID, "scale"),
    (dict(scale=math.nan), L.GX_ERR_INVALID, "scale"),
])
def test_embed_refusals(change, code, word):
    lib = L.load()
    for fn in (lib.gx_embed_lookup, lib.gx_embed_grad):
        assert fn(HANDLE, C.byref(_embed(**change)), None) == code
        assert word in lib.gx_last_error().decode()


def test_null_arguments():
    lib = L.load()
    size = C.c_uint64()
    s, e = C.byref(_sample()), C.byref(_embed())
    for rc in (lib.gx_sample_logits(None, s, None), lib.gx_sample_logits(HANDLE, None, None),
               lib.gx_sample_workspace(None, s, C.byref(size)), lib.gx_sample_workspace(HANDLE, s, None),
               lib.gx_vec_step_logits(None, s, None), lib.gx_embed_lookup(None, e, None), lib.gx_embed_grad(HANDLE, None, None),
               lib.gx_embed_grad_workspace(HANDLE, None, C.byref(size)), lib.gx_vec_embed_obs(None, e, None)):
        assert rc == L.GX_ERR_INVALID and b"null" in lib.gx_last_error()


def test_struct_sizes():
    assert C.sizeof(L.GxSample) == 136 and C.sizeof(L.GxEmbed) == 112


@pytest.mark.parametrize("c_name,cs_name,ct", [("gx_sample", "GxSample", L.GxSample), ("gx_embed", "GxEmbed", L.GxEmbed)])
def test_struct_fields_agree_in_all_three_languages(c_name, cs_name, ct):
    import test_csharp_conformance as T

    c, cs = T.header_struct(c_name), T.csharp_struct(cs_name)
    assert [T._norm(n) for n, _ in c] == [T._norm(n) for n, _ in cs] == [T._norm(f[0]) for f in ct._fields_]
    assert T._layout(c) == T._layout(cs) == ([getattr(ct, f[0]).offset for f in ct._fields_], C.sizeof(ct))
    assert T.header_enum("gx_op_flags") == {"GX_OP_DEFAULT_STREAM": L.OP_DEFAULT_STREAM}
    assert T.csharp_enum("GxOpFlags") == {"None": 0, "DefaultStream": L.OP_DEFAULT_STREAM}


def test_python_refuses_host_tensors():
    import torch

    from gym_amd import policy

    x, u, ids = torch.zeros(2, 3), torch.zeros(2), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="GPU"):
        policy.sample_logits(x, u)
    with pytest.raises(TypeError, match="torch tensor"):
        policy.sample_logits(np.zeros((2, 3), np.float32), u)
    with pytest.raises(ValueError, match="GPU"):
        policy.embed_lookup(x, ids)
    with pytest.raises(ValueError, match="GPU"):
        policy.embed_grad(x, ids, 4)
