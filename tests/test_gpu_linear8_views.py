"""Columns of tensors that other nodes write again, on the GPU against the oracle, which copies them."""
import numpy as np
import pytest

from oracle import graph_sim as og
from test_linear8_views import SHAPE, small, viewed, written_again  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def torch_gpu():
    import torch
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return torch


def same(got, want, what):
    for name, v in got.items():
        np.testing.assert_array_equal(v, np.asarray(want[name]).reshape(v.shape), err_msg=f"{what}: {name}")


@pytest.mark.parametrize("kind", ["columns", "reshape"])
@pytest.mark.parametrize("weights8", [False, True])
def test_views_of_attention_rows_outlive_the_next_layer(small, kind, weights8):  # noqa: F811
    """Views of every layer's attention rows, read by the o projection and returned behind the last layer."""
    from cormorant_amd.simulate import Simulator
    g, views = viewed(small, kind, weights8)
    g.output_tensors = g.output_tensors + views
    f = {"ids": np.random.default_rng(1).integers(0, SHAPE.vocab, 6).astype(np.float64), "q_start": np.array([0.0, 4, 6]),
         "kv_len": np.array([4.0, 2]), "table": np.array([[3.0, 1, 6], [0, 7, 2]])}
    st = {t.onnx_name: np.zeros(t.shape) for t in g.state_tensors}
    want = og.forward(g, f, states={k: v.copy() for k, v in st.items()})
    assert (want[views[0].onnx_name] != want[views[1].onnx_name]).any()
    same(Simulator(g)._forward_pass(f, states=st, keep=[t.onnx_name for t in g.output_tensors]), want, kind)


@pytest.mark.parametrize("kind", ["state", "reshape"])
def test_columns_of_a_state_written_later(kind):
    from cormorant_amd.simulate import Simulator
    g, f, c = written_again(kind)
    states = {"x": f.pop("x")}
    want = og.forward(g, f, states={k: v.copy() for k, v in states.items()})[c.onnx_name]
    for _ in range(2):
        got = Simulator(g)._forward_pass(f, states={k: v.copy() for k, v in states.items()}, keep=[c.onnx_name])
        np.testing.assert_array_equal(got[c.onnx_name], want)
