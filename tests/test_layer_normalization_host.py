"""CPU: variables of layers.LayerNormalization."""
import numpy as np
import pytest
import torch

from agents_amd.networks import layers as L
from agents_amd.networks import sequential
from agents_amd.specs import tensor_spec


def weights(layer):
    net = sequential.Sequential([layer], input_spec=tensor_spec.TensorSpec((6,), torch.float32), seed=1)
    net.create_variables(device="cpu")
    return net.get_weights()


@pytest.mark.parametrize("kw,gamma,beta", [
    ({}, 1.0, 0.0), (dict(gamma_initializer="ones", beta_initializer="zeros"), 1.0, 0.0),
    (dict(gamma_initializer="zeros", beta_initializer="ones"), 0.0, 1.0),
    (dict(gamma_initializer=L.Constant(0.5), beta_initializer=L.Constant(-2.0)), 0.5, -2.0)])
def test_initializers(kw, gamma, beta):
    g, b = weights(L.LayerNormalization(**kw))
    np.testing.assert_array_equal(g, np.full(6, gamma, np.float32))
    np.testing.assert_array_equal(b, np.full(6, beta, np.float32))
