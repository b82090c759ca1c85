"""CPU: what the Embedding encoding refuses when it is made."""
import pytest

from rise_sdf_amd import Config
from rise_sdf_amd.network_utils import get_encoding


@pytest.mark.parametrize("padding", [-1, 7, -7, 100])
def test_padding_outside_the_codes(padding):
    """Not only at the first lookup: a negative one would clear a code that is used."""
    with pytest.raises(ValueError, match="padding_idx"):
        get_encoding(1, Config({"otype": "Embedding", "n_embeddings": 7, "n_features": 5, "padding_idx": padding}))


@pytest.mark.parametrize("padding", [None, 0, 6])
def test_padding_inside_the_codes(padding):
    e = get_encoding(1, Config({"otype": "Embedding", "n_embeddings": 7, "n_features": 5, "padding_idx": padding}))
    zero = [i for i in range(7) if not bool(e.params[i].any())]
    assert zero == ([] if padding is None else [padding])
