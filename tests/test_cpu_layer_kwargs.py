"""``ctor_kwargs`` builds a layer of the same form."""
import pytest


@pytest.mark.parametrize("sandwich", [False, True])
def test_graphormer_layer(sandwich):
    from graphgps_amd.layer.graphormer_layer import GraphormerLayer
    first = GraphormerLayer(32, 4, 0.1, 0.0, 0.0, sandwich=sandwich)
    again = GraphormerLayer(**first.ctor_kwargs)
    assert again.sandwich == sandwich and list(again.state_dict()) == list(first.state_dict())
    again.load_state_dict(first.state_dict())
