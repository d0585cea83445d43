"""Steps with collectives are not captured."""
import types

import pytest
import torch

from distributed_pytorch_amd.parallel.graph import GraphedTrainStep


def test_an_engine_with_collectives_is_refused():
    engine = types.SimpleNamespace(_dist=True, device=torch.device("cuda"))
    with pytest.raises(RuntimeError, match="collectives"):
        GraphedTrainStep(engine)
