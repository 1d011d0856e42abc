"""CPU: layers with rotary positions and norms, and layers from before they had these options, copied and pickled."""
import copy
import io

import pytest
import torch

from vision_longformer_amd import rotary
from vision_longformer_amd.longformer2d import Long2DSCSelfAttention
from vision_longformer_amd.msvit import Attention, Mlp


def through_a_pickle(x):
    f = io.BytesIO()
    torch.save(x, f)
    f.seek(0)
    return torch.load(f, map_location="cpu", weights_only=False)             # (written three lines above)


@pytest.mark.parametrize("how", [copy.deepcopy, copy.copy, through_a_pickle])
def test_a_grid_s_positions_do_not_travel(how):
    """they are kept by device: loaded onto another one they would be handed out for the first"""
    turn = rotary.GridTurn(32, base=100.0, layout="interleaved")
    made = turn.of(3, 2, 1, torch.device("cpu"))
    turn._made[(3, 2, 1, torch.device("cuda", 0))] = made                     # (what the first of several devices would have left)
    again = how(turn)
    assert again._made == {} and len(turn._made) == 2
    assert (again.sections, again.base, again.layout) == (turn.sections, turn.base, turn.layout)
    for k, v in again.of(3, 2, 1, torch.device("cpu")).items():
        assert torch.equal(v, made[k]) if torch.is_tensor(v) else v == made[k]
