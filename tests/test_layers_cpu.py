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


def before_the_options(m):
    """the module as a pickle from before the options holds it"""
    state = {k: v for k, v in m.__dict__.items() if k not in ("q_norm", "k_norm", "turn", "act8")}
    old = type(m).__new__(type(m))
    old.__setstate__(state)
    return old


def test_layers_pickled_before_the_options_run():
    x = torch.randn(2, 17, 32)
    for m in (Attention(32, num_heads=2, rpe=True, wx=4, wy=4, nglo=1), Mlp(32, 64), Long2DSCSelfAttention(32, num_heads=2, w=4, sharew=True)):
        old = before_the_options(m)
        assert [n for n, _ in old.named_modules()] == [n for n, _ in m.named_modules()]
        if isinstance(m, Long2DSCSelfAttention):
            assert old.q_norm is None and old.k_norm is None and old.turn is None        # (runs on the device alone)
        else:
            args = (x, 4, 4) if isinstance(m, Attention) else (x,)
            assert torch.equal(old(*args), m(*args))


def test_layers_with_the_options_keep_them_through_a_pickle():
    for m in (Attention(32, num_heads=2, wx=4, wy=4, qk_norm=True, rotary=True),
              Long2DSCSelfAttention(32, num_heads=2, w=4, sharew=True, qk_norm=True, rotary=True), Mlp(32, 64, act8=True)):
        for again in (copy.deepcopy(m), through_a_pickle(m)):
            assert list(again.state_dict()) == list(m.state_dict())
            if isinstance(m, Mlp):
                assert again.act8
            else:
                assert torch.equal(again.q_norm.weight, m.q_norm.weight) and again.turn.sections == m.turn.sections
