"""packed_towers and fp8_towers from the command line and from the JSON config, as eval_itm / train_itm read them."""
import json

import pytest

from lightningdot_amd.options import build_parser, parse_with_config
from lightningdot_amd.towers import BiEncoder, TowerConfig


@pytest.mark.parametrize('packed', [False, True])
@pytest.mark.parametrize('fp8', [False, True])
@pytest.mark.parametrize('config', [False, True])
def test_tower_options(packed, fp8, config, tmp_path):
    wanted = dict(packed_towers=packed, fp8_towers=fp8)
    if config:
        (tmp_path / 'c.json').write_text(json.dumps(wanted))
        cmds = ['--config', str(tmp_path / 'c.json')]
    else:
        cmds = ['--' + k for k, v in wanted.items() if v]
    args = parse_with_config(build_parser(), cmds)
    assert getattr(args, 'packed_towers', False) is packed and getattr(args, 'fp8_towers', False) is fp8
    cfg = TowerConfig(vocab_size=50, hidden_size=32, num_hidden_layers=1, num_attention_heads=2, intermediate_size=64, max_position_embeddings=16)
    be = BiEncoder(args, project_dim=16, txt_config=cfg, img_config=cfg)
    for tower in (be.txt_model, be.img_model):
        assert tower.bert.packed is packed and tower.bert.fp8 is fp8


def test_the_command_line_wins(tmp_path):
    (tmp_path / 'c.json').write_text(json.dumps(dict(packed_towers=False)))
    assert parse_with_config(build_parser(), ['--config', str(tmp_path / 'c.json'), '--packed_towers']).packed_towers is True
