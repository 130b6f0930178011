"""p0pc0rn_amd.f8_layer's refusals, which come before any device work (no GPU)."""
from types import SimpleNamespace

import numpy as np
import pytest

from p0pc0rn_amd import f8_layer as L


@pytest.mark.parametrize("rows,pos", [((2, 0, 64), (1, 2, 0)), ((1, 3, 64), (1, 1, 3)), ((2, 3, 65), (1, 2, 3)), ((2, 3, 64), (2, 2, 3)), ((2, 3, 64), (1, 2, 4)),
                                      ((2, 64), (1, 2, 1))])
def test_rows_and_positions_of_another_shape(rows, pos):
    run = object.__new__(L.Run)
    run.m, run.B, run.most, run.longest, run.length = SimpleNamespace(K=64, axis_dim=[32]), 2, 8, 100, 0
    with pytest.raises(ValueError, match="2 sequences of 64 channels, 1 axes"):
        run.step(np.zeros(rows), np.zeros(pos))


def test_a_decoder_has_a_layer():
    with pytest.raises(ValueError, match="0 layers"):
        L.Decoder(0)


@pytest.mark.parametrize("args", [["--prompt", "0"], ["--prompt", "-4"], ["--tokens", "-1"]])
def test_the_command_refuses_nothing_to_run(args, monkeypatch, capsys):
    monkeypatch.setattr("sys.argv", ["f8_layer"] + args)
    with pytest.raises(SystemExit) as e:
        L.main()
    assert e.value.code == 2 and "at least one row" in capsys.readouterr().err
