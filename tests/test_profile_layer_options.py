"""Options of the command that make no sense are refused before anything is measured."""
import pytest

from superscaler_amd import profile_layer


@pytest.mark.parametrize("bad", [["--steps", "-1"], ["--policy-steps", "-2"]])
def test_numbers_of_steps(bad, monkeypatch, capsys):
    monkeypatch.setattr(profile_layer, "measure", lambda *a, **k: pytest.fail("measured"))
    with pytest.raises(SystemExit):
        profile_layer.main(["--workload", "gpt3_1_3b"] + bad)
    assert "0 or more" in capsys.readouterr().err
