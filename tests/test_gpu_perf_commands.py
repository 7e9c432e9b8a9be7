"""The measuring commands of the operators behind the collectives run and report."""
import pytest

from flagcx_amd import perf

pytestmark = pytest.mark.gpu


def test_norm_and_experts_commands(capsys):
    perf.main(["norm", "-k", "2", "-d", "bf16", "--cols", "640", "-b", "1", "-e", "8", "-f", "8"])
    out = capsys.readouterr().out
    assert out.count("GB/s") == 6 and "to e4m3" in out and "gradients" in out
    perf.main(["experts", "-d", "fp16", "--experts", "4", "--cols", "256", "--width", "384", "-b", "8", "-e", "64", "-f", "8"])
    out = capsys.readouterr().out
    assert out.count("TFLOP/s") == 8 and "dW = dy^T x" in out and "e4m3" in out


def test_norm_command_with_fewer_rows_in_the_workspace_of_more(capsys):
    perf.main(["norm", "-k", "1", "-d", "bf16", "--cols", "8192", "-b", "256", "-e", "300", "-f", "2"])
    assert capsys.readouterr().out.count("GB/s") == 3
