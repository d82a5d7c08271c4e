"""The benchmark's reference arm times the reference's compiled code or says that it is not there:
never the restatement of the test oracle under the reference's name."""
import argparse
import json


def test_reference_arm_without_the_reference(monkeypatch, capsys):
    import bench
    import oracle

    def restatement(*args, **kw):
        raise AssertionError("the restatement was timed")

    monkeypatch.setattr(oracle, "ref_lib", lambda: None)
    monkeypatch.setattr(oracle, "oracle_lib", restatement)
    monkeypatch.setattr(bench, "make_host_inputs", restatement)
    bench.run_reference(argparse.Namespace(gpus=1, steps=1, warmup=0), 0, 1)
    lines = capsys.readouterr().out.strip().splitlines()
    assert len(lines) == 1
    line = json.loads(lines[0])
    assert line["impl"] == "reference" and line["unavailable"] and "value" not in line
