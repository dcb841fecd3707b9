"""bench.py's own arm keeps its line when the CPU baseline cannot be measured."""
import argparse

from test_bench_contract import _bench


def test_a_missing_reference_is_noted_in_the_line(monkeypatch, tmp_path):
    bench = _bench()
    monkeypatch.setattr(bench, 'REF_DIR', str(tmp_path / 'nothing_here'))
    line = bench.cpu_baseline_or_reason(argparse.Namespace(cpu_sample_tokens=16, layers=80))
    assert set(line) == {'unavailable'} and 'missing' in line['unavailable'] and len(line['unavailable']) <= 300


def test_a_measured_baseline_is_passed_on(monkeypatch):
    bench = _bench()
    monkeypatch.setattr(bench, 'cpu_baseline', lambda tokens, layers: {'value': tokens * layers})
    assert bench.cpu_baseline_or_reason(argparse.Namespace(cpu_sample_tokens=16, layers=80)) == {'value': 1280}
