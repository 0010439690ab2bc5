"""Flags of the configuration benchmark (CPU)."""
import importlib.util
import os

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def parse_args():
    spec = importlib.util.spec_from_file_location("bench_configs", os.path.join(ROOT, "benchmarks", "bench_configs.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module.parse_args


@pytest.mark.parametrize("flags", [
    ["--config", "tp", "--ragged"],
    ["--config", "cppp", "--state-bits", "8"],
    ["--config", "tp", "--ragged", "--expert-dtype", "bf16"],
    ["--config", "moe", "--impl", "reference", "--ragged", "--expert-dtype", "bf16"],
    ["--config", "moe", "--impl", "reference", "--state-bits", "8"],
    ["--config", "moe", "--expert-dtype", "bf16"],
])
def test_flags_that_nothing_would_read_are_refused(parse_args, flags):
    with pytest.raises(SystemExit):
        parse_args(flags)


@pytest.mark.parametrize("flags", [
    ["--config", "tp"],
    ["--config", "moe", "--impl", "reference"],
    ["--config", "moe", "--ragged", "--expert-dtype", "bf16", "--state-bits", "8"],
    ["--config", "moe", "--state-bits", "8"],
])
def test_flags_that_count(parse_args, flags):
    assert parse_args(flags).config == flags[1]
