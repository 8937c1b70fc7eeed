"""Package resource locations, resolved from this file (reference: tilebench/paths.py:22-60,192-206)."""
from __future__ import annotations

import os
from pathlib import Path

PACKAGE_ROOT = Path(__file__).resolve().parent
DATA_ROOT = PACKAGE_ROOT / "data"
OPERATOR_ROOT = PACKAGE_ROOT / "benchmarks" / "operators"
#: Operators of a model's layers (forward and backward pass); same layout and contract as OPERATOR_ROOT.
LAYER_ROOT = PACKAGE_ROOT / "benchmarks" / "layers"
PEAK_PERFORMANCE_ROOT = DATA_ROOT / "peak_performance"
REPO_ROOT = Path(os.environ.get("TILEBENCH_REPO_ROOT") or PACKAGE_ROOT.parent).resolve()
RESULTS_ROOT = REPO_ROOT / "results"


def operator_dir(name: str) -> Path:
    return (LAYER_ROOT if name in list_layer_operators() else OPERATOR_ROOT) / name


def operator_package(name: str) -> str:
    """The Python package that holds an operator's impl_torch and impl_cuda."""
    return f"tilebench_b200.benchmarks.{operator_dir(name).parent.name}.{name}"


def operator_config(name: str) -> Path:
    return operator_dir(name) / "config.yaml"


def _operators_in(root: Path) -> list[str]:
    if not root.is_dir():
        return []
    return sorted(p.name for p in root.iterdir() if (p / "config.yaml").is_file())


def list_operators() -> list[str]:
    """Every operator directory that has a config.yaml, sorted."""
    return _operators_in(OPERATOR_ROOT)


def list_layer_operators() -> list[str]:
    """The same for the operators of a model's layers."""
    return _operators_in(LAYER_ROOT)


def results_csv_dir(gpu: str) -> Path:
    return RESULTS_ROOT / gpu / "csv"


def results_logs_dir(gpu: str) -> Path:
    return RESULTS_ROOT / gpu / "logs"
