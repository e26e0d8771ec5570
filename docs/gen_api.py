"""Regenerate ``docs/api.md``: the public classes and functions of every user-facing module with their
signatures and their docstrings: the first paragraph of a module's, a class's or a method's, all of a function's.

    python docs/gen_api.py            # rewrite docs/api.md
    python docs/gen_api.py --check    # exit 1 if docs/api.md is out of date
"""

from __future__ import annotations

import importlib
import inspect
import os
import re
import sys
from pathlib import Path

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))
os.environ.setdefault("TORCHFT_USE_OTEL", "false")

MODULES = [
    ("torchft_b200", "top-level exports"),
    ("torchft_b200.manager", "per-rank fault-tolerance state machine"),
    ("torchft_b200.coordination", "lighthouse / manager servers and clients (C++ control plane)"),
    ("torchft_b200.optim", "commit-gated optimizer wrapper"),
    ("torchft_b200.ddp", "fault-tolerant DistributedDataParallel"),
    ("torchft_b200.data", "sampler over replica groups x ranks"),
    ("torchft_b200.local_sgd", "LocalSGD, DiLoCo, streaming DiLoCo"),
    ("torchft_b200.process_group", "reconfigurable process groups"),
    ("torchft_b200.process_group_baby", "process groups isolated in a child process"),
    ("torchft_b200.device_mesh", "device mesh with a managed replica dimension"),
    ("torchft_b200.collectives", "quantised collectives"),
    ("torchft_b200.quantization", "fp8 block quantisation"),
    ("torchft_b200.futures", "timeouts for futures, streams and code blocks"),
    ("torchft_b200.work", "completed-work helper"),
    ("torchft_b200.multiprocessing", "pipe with timeouts"),
    ("torchft_b200.multiprocessing_dummy_context", "thread-backed multiprocessing context for tests"),
    ("torchft_b200.parameter_server", "parameter-server prototype"),
    ("torchft_b200.otel", "structured event loggers"),
    ("torchft_b200.checkpointing.transport", "checkpoint transport interface"),
    ("torchft_b200.checkpointing.http_transport", "HTTP transport"),
    ("torchft_b200.checkpointing.pg_transport", "process-group transport"),
    ("torchft_b200.checkpointing.p2p_transport", "NVLink peer-memory transport"),
    ("torchft_b200.checkpointing.durable", "durable on-disk checkpoints"),
    ("torchft_b200.parallel.team", "peer-memory team and ProcessGroupB200"),
    ("torchft_b200.parallel.hsdp", "sharded Llama trainer with a managed replica dimension"),
    ("torchft_b200.parallel.diloco", "DiLoCo on the explicit engine"),
    ("torchft_b200.models.llama", "explicit Llama engine"),
    ("torchft_b200.ops.kernels", "Python face of the sm_100a kernel library"),
    ("torchft_b200.ops.diloco", "fused DiLoCo outer step"),
    ("torchft_b200.bench_support", "manager/lighthouse set-up shared by the benchmarks and train_hsdp.py"),
    ("torchft_b200.launch.runner", "local job runner with failure injection"),
    ("torchft_b200.launch.slurm", "Slurm runner and punisher"),
    ("torchft_b200.launch.torchx", "torchx component"),
]


def _first_paragraph(obj) -> str:
    # the object's own docstring only: text inherited from torch base classes is not ours to reprint
    doc = inspect.cleandoc(getattr(obj, "__doc__", None) or "") if not isinstance(obj, property) else inspect.cleandoc(obj.__doc__ or "")
    para = doc.split("\n\n", 1)[0].strip()
    return " ".join(line.strip() for line in para.splitlines())


def _paragraphs(obj) -> list:
    doc = inspect.cleandoc(getattr(obj, "__doc__", None) or "")
    return [" ".join(line.strip() for line in para.splitlines()) for para in doc.split("\n\n") if para.strip()]


def _bound_signature(obj) -> str:
    """Signature of an extension-module (pybind11) callable: its docstring starts with ``name(args) -> ret``."""
    target = obj.__init__ if inspect.isclass(obj) else obj
    first = (getattr(target, "__doc__", None) or "").strip().splitlines()
    if first and "(" in first[0]:
        sig = first[0][first[0].index("("):]
        sig = sig.replace("torchft_b200._ftcp.", "")
        return re.sub(r"^\(self: [\w.]+(, )?", "(", sig) if inspect.isclass(obj) else sig
    return "(...)"


def _signature(obj) -> str:
    try:
        sig = str(inspect.signature(obj))
    except (TypeError, ValueError):
        return re.sub(r" at 0x[0-9a-f]+", "", _bound_signature(obj))
    sig = re.sub(r"(: |-> )(['\"])(.*?)\2", r"\1\3", sig)  # postponed annotations print as quoted strings
    sig = re.sub(r" at 0x[0-9a-f]+", "", sig)  # object addresses differ from run to run
    sig = re.sub(r"hostname: str = '[^']*'", "hostname: str = <this host's name>", sig)
    return sig


def _public_names(mod):
    names = getattr(mod, "__all__", None)
    if names is None:
        names = [n for n, v in vars(mod).items() if not n.startswith("_") and getattr(v, "__module__", None) == mod.__name__]
    return sorted(set(names))


def render() -> str:
    out = ["# API reference", "",
           "Generated by `python docs/gen_api.py`; do not edit by hand. Signatures are those of the installed sources.", ""]
    for modname, blurb in MODULES:
        mod = importlib.import_module(modname)
        out += [f"## `{modname}` — {blurb}", ""]
        head = _first_paragraph(mod)
        if head:
            out += [head, ""]
        for name in _public_names(mod):
            obj = getattr(mod, name, None)
            if obj is None or inspect.ismodule(obj):
                continue
            if inspect.isclass(obj):
                out.append(f"### class `{name}{_signature(obj)}`")
                out.append("")
                d = _first_paragraph(obj)
                if d:
                    out += [d, ""]
                methods = []
                for mname, m in sorted(vars(obj).items()):
                    if mname.startswith("_"):
                        continue
                    fn = m.__func__ if isinstance(m, (staticmethod, classmethod)) else m
                    if inspect.isfunction(fn):
                        methods.append(f"* `{mname}{_signature(fn)}`" + (f" — {_first_paragraph(fn)}" if _first_paragraph(fn) else ""))
                    elif type(m).__name__ == "instancemethod":  # a method bound by the extension module
                        methods.append(f"* `{mname}{_signature(m)}`")
                    elif isinstance(m, property):
                        methods.append(f"* `{mname}` (property)" + (f" — {_first_paragraph(m)}" if _first_paragraph(m) else ""))
                if methods:
                    out += methods + [""]
            elif callable(obj):
                out.append(f"### `{name}{_signature(obj)}`")
                out.append("")
                for d in _paragraphs(obj):
                    out += [d, ""]
    return "\n".join(out).rstrip() + "\n"


def main() -> int:
    target = Path(__file__).resolve().parent / "api.md"
    text = render()
    if "--check" in sys.argv:
        if not target.exists() or target.read_text() != text:
            print("docs/api.md is out of date: run python docs/gen_api.py")
            return 1
        return 0
    target.write_text(text)
    print(f"wrote {target} ({len(text.splitlines())} lines)")
    return 0


if __name__ == "__main__":
    sys.exit(main())
