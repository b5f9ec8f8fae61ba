"""Runs the checks of leaf_ops_checks.py in a process that imports torch before the library,
as programs that hold torch tensors do: the library then shares torch's HIP runtime.  (The
rest of the GPU tests run without torch, on the runtime that the library is linked to.)

One JSON line in for each check, {"name": ..., "args": {...}}; one out, {"error": text or
null}.  The process ends when its input does.
"""
import json
import os
import sys
import traceback

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))


def main():
    answers = os.fdopen(os.dup(1), "w")
    os.dup2(2, 1)  # what a check prints does not get between the answers
    torch.zeros(1, device="cuda")
    from tests import leaf_ops_checks as checks
    answers.write(json.dumps({"error": None}) + "\n")
    answers.flush()
    for line in sys.stdin:
        asked = json.loads(line)
        print(asked, file=sys.stderr, flush=True)
        error = None
        try:
            getattr(checks, asked["name"])(**asked["args"])
            torch.cuda.synchronize()
        except Exception:
            error = traceback.format_exc()
        answers.write(json.dumps({"error": error}) + "\n")
        answers.flush()
    checks.close()


main()
