"""The kernel launches of calls of the operators on logits, without a GPU:
launches.py with descriptors {"logits": [...]} and {"distill": [...]}."""
import ctypes as C
import json
import os
import subprocess
import sys

import launches

HERE = os.path.dirname(os.path.abspath(__file__))


def main(recorder):
    rec = C.CDLL(recorder, mode=C.RTLD_GLOBAL)
    rec.rec_launch.restype = C.POINTER(launches.Launch)
    sys.path.insert(0, os.path.join(os.path.dirname(HERE), "aet-cnn_amd"))
    import aetcnn
    ops, out = aetcnn.ops(), []
    make = {"logits": aetcnn.LogitsDesc, "distill": aetcnn.DistillDesc}
    for name, args in json.load(sys.stdin):
        rec.rec_reset()
        a = []
        for i, v in enumerate(args):
            if isinstance(v, dict):
                (kind, fields), = v.items()
                v = C.byref(make[kind](*fields))
            a.append((i + 1) << 32 if v == "p" else v)
        rc = getattr(ops, name)(*a)
        ls = [rec.rec_launch(i)[0] for i in range(rec.rec_count())]
        out.append(dict(rc=rc, launches=[dict(grid=list(v.grid), block=list(v.block), lds=v.lds,
                                              lds_limit=v.lds_limit) for v in ls]))
    json.dump(out, sys.stdout)


def record(calls, tmp_path):
    so = os.path.join(str(tmp_path), "recorder.so")
    subprocess.run(["gcc", "-shared", "-fPIC", "-O1", "-o", so,
                    os.path.join(HERE, "launch_recorder.c")], check=True)
    r = subprocess.run([sys.executable, os.path.join(HERE, "logits_launches.py"), so],
                       input=json.dumps(calls), capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr
    return json.loads(r.stdout)


if __name__ == "__main__":
    main(sys.argv[1])
