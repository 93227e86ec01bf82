"""Per-launch HBM traffic of the bench's kernels from separate rocprofv3 --pmc
FETCH_SIZE / WRITE_SIZE passes (tools/profile_round.sh), corrected as
MI355X_MICROARCH.md prescribes for gfx950 (FETCH_SIZE counts half of the
bytes of wide coalesced reads: doubled; both counters in KB), written as
profiles/pmc_traffic.json for bench.py's roofline.traffic.
python tools/pmc_traffic.py <fetch dir> <write dir> <workload> <out.json> [source note]"""
import hashlib
import json
import os
import sys

sys.path.insert(0, __file__.rsplit("/", 1)[0])
from hbm_summary import load  # noqa: E402

# bench.py kernel names -> fragments of the mangled kernel symbols
NAMES = {
    "qkv_attention": ["qkv_attention_pc_kernel", "qkv_attention_kernel"],
    "gemm_up_gelu": ["i8_up_gelu_kernel", "q4r_up_gelu_kernel", "gemm_kernelILi2ELi1", "gemm_kernel<2, 1,"],
    # o-proj: the split-fp16 LN GEMM (rounds 2-5 default) or the int8 one (round 6
    # default for Q4_0, the same kernel as FFN-down: main() splits its dispatches)
    "gemm_o_ln": ["gemm_kernelILi2ELi2", "gemm_kernel<2, 2,", "i8_ln384_kernel"],
    "gemm_down_ln": ["i8_ln384_kernel", "gemm_kernelILi2ELi2", "gemm_kernel<2, 2,"],
    "embed_ln": ["embed_ln_kernel"],
    "pool_l2": ["pool_l2_kernel"],
}


def main():
    fetch, write = load(sys.argv[1], "FETCH_SIZE"), load(sys.argv[2], "WRITE_SIZE")
    out = {"workload": sys.argv[3], "source": sys.argv[5] if len(sys.argv) > 5 else "", "bytes_per_launch": {},
           "fetch_bytes": {}, "write_bytes": {},
           "note": "FETCH_SIZE x2 + WRITE_SIZE, KB -> bytes, per dispatch; each name takes the kernels of "
                   "its first symbol fragment that occurs; names on one kernel split its dispatches in order"}
    # the build these counters describe (bench.py marks the traffic stale for any other build)
    repo = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    lib = os.path.join(repo, "build", "libbert.so")
    if os.path.exists(lib):
        with open(lib, "rb") as f:
            out["lib_sha256"] = hashlib.sha256(f.read()).hexdigest()
    bi = os.path.join(repo, "build", "BUILD_INFO")
    if os.path.exists(bi):
        with open(bi) as f:
            out["git_head"] = f.read().strip()
    out["kernel_symbols"] = sorted(set(fetch) | set(write))
    keys = set(fetch) | set(write)

    def resolve(frags):
        for f in frags:
            hit = sorted(k for k in keys if f in k)
            if hit:
                return hit
        return []

    hits = {name: resolve(frags) for name, frags in NAMES.items()}
    # names that resolve to the same kernel (o-proj and FFN-down both on
    # i8_ln384_kernel): its dispatches alternate o, down in every layer (one row
    # group, BERT_AMD_SPLIT=0), so they are dealt out in dispatch order
    share = {}
    for name, h in hits.items():
        share.setdefault(tuple(h), []).append(name)
    out["shared_kernels"] = {", ".join(v): list(k) for k, v in share.items() if len(v) > 1 and k}
    for name, frags in NAMES.items():
        fv, wv = [], []
        group = share.get(tuple(hits[name]), [name])
        slot, n_share = group.index(name), len(group)
        for src, dst in ((fetch, fv), (write, wv)):
            # of all the kernels it resolves to in one order: the last layer's FFN-down is another one
            ds = sorted((kv for k in hits[name] for kv in src.get(k, {}).items()),
                        key=lambda kv: int(kv[0]) if str(kv[0]).isdigit() else 0)
            dst += [v for i, (_, v) in enumerate(ds) if i % n_share == slot]
        if fv and wv:
            fb = 2.0 * sum(fv) / len(fv) * 1024.0
            wb = sum(wv) / len(wv) * 1024.0
            out["fetch_bytes"][name] = round(fb)
            out["write_bytes"][name] = round(wb)
            out["bytes_per_launch"][name] = round(fb + wb)
    # whole step: every layer kernel launches n_layer (6) times per step, embed and pool once
    per_step = {"embed_ln": 1, "pool_l2": 1}
    bl = out["bytes_per_launch"]
    step = list(NAMES)
    if all(k in bl for k in step):
        out["bytes_per_step"] = round(sum(bl[k] * per_step.get(k, 6) for k in step))
    with open(sys.argv[4], "w") as f:
        json.dump(out, f, indent=1)
    print(json.dumps(out["bytes_per_launch"]))


if __name__ == "__main__":
    main()
