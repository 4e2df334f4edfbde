"""layer_profile.sh's output as tables: python scratch/layer_profile_summary.py OUT (profiles/layers/listed_cases_kernel_medians.txt and listed_cases_counters.txt)"""
import collections
import csv
import glob
import os
import sys

out = sys.argv[1]


def name(row):
    n = row["Kernel_Name"]
    return n.split("ibl::(anonymous namespace)::")[1].split("(")[0] if "ibl::" in n else None


def middle(v):
    return sorted(v)[len(v) // 2]


times = collections.OrderedDict()
for r in csv.DictReader(open(os.path.join(out, "trace", "p_kernel_trace.csv"))):
    if name(r):
        times.setdefault((name(r), int(r["Grid_Size_X"])), []).append((int(r["End_Timestamp"]) - int(r["Start_Timestamp"])) / 1e3)
what = sys.argv[2]
if what == "medians":
    for (n, grid), v in times.items():
        print("%-44s grid %-10d n=%-3d median %9.2f us  min %9.2f" % (n, grid, len(v), middle(v), min(v)))
    sys.exit()

counters, under = collections.OrderedDict(), {}
for f in sorted(glob.glob(os.path.join(out, "pmc_*", "c_counter_collection.csv"))):
    for r in csv.DictReader(open(f)):
        if name(r):
            counters.setdefault((name(r), int(r["Grid_Size"])), collections.OrderedDict()).setdefault(r["Counter_Name"], []).append(float(r["Counter_Value"]))
for r in csv.DictReader(open(os.path.join(out, "pmc_wait", "c_kernel_trace.csv"))):
    if name(r):
        under.setdefault((name(r), int(r["Grid_Size_X"])), []).append((int(r["End_Timestamp"]) - int(r["Start_Timestamp"])) / 1e3)
print("""Counters of the listed cases' kernels of 50 us and more (rocprofv3 --pmc, a run for each pass; medians a launch; us and GHz are the counted run's).
HBM read = 2 x FETCH_SIZE KiB, written = WRITE_SIZE KiB, at the time without counters; cycles = GRBM_GUI_ACTIVE / 8 XCDs; matrix cores = SQ_VALU_MFMA_BUSY_CYCLES and
vector units = 4 SQ_ACTIVE_INST_VALU (matrix instructions' issue among them) of cycles x 1 024 SIMDs; LDS = SQ_LDS_IDX_ACTIVE of cycles x 256 CUs, and its share that is
conflicts; address units = TA_BUSY of cycles; waiting = SQ_WAIT_ANY of SQ_WAVE_CYCLES.
""")
for (n, grid), c in counters.items():
    m = {k: middle(v) for k, v in c.items()}
    t = middle(times[(n, grid)]) if (n, grid) in times else 0
    if t < 50:
        continue
    cyc, tc = m["GRBM_GUI_ACTIVE"] / 8, middle(under[(n, grid)])
    print("%s grid %d: %.0f us (%.0f counted, %.2f GHz)" % (n, grid, t, tc, cyc / tc / 1e3))
    read, written = 2 * 1024 * m["FETCH_SIZE"], 1024 * m["WRITE_SIZE"]
    print("    HBM read %.3f GB, written %.3f GB: %.2f TB/s; L2 hits %.0f %% of %.1f M requests" % (read / 1e9, written / 1e9, (read + written) / t / 1e6, 100 * m["TCC_HIT_sum"] / m["TCC_REQ_sum"], m["TCC_REQ_sum"] / 1e6))
    print("    matrix cores %.0f %%, vector units %.0f %%, LDS %.0f %% (conflicts %.0f %% of it), address units %.0f %%; waves waiting %.0f %%, on LDS %.0f %%" % (
        100 * m["SQ_VALU_MFMA_BUSY_CYCLES"] / (cyc * 1024), 400 * m["SQ_ACTIVE_INST_VALU"] / (cyc * 1024), 100 * m["SQ_LDS_IDX_ACTIVE"] / (cyc * 256),
        100 * m["SQ_LDS_BANK_CONFLICT"] / max(1.0, m["SQ_LDS_IDX_ACTIVE"]), 100 * m["TA_BUSY_avr"] / cyc, 100 * m["SQ_WAIT_ANY"] / m["SQ_WAVE_CYCLES"], 100 * m["SQ_WAIT_INST_LDS"] / m["SQ_WAVE_CYCLES"]))
