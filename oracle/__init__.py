"""CPU oracle for the HALO chunked-attention hot path.

TEST INFRASTRUCTURE ONLY. Nothing in the shipped package (``halo_b200``)
imports, links or executes anything under ``oracle/``. Only ``tests/``,
``__graft_entry__.smoke()`` and the CPU-baseline leg of ``bench.py`` use it,
and only as the checker or the timed CPU reference, never as the product.

Each function restates one piece of the reference algorithm on the CPU and
cites the reference ``file:line`` it follows (paths are relative to the
lzbaclz/HALO project root):

* ``oracle.attention`` -- chunk attention, two-way LSE merge and the
  cold+recent walk (``halo/kv_cache_chunked.py``), plus the (m, l, o)
  accumulator semantics of ``halo/triton_chunked.py``.  torch CPU, fp32.
* ``oracle.scorer`` -- Quest page summaries, GQA mean-pooled upper-bound
  scores and top-k (``baselines/quest_path_d.py``).  numpy.
* ``oracle.kivi`` -- KIVI per-group quantise / dequantise with per-op fp16 /
  bf16 rounding (``baselines/kivi_cache.py``).  numpy, cross-checked against
  the plain-C restatement in ``oracle/kivi_ref.c`` (built by
  ``oracle/Makefile`` into ``oracle/_build/liboracle_kivi.so``).
* ``oracle.paged`` -- block tables, row moves and tree attention of the paged
  cache (no reference counterpart: written from the definitions).  torch CPU,
  64 bits.

Pinning: every function of the reference's algorithm is checked against golden vectors that were
generated by running the reference's own Python code in the build container
(``tests/golden/make_golden.py``; fixtures in ``tests/golden/*.npz``).
"""
