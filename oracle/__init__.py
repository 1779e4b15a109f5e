"""CPU oracle for the block-sparse attention path -- TEST INFRASTRUCTURE ONLY.

This package restates, on the CPU, what the reference computes on the path the
product accelerates.  It is the checker the parity tests, ``__graft_entry__.smoke``
and ``bench.py``'s CPU-baseline leg compare against.  Nothing in the product
package (``polyhedral_b200``) imports it, and no product call falls back to it.

Pinned: every function here (the operators that the reference lacks are stated in
``paged_oracle``, against nothing but their definitions) is checked against golden vectors generated by the
reference's own Python (``tests/golden/make_golden.py``) in ``tests/test_oracle_golden.py``.
"""
from .polyattn_oracle import *  # noqa: F401,F403
