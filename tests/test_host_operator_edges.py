"""Refusals and host-side choices of the operators on long shared caches: nothing is launched (no GPU needed)."""
