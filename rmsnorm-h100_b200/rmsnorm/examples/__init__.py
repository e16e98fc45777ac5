# SPDX-License-Identifier: MIT
"""Examples of the package's operators together."""
