"""Small programs that use the package as its callers do."""
