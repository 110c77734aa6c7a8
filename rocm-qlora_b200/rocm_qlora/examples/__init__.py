"""Small programs that run the package's operators together."""
